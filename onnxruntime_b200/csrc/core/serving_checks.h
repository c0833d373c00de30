// Operands of the serving operators (kernels_serving.cc, kernels_cuda5.cc), checked the same way for every provider.
#pragma once
#include <ATen/ATen.h>

#include "kernel.h"

namespace ortb {

// com.ortb200 SharedPrefixPagedAttention
// inputs: query, key?, value?, key_cache, value_cache, cumulative_sequence_length, past_seqlens, block_table, shared_prefix,
//         cos_cache?, sin_cache?, positions?, slot_mapping?
struct SharedPrefixSizes {
  int64_t T = 0, B = 0, N = 0, Nk = 0, H = 0;
  int64_t block_size = 0, num_blocks = 0, max_blocks = 0, rot_dim = 0;
  bool packed = true, rotary = false, interleaved = false, placed = false;   // placed: positions and slots are given
  float scale = 0.f, softcap = 0.f;
};
SharedPrefixSizes CheckSharedPrefix(OpKernelContext& ctx);

// com.ortb200 PagedBatchLayout: past_seqlens, new_tokens, block_table, free_blocks, rows
struct BatchLayoutSizes {
  int64_t B = 0, max_blocks = 0, num_free = 0, rows = 0, block_size = 0;
  bool strict = false;   // a batch that cannot be laid out is an error of the run, not of `blocks_used` alone
};
BatchLayoutSizes CheckBatchLayout(OpKernelContext& ctx);

// com.ortb200 TokenLogProbs: logits, tokens.  com.ortb200 TokenLogProbsGrad: logits, tokens, log_sum_exp, entropy?, d_log_prob?,
// d_entropy?, top_tokens?, d_top_log_probs?, d_log_sum_exp?, log_sum_exp_rest?
struct TokenLogProbsSizes {
  int64_t rows = 0, vocab = 0, top_k = 0;
  std::vector<int64_t> lead;   // shape of one value per row
};
TokenLogProbsSizes CheckTokenLogProbs(OpKernelContext& ctx);
TokenLogProbsSizes CheckTokenLogProbsGrad(OpKernelContext& ctx);

}  // namespace ortb
