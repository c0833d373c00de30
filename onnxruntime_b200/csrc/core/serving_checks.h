// Operands of the serving operators (kernels_serving.cc, kernels_drafts.cc, kernels_cuda5.cc, kernels_cuda6.cc), checked the same way for every provider.
#pragma once
#include <ATen/ATen.h>

#include "kernel.h"

namespace ortb {

// Two tensors have memory in common.  (By addresses: buffers that are bound by their pointers have storages of their own.)
inline bool Overlap(const at::Tensor& a, const at::Tensor& b) {
  const auto end = [](const at::Tensor& t) {
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    return static_cast<const char*>(t.data_ptr()) + (last + 1) * t.element_size();
  };
  return a.defined() && b.defined() && a.numel() > 0 && b.numel() > 0 && a.device() == b.device() && a.data_ptr() < static_cast<const void*>(end(b)) &&
         b.data_ptr() < static_cast<const void*>(end(a));
}

// com.ortb200 SharedPrefixPagedAttention and, with parents in the place of shared_prefix and nothing behind sin_cache, TreePagedAttention
// inputs: query, key?, value?, key_cache, value_cache, cumulative_sequence_length, past_seqlens, block_table, shared_prefix,
//         cos_cache?, sin_cache?, positions?, slot_mapping?
struct SharedPrefixSizes {
  int64_t T = 0, B = 0, N = 0, Nk = 0, H = 0;
  int64_t block_size = 0, num_blocks = 0, max_blocks = 0, rot_dim = 0;
  bool packed = true, rotary = false, interleaved = false, placed = false;   // placed: positions and slots are given
  bool tree = false;     // the rows of a sequence form a tree
  float scale = 0.f, softcap = 0.f;
};
SharedPrefixSizes CheckSharedPrefix(OpKernelContext& ctx);
constexpr int64_t kMostTreeNodes = 256;   // of a sequence; more rows are a prompt, each row behind the one before it
SharedPrefixSizes CheckTreeAttention(OpKernelContext& ctx);

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

// com.ortb200 PagedCacheMove: sources, targets, caches...
struct CacheMoveSizes {
  int64_t moves = 0, units = 0;   // units of a cache: its tokens, or with `blocks` its blocks
  int caches = 0;
  bool blocks = false;
};
CacheMoveSizes CheckCacheMove(OpKernelContext& ctx);

// com.ortb200 ProcessLogits: logits, history?, history_starts?, generated_starts?, row_list?, drafted?, repetition?, presence?,
// frequency?, bias_tokens?, bias_values?, bias_starts?, allowed?, row_mask?, temperature?
struct ProcessLogitsSizes {
  int64_t rows = 0, vocab = 0, lists = 0, history = 0, drafted = 0, biases = 0, masks = 0, mask_words = 0;
};
ProcessLogitsSizes CheckProcessLogits(OpKernelContext& ctx);

}  // namespace ortb
