// C interface of the kernels around one step of a serving batch: layout of the batch (batch_layout.cu), attention of
// sequences that begin with the same tokens (prefix_attn.cu), log probabilities of what was chosen (token_log_probs.cu).
// Types, status word and return codes as in ortb200_kernels.h: 0, -1 a missing or impossible argument, -2 a size or form that
// the kernel does not take, -3 alignment, -4 type, -6 / -10 / -11 a refusal of the CUDA runtime.
#pragma once
#include "ortb200_kernels.h"

#ifdef __cplusplus
extern "C" {
#endif

// Block table, packing, positions and cache slots of a batch out of the lengths of its requests, all in one launch.
//   held_b = ceil(past_b / s), need_b = ceil((past_b + new_b) / s) - held_b, first_b = sum of need over the requests before b
//   table_out[b, j] = free_blocks[first_b + j - held_b] for held_b <= j < held_b + need_b, else table_in[b, j]
//   cum[b] = sum of new over the requests before b; row t of request b: position past_b + t - cum[b], slot = block * s + offset
// Rows behind the last request get position and slot -1.  blocks_used: the sum of need, or, when the batch cannot be laid out,
// -1 (too few free blocks), -2 (the table is too narrow), -3 (more tokens than rows) or -4 (a negative length): then the table
// stays as it was, cum is 0 and every position and slot -1, and the status word, if there is one, says so too.
typedef struct {
  const int* past_seqlens;    // [B]
  const int* new_tokens;      // [B]
  const int* table_in;        // [B, max_blocks]
  const int* free_blocks;     // [num_free], may be null when num_free is 0
  int* table_out;             // [B, max_blocks]; may be table_in
  int* cum;                   // [B + 1]
  int64_t* positions;         // [rows]
  int64_t* slot_mapping;      // [rows]
  int* blocks_used;           // [1]
  int B, max_blocks, block_size;
  int64_t num_free, rows;
  int* status;                // null: blocks_used alone reports a refusal
} ortb200_batch_layout_args;
int ortb200_batch_layout(const ortb200_batch_layout_args* args, ortb200_stream_t stream);
int ortb200_batch_layout_max_requests(void);
int64_t ortb200_batch_layout_max_rows(void);

// Attention of packed queries over a paged cache whose sequences share their first *shared_prefix tokens: rotary embedding and
// cache append, then the keys of the prefix (rounded down to whole tiles of 64, cut to the shortest past) once for the rows of
// all sequences and every sequence's own keys for its own rows, joined by their softmax maxima and sums.
// workspace: ortb200_prefix_attn_workspace_bytes(), 256-byte aligned, any content.  With tensor_cores the caches and out are 16-byte
// aligned.
typedef struct {
  const void* qkv;            // [T, (N + 2 Nk) H], or queries alone [T, N H] when k and v are given
  const void* k;              // [T, Nk H]
  const void* v;
  void* k_cache;              // [num_blocks, block_size, Nk, H]
  void* v_cache;
  const int* cu_seqlens;      // [B + 1]
  const int* past_seqlens;    // [B]: tokens in the cache, the shared ones among them
  const int* block_table;     // [B, max_blocks]
  const int* shared_prefix;   // [1]
  const void* cos_cache;      // [cos_rows, rot_dim / 2], null: no rotary embedding
  const void* sin_cache;
  const int64_t* positions;   // [T] and
  const int64_t* slot_mapping;  // [T]: rotary position and cache slot of every row; both null: from the lengths and the table
  void* out;                  // [T, N H]; rows of no sequence become 0
  void* workspace;
  int64_t workspace_bytes;
  int64_t T;
  int B, N, Nk, H;
  int block_size, max_blocks, num_blocks;
  int cos_rows, rot_dim, interleaved;
  float scale;                // 0: 1 / sqrt(H)
  float softcap;              // 0: none
  int dtype;
  int tensor_cores;           // 1: tcgen05 (16-bit types, H 64 or 128, blocks of 8, 16, 32 or a multiple of 64); 0: any type, H <= 256
  int use_pdl;
  int* status;
} ortb200_prefix_attn_args;
int ortb200_prefix_attn(const ortb200_prefix_attn_args* args, ortb200_stream_t stream);
int64_t ortb200_prefix_attn_max_keys(void);   // of a sequence: max_blocks x block_size
int64_t ortb200_prefix_attn_workspace_bytes(int64_t T, int B, int N, int Nk, int H, int tensor_cores);

// Row by row over logits x [rows, vocab], with m the largest and S = sum exp(x - m):
//   log_sum_exp = m + log S;  log_prob = (x[token] - m) - log S;  entropy = log S - sum exp(x - m) (x - m) / S
// and the top_k largest, equal ones by the lower index.  A token outside [0, vocab) is padding: log_prob 0.
// log_sum_exp_rest is what rounding took from log_sum_exp (2^-24 of m, which may be more than log S): x - log_sum_exp - log_sum_exp_rest
// is the log probability of every x.
typedef struct {
  const void* logits;         // [rows, vocab] dtype
  const int64_t* tokens;      // [rows]
  float* log_prob;            // [rows]; outputs may be null
  float* entropy;             // [rows]
  float* log_sum_exp;         // [rows]
  float* top_log_probs;       // [rows, top_k]
  int64_t* top_tokens;        // [rows, top_k]
  float* log_sum_exp_rest;    // [rows]
  int64_t rows;
  int vocab, top_k;           // 0 <= top_k <= min(32, vocab)
  int dtype;
  int use_pdl;
} ortb200_token_log_probs_args;
int ortb200_token_log_probs(const ortb200_token_log_probs_args* args, ortb200_stream_t stream);
int ortb200_token_log_probs_max_vocab(void);

//   d_logits[v] = p_v (d_log_sum_exp - d_log_prob - sum_k d_top[k] - d_entropy (log p_v + entropy))
//                 + d_log_prob [v = token] + sum_k d_top[k] [v = top_tokens[k]]
// with log p_v = logits[v] - log_sum_exp - log_sum_exp_rest.  d_logits may be logits.  Of the gradients any may be null; a padding
// token has no d_log_prob.
typedef struct {
  const void* logits;
  const int64_t* tokens;
  const float* log_sum_exp;
  const float* entropy;         // needed with d_entropy
  const float* d_log_prob;      // [rows]
  const float* d_entropy;       // [rows]
  const int64_t* top_tokens;    // [rows, top_k], needed with d_top_log_probs
  const float* d_top_log_probs; // [rows, top_k]
  const float* d_log_sum_exp;   // [rows]
  const float* log_sum_exp_rest;  // [rows], null: 0
  void* d_logits;               // [rows, vocab] dtype
  int64_t rows;
  int vocab, top_k;
  int dtype;
  int use_pdl;
} ortb200_token_log_probs_grad_args;
int ortb200_token_log_probs_grad(const ortb200_token_log_probs_grad_args* args, ortb200_stream_t stream);

#ifdef __cplusplus
}
#endif
