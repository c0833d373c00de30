// C interface of the kernels around a decode step with drafted tokens: attention of a tree of drafted tokens over a paged cache
// (prefix_attn.cu), the move of cache entries (cache_move.cu), penalties, biases and masks on logits (process_logits.cu).
// Types, status word and return codes as in serving_ops.h.
#pragma once
#include "serving_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

// Attention of packed queries over a paged cache, where the new rows of a sequence form a tree: row i of a sequence (counted from
// its first row) has the parent parents[t] < i, or -1, the last token in the cache.  It sees the tokens in the cache, its
// ancestors and itself; its rotary position is past + depth, its key and value go to place past + i of the sequence.
// Up to ortb200_tree_attn_max_nodes() rows of a sequence form a tree; of more, every row's parent has to be the one before it.
// A parent that is none (i or behind it, or below -1) is reported through the status word, and the row counted as a root.
// attn: shared_prefix, positions and slot_mapping are null, the rest as for ortb200_prefix_attn; the workspace has
// ortb200_tree_attn_workspace_bytes().
typedef struct {
  ortb200_prefix_attn_args attn;
  const int* parents;   // [T]
} ortb200_tree_attn_args;
int ortb200_tree_attn(const ortb200_tree_attn_args* args, ortb200_stream_t stream);
int ortb200_tree_attn_max_nodes(void);
int64_t ortb200_tree_attn_workspace_bytes(int64_t T, int B, int N, int Nk, int H, int tensor_cores);

// cache[targets[m]] = cache[sources[m]] for every cache and every move, as if all sources were read before any target is written.
// A cache is `units` units of unit_bytes[c] bytes.  A negative target is no move; a place outside the cache, or a target that is
// named twice, is reported through the status word (the former is left out; what lies at the latter then comes from any of its moves, piece by piece).
// The caches do not overlap.
typedef struct {
  void* const* caches;          // [num_caches], host array
  const int64_t* unit_bytes;    // [num_caches], host array
  int num_caches;
  int64_t units;
  const int64_t* sources;       // [moves]
  const int64_t* targets;       // [moves]
  int64_t moves;                // up to ortb200_cache_move_max_moves()
  int use_pdl;
  int* status;
} ortb200_cache_move_args;
int ortb200_cache_move(const ortb200_cache_move_args* args, ortb200_stream_t stream);
int64_t ortb200_cache_move_max_moves(void);

// Row by row over logits x [rows, vocab], in 32 bits, in this order:
//   c: how often the token occurs in the row's text, counted from generated_starts of its list on, and seen: whether it occurs at all
//   seen:      x = x < 0 ? x repetition : x / repetition
//   always:    x = x - (frequency c + presence [c > 0])
//   biased:    x = x + the sum of the token's biases, in their order; -inf where that sum is -inf, whatever x is
//   masked:    x = -inf where the row's mask has the bit 0
//   always:    x = x / temperature (a temperature that is not above 0 leaves x)
// The text of a row is the tokens of its list, history[history_starts[l], history_starts[l + 1]), and the `drafted_width` tokens of its
// row of `drafted`; tokens outside [0, vocab) are none.  Any input but logits may be null; presence and frequency need history or
// drafted tokens to mean anything.
typedef struct {
  const void* logits;               // [rows, vocab] dtype
  float* scores;                    // [rows, vocab]
  const int64_t* history;           // [history_len]
  const int64_t* history_starts;    // [lists + 1]
  const int64_t* generated_starts;  // [lists], places in `history`; null: all of a list counts
  const int* row_list;              // [rows]; null: row r has list r; a negative one: none
  const int64_t* drafted;           // [rows, drafted_width]
  const float* repetition;          // [rows]; null: 1
  const float* presence;            // [rows]; null: 0
  const float* frequency;           // [rows]; null: 0
  const int64_t* bias_tokens;       // [bias_len]
  const float* bias_values;         // [bias_len]
  const int64_t* bias_starts;       // [rows + 1]; may be given without biases
  const int* allowed;               // [masks, mask_words]: bit v % 32 of word v / 32 is token v's
  const int* row_mask;              // [rows]; a negative one: no mask
  const float* temperature;         // [rows]; null: 1
  int64_t rows, history_len, bias_len;
  int64_t lists;
  int vocab, drafted_width, masks, mask_words;
  int dtype;
  int use_pdl;
  int* status;                      // lists, masks and starts that are none are reported, and left out
} ortb200_process_logits_args;
int ortb200_process_logits(const ortb200_process_logits_args* args, ortb200_stream_t stream);
int ortb200_process_logits_max_vocab(void);

#ifdef __cplusplus
}
#endif
