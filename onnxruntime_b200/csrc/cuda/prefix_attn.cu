// Attention of a batch whose sequences begin with the same tokens (com.ortb200.SharedPrefixPagedAttention).
//
// softmax(q K^T) V splits over any partition of the keys: with m the largest score of a part, l = sum exp(s - m) and
// o = sum exp(s - m) v, two parts join as m = max(m1, m2), l = l1 e^(m1 - m) + l2 e^(m2 - m), o likewise; the result is o / l.
//
// Step 1 rotates the queries and the new keys and appends keys and values to the cache; step 2 attends; step 3 joins the parts.
//
// Tensor-core form.  A unit of work is a tile of up to 128 query rows (a row is one token and one of the G query heads that
// share a key head) against the keys of one key head: rows of all sequences against the prefix, or rows of one sequence
// against its own keys.  The units' 64-key tiles are numbered consecutively and every CTA takes an equal share of the numbers,
// so that one long prefix and many short tails fill the machine alike, without a word about it from the host, which does not
// know the lengths.  A CTA's share of a unit is a segment; it leaves (m, l, o) of its rows in 32 bits, and step 3 joins the
// segments of a row.  Which CTA wrote what follows from the same arithmetic: nothing is counted, nothing waited for.
//
// Within a CTA (192 threads, two per SM): warp 0 loads tiles by TMA through the block table, warp 1 issues the products
// (S = Q K^T into tensor memory, O += P V with P in tensor memory over the scores), warps 2 to 5 hold one row per thread.  Units of
// up to eight rows, which sequences with single tokens have, leave tensor memory out: those four warps multiply themselves, out of
// the same tiles (few_rows).
//
// What bounds it.  Many rows (24 prompts of up to 150 tokens behind 6000, 28 heads of 128): the tensor pipe, which has half as much
// again to do as the formula because weights count as two 16-bit values; a tile of 128 rows and 64 keys takes 768 clocks of it and
// a CTA is done with one in 2000 to 2500, two CTAs side by side; 512 clocks of exponentials per tile run beside it.  284 us in all on
// one GPU, of which the product kernel has 234 and the join 37, and up to 330 on others, whose clocks settle lower.  Single tokens behind a long prefix: segments and their hand-overs; 180 sequences of 16
// heads of 64 behind 20011 tokens take 117 us, 64 of 64 heads of 128 behind 8192 tokens 61 to 63 us, where the bytes need 37 and 23.
// Slower, each against the form of its time at (180 behind 20011, 64 behind 8192): 128-key tiles with one score buffer 164 and 82 us
// instead of 149 and 70; eight softmax warps with half a row each 150 and 80; rows held four times with a quarter of the keys to each
// warp 162 and 78; the next tiles asked into L2 ahead of their loads 198 and 81 instead of 132 and 65; one thread for loads and
// scores and one for the products with V 147 and 72 instead of 140 and 67; few rows through tensor memory like all others 139 and 68
// instead of 115 and 64.
#include <cuda.h>
#include <cuda_runtime.h>
#include <math.h>
#include <algorithm>
#include <type_traits>
#include "attn_internal.h"
#include "launch_util.cuh"
#include "serving_ops.h"
#include "tensor_map.h"

namespace ortb200 {
namespace {

constexpr int kMaxHead = 256;
constexpr long long kMaxKeys = 0x7fff0000;

// Lengths of sequence b, cut to what the buffers hold: rows [row0, row0 + rows) of the batch, keys [0, past + rows) of the cache.
struct Span {
  int row0, rows, past;
};
__device__ __forceinline__ Span span_of(const ortb200_prefix_attn_args& a, int b) {
  const int T = static_cast<int>(a.T), cap = static_cast<int>(min(static_cast<long long>(a.max_blocks) * a.block_size, 0x7fffffffll));
  Span s;
  s.row0 = min(max(a.cu_seqlens[b], 0), T);
  s.rows = max(min(max(a.cu_seqlens[b + 1], 0), T) - s.row0, 0);
  s.past = min(max(a.past_seqlens[b], 0), cap);
  return s;
}
__device__ __forceinline__ int last_row(const ortb200_prefix_attn_args& a) {
  return a.B == 0 ? 0 : min(max(a.cu_seqlens[a.B], 0), static_cast<int>(a.T));   // (without sequences there are no lengths and no table to read)
}

// Lengths of sequence b that fit neither the batch nor the table are cut, and reported.
__device__ __forceinline__ void check_lengths(const ortb200_prefix_attn_args& a, int b, const Span& s, int* status) {
  const bool batch = a.cu_seqlens[b] >= 0 && a.cu_seqlens[b + 1] >= a.cu_seqlens[b] && a.cu_seqlens[b + 1] <= a.T;
  const bool table = s.rows == 0 || (a.past_seqlens[b] == s.past && s.past + static_cast<long long>(s.rows) <= static_cast<long long>(a.max_blocks) * a.block_size);
  if (!batch || !table) atomicExch(status, kStatusBadLength);
}

// Rows in front of the first sequence, and those between lengths that run backwards, are nobody's: nothing of them is cached.
__device__ __forceinline__ bool owned(const ortb200_prefix_attn_args& a, int b, int t) { return t >= a.cu_seqlens[b] && t < a.cu_seqlens[b + 1]; }

// CTA t: rotate row t's query heads into `q_out` [T, N, H], its key heads into the cache beside the values.
template <typename T>
__global__ void __launch_bounds__(128) prefix_prep_kernel(const ortb200_prefix_attn_args a, T* q_out) {
  const int t = blockIdx.x, H = a.H, heads = a.N + 2 * a.Nk, half = a.rot_dim / 2;
  pdl_wait_prior_grids();
  if (t == a.T) {   // one more CTA for the lengths
    if (a.status)
      for (int b = threadIdx.x; b < a.B; b += blockDim.x) check_lengths(a, b, span_of(a, b), a.status);
    return;
  }
  if (t >= last_row(a)) return;
  const int b = sequence_of(a.cu_seqlens, a.B, t);
  if (!owned(a, b, t)) return;
  const long long place = static_cast<long long>(a.past_seqlens[b]) + (t - a.cu_seqlens[b]);
  long long slot, pos = place;
  if (a.positions) {
    pos = a.positions[t];
    slot = a.slot_mapping[t];
  } else {
    const long long j = place / a.block_size;
    slot = place >= 0 && j < a.max_blocks ? static_cast<long long>(a.block_table[static_cast<long long>(b) * a.max_blocks + j]) * a.block_size + place % a.block_size : -1;
  }
  const bool keep = slot >= 0 && slot < static_cast<long long>(a.num_blocks) * a.block_size;
  if (!keep && threadIdx.x == 0 && a.status) atomicExch(a.status, kStatusBadArgument);
  if (a.cos_cache && (pos < 0 || pos >= a.cos_rows)) {   // never past the rotary tables
    if (threadIdx.x == 0 && a.status) atomicExch(a.status, kStatusBadLength);
    pos = pos < 0 ? 0 : a.cos_rows - 1;
  }
  const T* cosr = a.cos_cache ? static_cast<const T*>(a.cos_cache) + pos * half : nullptr;
  const T* sinr = a.cos_cache ? static_cast<const T*>(a.sin_cache) + pos * half : nullptr;
  for (int idx = threadIdx.x; idx < heads * H; idx += blockDim.x) {
    const int head = idx / H, d = idx % H;
    const int kind = head < a.N ? 0 : head < a.N + a.Nk ? 1 : 2;
    const T* src;
    if (a.k == nullptr) src = static_cast<const T*>(a.qkv) + static_cast<long long>(t) * heads * H + head * H;
    else if (kind == 0) src = static_cast<const T*>(a.qkv) + static_cast<long long>(t) * a.N * H + head * H;
    else src = static_cast<const T*>(kind == 1 ? a.k : a.v) + static_cast<long long>(t) * a.Nk * H + (head - (kind == 1 ? a.N : a.N + a.Nk)) * H;
    T y = src[d];
    if (kind < 2 && cosr && d < a.rot_dim) {
      const int i = a.interleaved ? d >> 1 : d % half;
      const bool upper = a.interleaved ? d & 1 : d >= half;
      const float c = to_float<T>(cosr[i]), s = to_float<T>(sinr[i]), own = to_float<T>(src[d]);
      const float other = to_float<T>(src[a.interleaved ? d ^ 1 : upper ? d - half : d + half]);
      y = from_float<T>(upper ? own * c + other * s : own * c - other * s);
    }
    if (kind == 0) q_out[(static_cast<long long>(t) * a.N + head) * H + d] = y;
    else if (keep) static_cast<T*>(kind == 1 ? a.k_cache : a.v_cache)[(slot * a.Nk + (head - (kind == 1 ? a.N : a.N + a.Nk))) * H + d] = y;
  }
}

// One warp per row and query head, any type and any head size up to 256: lane i holds the elements i, i + 32, ... of the head.
// It reads the table row of its own sequence, which names the shared blocks too.
template <typename T>
__global__ void __launch_bounds__(128) prefix_rows_kernel(const ortb200_prefix_attn_args a, const T* q) {
  constexpr int R = kMaxHead / 32;
  const int lane = threadIdx.x & 31, H = a.H;
  const long long item = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  pdl_wait_prior_grids();
  if (item >= a.T * a.N) return;
  const int t = static_cast<int>(item / a.N), head = static_cast<int>(item % a.N), kvh = head / (a.N / a.Nk);
  T* out = static_cast<T*>(a.out) + item * H;
  float o[R], qv[R], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r) o[r] = 0.f;
  const int b = t < last_row(a) ? sequence_of(a.cu_seqlens, a.B, t) : -1;
  if (b >= 0 && owned(a, b, t)) {
    const Span s = span_of(a, b);
    const long long cap = static_cast<long long>(a.max_blocks) * a.block_size;
    const int keys = static_cast<int>(min(static_cast<long long>(s.past) + (t - s.row0) + 1, cap));
    const float scale = a.scale != 0.f ? a.scale : 1.f / sqrtf(static_cast<float>(H));
#pragma unroll
    for (int r = 0; r < R; ++r) qv[r] = r * 32 + lane < H ? to_float<T>(q[item * H + r * 32 + lane]) : 0.f;
    for (int j = 0; j < keys; ++j) {
      const int block = a.block_table[static_cast<long long>(b) * a.max_blocks + j / a.block_size];
      if (block < 0 || block >= a.num_blocks) {
        if (lane == 0 && a.status) atomicExch(a.status, kStatusBadArgument);
        continue;
      }
      const long long at = ((static_cast<long long>(block) * a.block_size + j % a.block_size) * a.Nk + kvh) * H;
      float dot = 0.f;
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (r * 32 + lane < H) dot += qv[r] * to_float<T>(static_cast<const T*>(a.k_cache)[at + r * 32 + lane]);
      float sc = warp_sum(dot) * scale;
      if (a.softcap > 0.f) sc = a.softcap * tanhf(sc / a.softcap);
      if (sc == -INFINITY) continue;
      const float mm = fmaxf(m, sc), c = m == -INFINITY ? 0.f : expf(m - mm), p = expf(sc - mm);
      l = l * c + p;
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (r * 32 + lane < H) o[r] = o[r] * c + p * to_float<T>(static_cast<const T*>(a.v_cache)[at + r * 32 + lane]);
      m = mm;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (r * 32 + lane < H) out[r * 32 + lane] = from_float<T>(o[r] * inv);
}

// ------------------------------------------------------------------------------------------------------- tensor-core form
// Weights reach the product with V as the sum of two 16-bit values.  Rounded once they would be off by as much as the rounded
// queries are, and the result by 1.7 times the rounding of a 32-bit one instead of 1.4; it costs half a product more, 7 % of the
// time where sequences bring single tokens and 12 % where the tensor pipe is full.
// The reference maximum of a row is raised only when a tile exceeds it by 2^8 (weights stay below 256), so that O is rescaled a few
// times per row.
constexpr float kRaise = 8.f;
constexpr int kQT = 128;          // query rows of a unit
constexpr int kKT = 64;           // keys of a tile
constexpr int kFew = 8;           // units of so few rows go another way through the same tiles
constexpr int kThreads = 192;
constexpr int kGrid = 296;        // two CTAs on each of 148 SMs
constexpr int kTmemCols = 256;    // two score buffers of 64 columns, O in up to 128
constexpr int kPlanInSmem = 768;  // row tiles whose running sums a CTA keeps in shared memory

// What follows from the lengths.
struct Plan {
  long long total;       // length of the numbering
  int prefix_tiles;      // tiles of the prefix
  int prefix_row;        // row of the block table that the prefix is read from
};

struct Work {            // the workspace's parts
  Plan* plan;
  long long* first;      // [row tiles of all sequences + 1]: where the own units of each start, behind the prefix's
  int* tile0;            // [B + 1]: which of those row tiles are a sequence's
  int4* token;           // [T]: the token's sequence, that sequence's first row, rows and past
  uint16_t* q;           // [Nk, T G, H]
  float2* ml;            // per row of a segment: m (in units of log 2) and l
  float* o;              // per row of a segment: H values
};
__host__ __device__ inline long long up256(long long n) { return (n + 255) / 256 * 256; }
// row tiles of all sequences, at most
__host__ __device__ inline long long most_row_tiles(long long T, int B, int N, int Nk) { return T * (N / Nk) / kQT + B; }
__host__ __device__ inline long long plan_bytes(long long T, int B, int N, int Nk) {
  return up256(sizeof(Plan) + 8 * (most_row_tiles(T, B, N, Nk) + 1) + 4ll * (B + 1));
}
__host__ __device__ inline long long segment_rows(long long T, int N) { return 2 * T * N + static_cast<long long>(kGrid) * kQT; }
__host__ __device__ inline Work work_of(const ortb200_prefix_attn_args& a) {
  char* p = static_cast<char*>(a.workspace);
  Work w;
  w.plan = reinterpret_cast<Plan*>(p);
  w.first = reinterpret_cast<long long*>(p + sizeof(Plan));
  w.tile0 = reinterpret_cast<int*>(w.first + most_row_tiles(a.T, a.B, a.N, a.Nk) + 1);
  p += plan_bytes(a.T, a.B, a.N, a.Nk);
  w.token = reinterpret_cast<int4*>(p);
  p += up256(a.T * 16);
  w.q = reinterpret_cast<uint16_t*>(p);
  p += up256(a.T * a.N * a.H * 2);
  w.ml = reinterpret_cast<float2*>(p);
  p += up256(segment_rows(a.T, a.N) * 8);
  w.o = reinterpret_cast<float*>(p);
  return w;
}

// A unit of n tiles takes n + extra(rows) places in the numbering, the tiles behind the others: beginning and ending a segment
// costs a CTA as much time as some tiles, and a share of many short units has to be worth as much as one of a long unit.  For 24
// prompts of up to 150 tokens behind 6000 (28 heads) 1, 2, 3 and 5 places took 303, 257, 234 and 238 us where rows are many; with
// few rows 0, 1 and 2 make 108, 104 and 112 us (180 single tokens behind 20011), 54, 52 and 52 us (64 behind 8192).
__device__ __forceinline__ int extra(int rows) { return rows > 32 ? 4 : 1; }
__device__ __forceinline__ int places(int tiles, int rows) { return tiles > 0 ? tiles + extra(rows) : 0; }
// The share of CTA i of `total` places starts at share(i); place x belongs to CTA owner(x).
__device__ __forceinline__ long long share(long long total, int i) { return total * i / kGrid; }
__device__ __forceinline__ int owner(long long total, long long x) {
  if (total < 0x7fffffffll / kGrid) return static_cast<int>((static_cast<unsigned>(x + 1) * kGrid - 1) / static_cast<unsigned>(total));   // a 64-bit quotient costs five times as much
  return static_cast<int>(((x + 1) * kGrid - 1) / total);
}

// Unit `rt` (rows [128 rt, 128 rt + 128) of the sequence's rows x G) of a sequence: its keys [prefix keys, end) in tiles of 64.
__device__ __forceinline__ int own_end(const ortb200_prefix_attn_args& a, int G, const Span& s, int rt) {
  const int last = min(rt * kQT + kQT, s.rows * G) - 1;
  return static_cast<int>(min(static_cast<long long>(s.past) + last / G + 1, static_cast<long long>(a.max_blocks) * a.block_size));
}
__device__ __forceinline__ int own_tiles(const ortb200_prefix_attn_args& a, int G, const Span& s, int rt, int prefix_tiles) {
  return max((own_end(a, G, s, rt) + kKT - 1) / kKT - prefix_tiles, 0);
}
__device__ __forceinline__ int row_tiles(int G, int rows) { return (rows * G + kQT - 1) / kQT; }
__device__ __forceinline__ int unit_rows(int G, int rows, int rt) { return min(kQT, rows * G - rt * kQT); }
__device__ __forceinline__ int own_places(const ortb200_prefix_attn_args& a, int G, const Span& s, int rt, int prefix_tiles) {
  return places(own_tiles(a, G, s, rt, prefix_tiles), unit_rows(G, s.rows, rt));
}
// all units of the prefix are numbered like the first
__device__ __forceinline__ long long prefix_places(const ortb200_prefix_attn_args& a, int G, int all_rows, int prefix_tiles) {
  return static_cast<long long>(row_tiles(G, all_rows)) * a.Nk * places(prefix_tiles, unit_rows(G, all_rows, 0));
}
// first row that the segments of a unit may use, before 128 rows per CTA number: units follow one another without a gap
__device__ __forceinline__ long long prefix_slot(const ortb200_prefix_attn_args& a, int rt, int kvh, int rows) {
  return static_cast<long long>(rt) * kQT * a.Nk + static_cast<long long>(kvh) * rows;
}
__device__ __forceinline__ long long own_slot(const ortb200_prefix_attn_args& a, int G, int row0, int rt, int kvh, int rows) {
  return a.T * a.N + static_cast<long long>(a.Nk) * (static_cast<long long>(row0) * G + static_cast<long long>(rt) * kQT) + static_cast<long long>(kvh) * rows;
}

// the last of n ascending places that is not behind x
template <typename I>
__device__ __forceinline__ int sequence_with(const I* places, int n, I x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (places[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}
// All THREADS of a CTA: how many tokens all sequences share, and where the own units of each row tile start (`first` and `tile0`,
// written for all to read after the next barrier).
template <int THREADS>
__device__ __forceinline__ Plan make_plan(const ortb200_prefix_attn_args& a, long long* first, int* tile0, int* status) {
  __shared__ int least_sm[THREADS / 32], row_sm[THREADS / 32];
  __shared__ long long sum_sm[THREADS / 32];
  __shared__ int tiles_sm[THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = a.N / a.Nk;
  int least = 0x7fffffff, row = 0x7fffffff, several = 0;
  const int promised = *a.shared_prefix, all_rows = last_row(a);
  for (int b = threadIdx.x; b < a.B; b += THREADS) {
    const Span s = span_of(a, b);
    if (status) check_lengths(a, b, s, status);
    if (s.rows == 0) continue;
    least = min(least, s.past);
    row = min(row, b);
    several |= s.rows * G > kQT;
  }
  least = __reduce_min_sync(0xffffffffu, least);
  row = __reduce_min_sync(0xffffffffu, row);
  if (lane == 0) {
    least_sm[warp] = least;
    row_sm[warp] = row;
  }
  several = __syncthreads_or(several);
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) {
    least = min(least, least_sm[i]);
    row = min(row, row_sm[i]);
  }
  Plan p;
  p.prefix_tiles = least == 0x7fffffff ? 0 : max(min(promised, least), 0) / kKT;
  p.prefix_row = row == 0x7fffffff ? 0 : row;
  // running sums of the threads' values, behind `base`, which then includes them
  auto running = [&](long long n, long long& base, bool again) {
    long long sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    if (again) __syncthreads();
    if (lane == 31) sum_sm[warp] = sum;
    __syncthreads();
    long long before = base;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
      if (i < warp) before += sum_sm[i];
      base += sum_sm[i];
    }
    return before + sum - n;
  };
  if (!several) {   // no sequence has more than one row tile: one pass instead of two (0.5 us of a step of two sequences)
    long long base = 0;
    int tiles = 0;
    for (int b0 = 0; b0 < a.B; b0 += THREADS) {
      const int b = b0 + threadIdx.x;
      const Span s = b < a.B ? span_of(a, b) : Span{0, 0, 0};
      const bool some = s.rows > 0;
      const unsigned with = __ballot_sync(0xffffffffu, some);
      if (b0 > 0) __syncthreads();
      if (lane == 31) tiles_sm[warp] = __popc(with);   // read behind the next barrier, as sum_sm is
      const long long at = running(some ? static_cast<long long>(own_places(a, G, s, 0, p.prefix_tiles)) * a.Nk : 0, base, false);
      int tile = tiles + __popc(with & ((1u << lane) - 1));
#pragma unroll
      for (int i = 0; i < THREADS / 32; ++i) {
        if (i < warp) tile += tiles_sm[i];
        tiles += tiles_sm[i];
      }
      if (b < a.B) tile0[b] = tile;
      if (some) first[tile] = at;
    }
    if (threadIdx.x == 0) {
      tile0[a.B] = tiles;
      first[tiles] = base;
    }
    p.total = base + prefix_places(a, G, all_rows, p.prefix_tiles);
    return p;
  }
  const long long most = most_row_tiles(a.T, a.B, a.N, a.Nk);   // more than these only lengths that overlap have: the rest is left out
  long long tiles = 0, base = 0;
  for (int b0 = 0; b0 < a.B; b0 += THREADS) {
    const int b = b0 + threadIdx.x;
    const long long at = running(b < a.B ? row_tiles(G, span_of(a, b).rows) : 0, tiles, b0 > 0);
    if (b < a.B) tile0[b] = static_cast<int>(min(at, most));
  }
  tiles = min(tiles, most);
  if (threadIdx.x == 0) tile0[a.B] = static_cast<int>(tiles);
  __syncthreads();
  for (int r0 = 0; r0 < tiles; r0 += THREADS) {
    const int r = r0 + threadIdx.x;
    long long n = 0;
    if (r < tiles) {
      const int b = sequence_with(tile0, a.B, r);
      n = static_cast<long long>(own_places(a, G, span_of(a, b), r - tile0[b], p.prefix_tiles)) * a.Nk;
    }
    const long long at = running(n, base, r0 > 0);
    if (r < tiles) first[r] = at;
  }
  if (threadIdx.x == 0) first[tiles] = base;
  p.total = base + prefix_places(a, G, all_rows, p.prefix_tiles);
  return p;
}

// Step 1: one CTA (or, for few tokens, several) per token and one more for the plan.  VEC: whole heads rotated in halves or not
// at all, every address a multiple of 16 bytes: a thread moves 2 x 16 bytes; otherwise one element.
template <typename T, bool VEC>
__global__ void __launch_bounds__(128) prefix_prep_tc_kernel(const ortb200_prefix_attn_args a) {
  const Work w = work_of(a);
  pdl_wait_prior_grids();
  pdl_launch_dependents();   // behind the wait: when step 2 begins, everything in front of this step has ended
  if (blockIdx.x == a.T) {
    if (blockIdx.y != 0) return;
    const Plan p = make_plan<128>(a, w.first, w.tile0, a.status);
    if (threadIdx.x == 0) *w.plan = p;
    return;
  }
  const int t = blockIdx.x, H = a.H, heads = a.N + 2 * a.Nk, G = a.N / a.Nk;
  if (t >= last_row(a)) return;
  const int b = sequence_of(a.cu_seqlens, a.B, t);
  if (blockIdx.y == 0 && threadIdx.x == 0) {
    const Span sp = span_of(a, b);
    w.token[t] = make_int4(b, sp.row0, sp.rows, sp.past);
  }
  if (!owned(a, b, t)) return;   // (its queries stay what the workspace holds; no row's result reaches another's)
  long long slot, pos;
  if (a.positions) {
    pos = a.positions[t];
    slot = a.slot_mapping[t];
  } else {
    pos = static_cast<long long>(a.past_seqlens[b]) + (t - a.cu_seqlens[b]);
    const long long j = pos / a.block_size;
    slot = pos >= 0 && j < a.max_blocks ? static_cast<long long>(a.block_table[static_cast<long long>(b) * a.max_blocks + j]) * a.block_size + pos % a.block_size : -1;
  }
  const bool keep = slot >= 0 && slot < static_cast<long long>(a.num_blocks) * a.block_size;
  if (!keep && threadIdx.x == 0 && a.status) atomicExch(a.status, kStatusBadArgument);
  const int half = a.rot_dim / 2;
  if (a.cos_cache && (pos < 0 || pos >= a.cos_rows)) {   // never past the rotary tables
    if (threadIdx.x == 0 && a.status) atomicExch(a.status, kStatusBadLength);
    pos = pos < 0 ? 0 : a.cos_rows - 1;
  }
  const T* cosr = a.cos_cache ? static_cast<const T*>(a.cos_cache) + pos * half : nullptr;
  const T* sinr = a.cos_cache ? static_cast<const T*>(a.sin_cache) + pos * half : nullptr;
  const int per_block = (heads + gridDim.y - 1) / gridDim.y;
  const int lo = blockIdx.y * per_block, hi = min(heads, lo + per_block), items = VEC ? H / 16 : H;
  for (int idx = lo * items + threadIdx.x; idx < hi * items; idx += 128) {
    const int head = idx / items, d = VEC ? idx % items * 8 : idx % items;
    const int kind = head < a.N ? 0 : head < a.N + a.Nk ? 1 : 2, kh = head - (kind == 1 ? a.N : a.N + a.Nk);
    const T* src;
    if (a.k == nullptr) src = static_cast<const T*>(a.qkv) + (static_cast<long long>(t) * heads + head) * H;
    else if (kind == 0) src = static_cast<const T*>(a.qkv) + (static_cast<long long>(t) * a.N + head) * H;
    else src = static_cast<const T*>(kind == 1 ? a.k : a.v) + (static_cast<long long>(t) * a.Nk + kh) * H;
    T* dst;
    if (kind == 0) {
      dst = reinterpret_cast<T*>(w.q) + ((static_cast<long long>(head / G) * a.T + t) * G + head % G) * H;
    } else {
      if (!keep) continue;
      dst = static_cast<T*>(kind == 1 ? a.k_cache : a.v_cache) + (slot * a.Nk + kh) * H;
    }
    const bool turn = kind < 2 && cosr;
    if (VEC) {
      const int far = H / 2;
      const uint4 u4 = *reinterpret_cast<const uint4*>(src + d), v4 = *reinterpret_cast<const uint4*>(src + d + far);
      if (!turn) {
        *reinterpret_cast<uint4*>(dst + d) = u4;
        *reinterpret_cast<uint4*>(dst + d + far) = v4;
        continue;
      }
      const uint4 c4 = *reinterpret_cast<const uint4*>(cosr + d), s4 = *reinterpret_cast<const uint4*>(sinr + d);
      const T *u = reinterpret_cast<const T*>(&u4), *v = reinterpret_cast<const T*>(&v4), *c = reinterpret_cast<const T*>(&c4), *s = reinterpret_cast<const T*>(&s4);
      __align__(16) T y0[8], y1[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x0 = to_float<T>(u[e]), x1 = to_float<T>(v[e]), cc = to_float<T>(c[e]), ss = to_float<T>(s[e]);
        y0[e] = from_float<T>(x0 * cc - x1 * ss);
        y1[e] = from_float<T>(x1 * cc + x0 * ss);
      }
      *reinterpret_cast<uint4*>(dst + d) = *reinterpret_cast<const uint4*>(y0);
      *reinterpret_cast<uint4*>(dst + d + far) = *reinterpret_cast<const uint4*>(y1);
    } else {
      T y = src[d];
      if (turn && d < a.rot_dim) {
        const int i = a.interleaved ? d >> 1 : d % half;
        const bool upper = a.interleaved ? d & 1 : d >= half;
        const float c = to_float<T>(cosr[i]), s = to_float<T>(sinr[i]), own = to_float<T>(src[d]);
        const float other = to_float<T>(src[a.interleaved ? d ^ 1 : upper ? d - half : d + half]);
        y = from_float<T>(upper ? own * c + other * s : own * c - other * s);
      }
      dst[d] = y;
    }
  }
}

template <int HD>
struct TcSmem {
  static constexpr int kStages = HD == 64 ? 3 : 2;
  static constexpr int kBoxes = HD / 64;                  // boxes of 64 elements per row
  static constexpr int kQBox = kQT * 128, kBox = kKT * 128;
  static constexpr int kStageBytes = 2 * kBoxes * kBox;   // K, then V
  static constexpr int kOffKV = kBoxes * kQBox;
  static constexpr int kOffBar = kOffKV + kStages * kStageBytes;
  static constexpr int kOffFirst = kOffBar + 256;
  static constexpr int kHalf = kQT / 2 * 128;             // the second of two places for queries of up to 64 rows
  static constexpr int kOffTile0 = kOffFirst + 8 * (kPlanInSmem + 1);
  static constexpr int kTotal = kOffTile0 + 4 * (kPlanInSmem + 1) + 1024;
};
enum { BAR_Q = 0, BAR_Q_FREE = BAR_Q + 2, BAR_K_FULL = BAR_Q_FREE + 2, BAR_K_EMPTY = BAR_K_FULL + 3, BAR_V_FULL = BAR_K_EMPTY + 3, BAR_V_EMPTY = BAR_V_FULL + 3, BAR_S = BAR_V_EMPTY + 3,
       BAR_P = BAR_S + 2, BAR_O = BAR_P + 2, BAR_END, BAR_O_FREE, BAR_FEW, BAR_FEW_END = BAR_FEW + 4, BAR_COUNT = BAR_FEW_END + 2 };
static_assert(BAR_COUNT * 8 + 4 <= 256, "barriers do not fit");

// A CTA's share of one unit.
struct Segment {
  int kvh, seq;          // key head; sequence, -1 for the prefix
  int q_row;             // first row of the unit among the T G rows of its key head
  int rows, tiles;       // rows of the unit, tiles of the segment
  int key0, end;         // first key of the segment, end of the unit's keys
  int past, in_seq;      // own units: tokens in front of the sequence's rows, first row of the unit among the sequence's rows x G
  int table_row;
  long long slot;
};
// The segments of a CTA one after the other: its first unit is searched for, the others follow from the one before.
struct Walk {
  const ortb200_prefix_attn_args& a;
  const int* tile0;
  int G, prefix_tiles, prefix_row, all_rows;
  long long left;        // places of the share that are left
  int seq, rt, kvh, at;  // the unit and the place within it
  int tiles, before;     // its tiles and the places in front of them
  Span s;
  Segment unit;          // what all key heads' segments of the unit have in common
  __device__ Walk(const ortb200_prefix_attn_args& args, const long long* first, const int* tiles_of, const Plan& p, int cta)
      : a(args), tile0(tiles_of), G(args.N / args.Nk), prefix_tiles(p.prefix_tiles), prefix_row(p.prefix_row) {
    all_rows = last_row(a);
    const long long prefix_total = prefix_places(a, G, all_rows, prefix_tiles);
    long long x = share(p.total, cta);
    left = share(p.total, cta + 1) - x;
    seq = -1;
    rt = kvh = at = 0;
    if (left == 0) return;
    if (x < prefix_total) {
      prefix_unit();
      const int all = tiles + before;
      const long long u = x / all;
      at = static_cast<int>(x - u * all);
      rt = static_cast<int>(u / a.Nk);
      kvh = static_cast<int>(u - static_cast<long long>(rt) * a.Nk);
      prefix_unit();
    } else {
      x -= prefix_total;
      const int r = sequence_with(first, tile0[a.B], x);
      x -= first[r];
      seq = sequence_with(tile0, a.B, r);
      rt = r - tile0[seq];
      s = span_of(a, seq);
      own_unit();
      kvh = static_cast<int>(x) / (tiles + before);
      at = static_cast<int>(x) - kvh * (tiles + before);
    }
  }
  __device__ void prefix_unit() {
    tiles = prefix_tiles;
    before = extra(unit_rows(G, all_rows, 0));
    unit.seq = -1;
    unit.q_row = rt * kQT;
    unit.rows = unit_rows(G, all_rows, rt);
    unit.key0 = 0;
    unit.end = tiles * kKT;
    unit.past = unit.in_seq = 0;
    unit.table_row = prefix_row;
    unit.slot = prefix_slot(a, rt, 0, unit.rows);
  }
  __device__ void own_unit() {
    tiles = own_tiles(a, G, s, rt, prefix_tiles);
    unit.rows = unit_rows(G, s.rows, rt);
    before = tiles > 0 ? extra(unit.rows) : 0;
    unit.seq = unit.table_row = seq;
    unit.in_seq = rt * kQT;
    unit.q_row = s.row0 * G + unit.in_seq;
    unit.key0 = prefix_tiles * kKT;
    unit.end = own_end(a, G, s, rt);
    unit.past = s.past;
    unit.slot = own_slot(a, G, s.row0, rt, 0, unit.rows);
  }
  __device__ void step() {   // to the next unit that has tiles; there is one while places are left
    at = 0;
    if (++kvh < a.Nk) return;
    kvh = 0;
    ++rt;
    if (seq < 0) {
      if (rt < row_tiles(G, all_rows)) {
        prefix_unit();
        return;
      }
    }
    do {
      if (seq >= 0 && rt < tile0[seq + 1] - tile0[seq]) {
        own_unit();
        if (tiles > 0) return;
        ++rt;
      } else {
        if (++seq >= a.B) {
          left = 0;
          return;
        }
        s = span_of(a, seq);
        rt = 0;
      }
    } while (true);
  }
  __device__ bool next(Segment& g) {
    while (left > 0) {
      if (at == tiles + before) {
        step();
        if (left == 0) break;
      }
      const int upto = static_cast<int>(min(static_cast<long long>(tiles + before), at + left)), t0 = max(at - before, 0);
      left -= upto - at;
      at = upto;
      g.tiles = max(upto - before, 0) - t0;
      if (g.tiles == 0) continue;
      const int n = g.tiles;
      g = unit;
      g.tiles = n;
      g.kvh = kvh;
      g.key0 += t0 * kKT;
      g.slot += static_cast<long long>(kvh) * g.rows;
      return true;
    }
    return false;
  }
};
// Queries of up to 64 rows take one of two places in turn, so that the next segment's arrive while this one's are in use; more
// take both.
struct QueryPlace {
  int place = 0;             // 0 or 1; 0 with `both`
  bool both = false;
  int fills0 = 0, fills1 = 0;   // loads reported on each place's barrier
  int uses0 = 0, uses1 = 0;     // segments that have had each place
  int turn = 0;
  __device__ int fills() const { return place ? fills1 : fills0; }
  __device__ int uses() const { return place ? uses1 : uses0; }
  __device__ void take(int rows) {
    both = rows > kQT / 2;
    place = both ? 0 : turn;
    turn = both ? 0 : turn ^ 1;
  }
  __device__ void done() {
    if (place) {
      ++fills1;
      ++uses1;
    } else {
      ++fills0;
      ++uses0;
      if (both) ++uses1;
    }
  }
};

__device__ __forceinline__ void store8(float* p, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]),
               "f"(v[7])
               : "memory");
}

// What one thread issues per tile decides how fast the tensor pipe turns: descriptors are one word plus an immediate (all operands
// use the 128-byte swizzle, so the upper words agree), and a wait is a loop of its own.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);   // 1024 bytes between groups of eight rows, version, swizzle
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t leading_bytes) { return ((addr & 0x3FFFF) >> 4) | (leading_bytes >> 4 << 16); }
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %4};\n\tmov.b64 b, {%2, %4};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
      ::"r"(d), "r"(a_low), "r"(b_low), "r"(idesc), "n"(kDescHigh), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %4};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b_low), "r"(idesc), "n"(kDescHigh), "r"(accumulate)
      : "memory");
}
// mbar_wait as one loop; false when the limit was reached
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\t"
      "mov.u32 n, %3;\n"
      "AGAIN:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra DONE;\n\t"
      "sub.u32 n, n, 1;\n\t"
      "setp.ne.u32 q, n, 0;\n\t"
      "@q bra AGAIN;\n"
      "DONE:\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity), "n"(ORTB200_SPIN_LIMIT)
      : "memory");
  return done != 0;
}

__device__ __forceinline__ void named_barrier(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait_bar(bar, parity)); }

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <bool BF16>
__device__ __forceinline__ void mma_warp(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float x, float y) {
  if (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Two weights as 16-bit values, and what that leaves of them.
template <bool BF16>
__device__ __forceinline__ void split2(float p0, float p1, uint32_t& high, uint32_t& rest) {
  high = pack16<BF16>(p0, p1);
  if (BF16) {
    const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&high);
    rest = pack16<BF16>(p0 - __low2float(h), p1 - __high2float(h));
  } else {
    const __half2 h = *reinterpret_cast<const __half2*>(&high);
    rest = pack16<BF16>(p0 - __low2float(h), p1 - __high2float(h));
  }
}
// cap tanh(scale x / cap) as an exponent to the base 2.  CAP 1, caps up to 64: c - 2 c / (1 + e^(2 scale x / cap)), off by some 2^-22 of
// the cap, so a weight by 2^-15 at most.  CAP 2, larger ones: tanhf, which is as exact where x is small beside the cap (50 us instead of
// 18.5 for 15 single tokens of 16 heads behind 514 tokens).
template <int CAP>
struct Cap {
  float in, out;
  __device__ Cap(float scale, float cap) : in(CAP == 2 ? scale / cap : 2.f * 1.4426950408889634f * scale / cap), out(cap * 1.4426950408889634f) {}
  __device__ float operator()(float x) const {
    if (CAP == 2) return out * tanhf(x * in);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ex2_approx(x * in)));
    return fmaf(-2.f * out, r, out);
  }
};
__device__ __forceinline__ float max_over_keys(float x) {   // lanes that hold the same row
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ float sum_over_keys(float x) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// A segment of up to eight rows.  In tensor memory they would fill 8 of 128 lanes, and a tile would still take the whole chain of
// S, softmax and O with its hand-overs; so each of the four warps multiplies a quarter of a tile's keys itself, keys and dims as
// the 16 rows of a product and the queries as its 8 columns: S^T = K Q^T, O^T += V^T P^T.  A warp has its own running maximum and
// sums; they meet once per segment, in the place of the queries.
template <int HD, bool BF16, int CAP>
__device__ __forceinline__ void few_rows(const ortb200_prefix_attn_args& a, const Work& w, const Segment& g, uint8_t* smem, uint64_t* bars, float2 (*part)[kFew],
                                         const QueryPlace& qp, float scale, int qw, int lane, int& stage, uint32_t& parity, int& few_tiles, int few_segments, bool& ok) {
  using L = TcSmem<HD>;
  const int G = a.N / a.Nk, n0 = (lane & 3) * 2;
  float fs = scale * 1.4426950408889634f;
  const Cap<CAP> cap(scale, a.softcap);
  if (CAP) fs = 1.f;
  const int seen0 = g.seq < 0 ? g.end : min(g.end, g.past + (g.in_seq + n0) / G + 1), seen1 = g.seq < 0 ? g.end : min(g.end, g.past + (g.in_seq + n0 + 1) / G + 1);
  if (ok && !wait_warp(&bars[BAR_Q + qp.place], qp.fills() & 1)) ok = false;
  uint32_t q[HD / 16][2];
  const uint32_t q_row = smem_u32(smem + qp.place * L::kHalf) + (lane & 7) * 128;
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) {
    const int chunk = 4 * i + (lane >> 3);
    ldmatrix4(q_row + (chunk >> 3) * L::kQBox + (((chunk & 7) ^ (lane & 7)) << 4), q[2 * i][0], q[2 * i][1], q[2 * i + 1][0], q[2 * i + 1][1]);
  }
  // (the rows of a warp's matrices start at a multiple of eight, so that the swizzle's row is the lane's)
  const uint32_t kv0 = smem_u32(smem + L::kOffKV), k_row = kv0 + (qw * 16 + (lane & 15)) * 128;
  const uint32_t v_row = kv0 + L::kBoxes * L::kBox + (qw * 16 + (lane & 7) + ((lane >> 4) << 3)) * 128;
  float o[HD / 16][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
  for (int d = 0; d < HD / 16; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
  for (int t = 0; t < g.tiles; ++t) {
    const int first = g.key0 + t * kKT + qw * 16, key = first + (lane >> 2);
    if (first < g.end) {
      if (ok && !wait_warp(&bars[BAR_K_FULL + stage], parity)) ok = false;
      float c[4] = {0.f, 0.f, 0.f, 0.f}, e[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        const int chunk = 2 * kk + (lane >> 4);
        uint32_t k[4];
        ldmatrix4(k_row + stage * L::kStageBytes + (kk / 4) * L::kBox + (((chunk & 7) ^ (lane & 7)) << 4), k[0], k[1], k[2], k[3]);
        mma_warp<BF16>(kk & 1 ? e : c, k, q[kk][0], q[kk][1]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[i] += e[i];
        if (CAP) c[i] = cap(c[i]);
      }
      if (key >= seen0) c[0] = -INFINITY;
      if (key >= seen1) c[1] = -INFINITY;
      if (key + 8 >= seen0) c[2] = -INFINITY;
      if (key + 8 >= seen1) c[3] = -INFINITY;
      float t0 = fmaxf(c[0], c[2]) * fs, t1 = fmaxf(c[1], c[3]) * fs;
      if (__any_sync(0xffffffffu, t0 > m0 + kRaise || t1 > m1 + kRaise)) {
        t0 = max_over_keys(t0);
        t1 = max_over_keys(t1);
        const bool raise0 = t0 > m0 + kRaise, raise1 = t1 > m1 + kRaise;
        const float corr0 = raise0 ? (m0 == -INFINITY ? 0.f : ex2_approx(m0 - t0)) : 1.f, corr1 = raise1 ? (m1 == -INFINITY ? 0.f : ex2_approx(m1 - t1)) : 1.f;
        if (raise0) m0 = t0;
        if (raise1) m1 = t1;
        l0 *= corr0;
        l1 *= corr1;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) {
          o[d][0] *= corr0;
          o[d][1] *= corr1;
          o[d][2] *= corr0;
          o[d][3] *= corr1;
        }
      }
      const float neg0 = m0 == -INFINITY ? 0.f : -m0, neg1 = m1 == -INFINITY ? 0.f : -m1;
      const float p00 = ex2_approx(fmaf(c[0], fs, neg0)), p01 = ex2_approx(fmaf(c[1], fs, neg1));
      const float p80 = ex2_approx(fmaf(c[2], fs, neg0)), p81 = ex2_approx(fmaf(c[3], fs, neg1));
      l0 += p00 + p80;
      l1 += p01 + p81;
      uint32_t h0, h1, r0, r1;
      split2<BF16>(p00, p01, h0, r0);
      split2<BF16>(p80, p81, h1, r1);
      h0 = transpose8(h0);
      h1 = transpose8(h1);
      r0 = transpose8(r0);
      r1 = transpose8(r1);
      if (ok && !wait_warp(&bars[BAR_V_FULL + stage], parity)) ok = false;
      const int live = g.end - first;
      if (live < 16) {   // what lies behind the last key may be anything, and 0 * NaN would reach the product: these rows of V become 0
        uint8_t* v = smem + L::kOffKV + stage * L::kStageBytes + L::kBoxes * L::kBox + (qw * 16 + live) * 128;
        for (int i = lane; i < (16 - live) * 8; i += 32)
#pragma unroll
          for (int bx = 0; bx < L::kBoxes; ++bx) *reinterpret_cast<uint4*>(v + bx * L::kBox + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async();
        __syncwarp();
      }
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) {
        const int chunk = 2 * d + ((lane >> 3) & 1);
        uint32_t v[4];
        ldmatrix4_trans(v_row + stage * L::kStageBytes + (d / 4) * L::kBox + (((chunk & 7) ^ (lane & 7)) << 4), v[0], v[1], v[2], v[3]);
        mma_warp<BF16>(o[d], v, h0, h1);
        mma_warp<BF16>(o[d], v, r0, r1);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars[BAR_FEW + (few_tiles & 3)]);
    ++few_tiles;
    if (++stage == L::kStages) {
      stage = 0;
      parity ^= 1u;
    }
  }
  l0 = sum_over_keys(l0);
  l1 = sum_over_keys(l1);
  named_barrier(1, 128);   // all have read the queries, and the sums of the segment before
  if (lane < 4) {
    part[qw][n0] = make_float2(m0, l0);
    part[qw][n0 + 1] = make_float2(m1, l1);
  }
  // [box of 64 dims][warp][row][dim], the dims in groups of eight exchanged by row so that the stores meet different banks
  auto sums = [&](int warp, int row, int dim) {
    return reinterpret_cast<float*>(smem + qp.place * L::kHalf + (dim >> 6) * L::kQBox) + (warp * kFew + row) * 64 + ((dim & 63) ^ ((row >> 1) << 3));
  };
#pragma unroll
  for (int d = 0; d < HD / 16; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) *sums(qw, n0 + (i & 1), d * 16 + (lane >> 2) + (i >> 1) * 8) = o[d][i];
  named_barrier(1, 128);
  constexpr int E = HD / 16;
  const int n = (qw * 32 + lane) >> 4, d0 = (lane & 15) * E;
  if (n < g.rows && ok) {
    float m = -INFINITY, l = 0.f, v[E];
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, part[i][n].x);
#pragma unroll
    for (int x = 0; x < E; ++x) v[x] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 ml = part[i][n];
      const float f = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - m);
      l += ml.x == -INFINITY ? ml.y : ml.y * f;   // (a sum without a maximum is 0 or NaN)
      const float* from = sums(i, n, d0);
#pragma unroll
      for (int x = 0; x < E; x += 4) {
        const float4 y = *reinterpret_cast<const float4*>(from + x);
        v[x] += f * y.x;
        v[x + 1] += f * y.y;
        v[x + 2] += f * y.z;
        v[x + 3] += f * y.w;
      }
    }
    const long long row = g.slot + static_cast<long long>(blockIdx.x) * kQT + n;
    if ((lane & 15) == 0) w.ml[row] = make_float2(m, l);
#pragma unroll
    for (int x = 0; x < E; x += 4) *reinterpret_cast<float4*>(w.o + row * HD + d0 + x) = make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]);
  }
  fence_proxy_async();   // the next queries arrive where the sums were
  __syncwarp();
  if (lane == 0) mbar_arrive(&bars[BAR_FEW_END + (few_segments & 1)]);
}

template <int HD, bool BF16, int CAP>
__global__ void __launch_bounds__(kThreads, 2)
prefix_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                   const ortb200_prefix_attn_args a, const float scale) {
  using L = TcSmem<HD>;
  constexpr int STAGES = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + BAR_COUNT);
  long long* first_sm = reinterpret_cast<long long*>(smem + L::kOffFirst);
  int* tile0_sm = reinterpret_cast<int*>(smem + L::kOffTile0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ float2 part[4][kFew];

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    for (int i = 0; i < BAR_COUNT; ++i) mbar_init(&bars[i], i == BAR_P || i == BAR_P + 1 || i >= BAR_O_FREE ? 4 : 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  // Step 1 has begun when this step begins, and what came before has ended: lengths, table and old cache entries may be read at
  // once.  Only the loading warp waits for step 1, in front of the first query or new key that it fetches.
  const Work w = work_of(a);
  Plan plan;
  const bool kept = most_row_tiles(a.T, a.B, a.N, a.Nk) <= kPlanInSmem;
  if (kept) {
    plan = make_plan<kThreads>(a, first_sm, tile0_sm, nullptr);
  } else {
    pdl_wait_prior_grids();
    plan = *w.plan;
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_s = __reduce_or_sync(0xffffffffu, *tmem_slot);   // S / P: two buffers of 64 columns; the same for all, and known to be
  const uint32_t tmem_o = tmem_s + 2 * kKT;

  Walk walk(a, kept ? first_sm : w.first, kept ? tile0_sm : w.tile0, plan, blockIdx.x);
  Segment g;
  bool ok = true;

  if (warp == 0) {
    // ---------------------------------------------------------------------------------------------------- loads
    const int piece = min(a.block_size, kKT), pieces = kKT / piece;   // rows that one block gives a tile
    int s = 0, k_tiles = 0, v_tiles = 0;
    uint32_t parity = 1;   // the first round over the stages waits for nothing
    QueryPlace qp;
    bool waited = !kept, outside = false;
    auto wait_step1 = [&]() {
      if (waited) return;
      pdl_wait_prior_grids();
      pdl_launch_dependents();
      waited = true;
    };
    if (!kept) pdl_launch_dependents();
    while (ok && walk.next(g)) {
      const int* table = a.block_table + static_cast<long long>(g.table_row) * a.max_blocks;
      qp.take(g.rows);
      // queries of the segment; the first one's are asked for behind the first tiles, which need not wait for step 1
      auto load_q = [&]() {
        if (qp.uses() > 0 && !wait_warp(&bars[BAR_Q_FREE + qp.place], (qp.uses() - 1) & 1)) return false;
        if (qp.both && qp.uses1 > 0 && !wait_warp(&bars[BAR_Q_FREE + 1], (qp.uses1 - 1) & 1)) return false;
        wait_step1();
        const int boxes = (g.rows + 15) / 16;
        if (lane == 0) mbar_expect_tx(&bars[BAR_Q + qp.place], L::kBoxes * boxes * 2048);
        __syncwarp();
        if (lane < boxes)
          for (int bx = 0; bx < L::kBoxes; ++bx)
            tma_load_3d(smem + bx * L::kQBox + qp.place * L::kHalf + lane * 2048, &tm_q, &bars[BAR_Q + qp.place], bx * 64, g.q_row + lane * 16, g.kvh);
        qp.done();
        return true;
      };
      bool q_asked = false;
      // behind the unit's last key the table may hold anything; in front of it a block outside the cache is reported
      auto block_at = [&](int key) {
        const int named = table[min(key / a.block_size, a.max_blocks - 1)], block = min(max(named, 0), a.num_blocks - 1);
        outside |= named != block && key < g.end;
        return block;
      };
      int block = lane < pieces ? block_at(g.key0 + lane * piece) : 0;
      for (int t = 0; t < g.tiles; ++t) {
        const int key = g.key0 + t * kKT + lane * piece, in_block = key % a.block_size;
        uint8_t* st = smem + L::kOffKV + s * L::kStageBytes + lane * piece * 128;
        const bool fresh = g.seq >= 0 && g.key0 + (t + 1) * kKT > g.past;   // the tile has keys of this call
        if (!q_asked && (waited || fresh || t == STAGES)) {
          if (!load_q()) { ok = false; break; }
          q_asked = true;
        }
        if (!wait_warp(&bars[BAR_K_EMPTY + s], parity)) { ok = false; break; }
        if (lane == 0) mbar_expect_tx(&bars[BAR_K_FULL + s], L::kBoxes * L::kBox);
        __syncwarp();
        ++k_tiles;
        if (lane < pieces)
          for (int bx = 0; bx < L::kBoxes; ++bx) tma_load_4d(st + bx * L::kBox, &tm_k, &bars[BAR_K_FULL + s], bx * 64, in_block, g.kvh, block);
        if (!wait_warp(&bars[BAR_V_EMPTY + s], parity)) { ok = false; break; }
        if (lane == 0) mbar_expect_tx(&bars[BAR_V_FULL + s], L::kBoxes * L::kBox);
        __syncwarp();
        ++v_tiles;
        if (lane < pieces)
          for (int bx = 0; bx < L::kBoxes; ++bx) tma_load_4d(st + (L::kBoxes + bx) * L::kBox, &tm_v, &bars[BAR_V_FULL + s], bx * 64, in_block, g.kvh, block);
        if (t + 1 < g.tiles && lane < pieces) block = block_at(key + kKT);
        if (++s == STAGES) { s = 0; parity ^= 1u; }
      }
      if (ok && !q_asked && !load_q()) ok = false;
    }
    wait_step1();
    // whoever gave up: no copy may be on its way when the CTA ends
    if (qp.fills0 > 0 && !wait_warp(&bars[BAR_Q], (qp.fills0 - 1) & 1)) ok = false;
    if (qp.fills1 > 0 && !wait_warp(&bars[BAR_Q + 1], (qp.fills1 - 1) & 1)) ok = false;
    for (int i = 0; i < STAGES; ++i) {
      const int k = (k_tiles - i + STAGES - 1) / STAGES, v = (v_tiles - i + STAGES - 1) / STAGES;   // loads into stage i
      if (k > 0 && !wait_warp(&bars[BAR_K_FULL + i], (k - 1) & 1)) ok = false;
      if (v > 0 && !wait_warp(&bars[BAR_V_FULL + i], (v - 1) & 1)) ok = false;
    }
    if (outside && a.status) atomicExch(a.status, kStatusBadArgument);
    if (!ok && lane == 0 && a.status) atomicExch(a.status, kStatusTimeoutProducer);
  } else if (warp == 1) {
    // ------------------------------------------------------------------------------------------------- products
    if (elect_one()) {
      constexpr uint32_t idesc_s = umma_idesc_f16(BF16, kQT, kKT), idesc_o = umma_idesc_f16_bmn(BF16, kQT, HD);
      const uint32_t kv_low = desc_low(smem_u32(smem + L::kOffKV), 16), v_low = desc_low(smem_u32(smem + L::kOffKV + L::kBoxes * L::kBox), L::kBox);
      int s = 0, seg = 0, it = 0;   // stage, segment and tile of this CTA
      uint32_t parity = 0;
      QueryPlace qp;
      auto issue_s = [&](int tile, int stage, bool last) {
        const uint32_t q_low = desc_low(smem_u32(smem + qp.place * L::kHalf), 16), k_low = kv_low + stage * (L::kStageBytes >> 4), d = tmem_s + (tile & 1) * kKT;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          mma_ss(d, q_low + (kk / 4) * (L::kQBox >> 4) + (kk % 4) * 2, k_low + (kk / 4) * (L::kBox >> 4) + (kk % 4) * 2, idesc_s, kk > 0 ? 1u : 0u);
        umma_commit(&bars[BAR_S + (tile & 1)]);
        umma_commit(&bars[BAR_K_EMPTY + stage]);
        if (last) {
          umma_commit(&bars[BAR_Q_FREE + qp.place]);
          if (qp.both) umma_commit(&bars[BAR_Q_FREE + 1]);
        }
      };
      int few_tiles = 0, few_segments = 0;
      while (ok && walk.next(g)) {
        if (g.rows <= kFew) {   // the other warps do these; what they have read goes back in the order of the tiles
          qp.take(g.rows);
          for (int t = 0; t < g.tiles; ++t, ++few_tiles) {
            if (!wait_bar(&bars[BAR_FEW + (few_tiles & 3)], (few_tiles >> 2) & 1)) { ok = false; break; }
            mbar_arrive(&bars[BAR_K_EMPTY + s]);
            mbar_arrive(&bars[BAR_V_EMPTY + s]);
            if (++s == STAGES) {
              s = 0;
              parity ^= 1u;
            }
          }
          if (ok && !wait_bar(&bars[BAR_FEW_END + (few_segments & 1)], (few_segments >> 1) & 1)) ok = false;
          mbar_arrive(&bars[BAR_Q_FREE + qp.place]);
          ++few_segments;
          qp.done();
          continue;
        }
        // scores go over the weights of two tiles before; the products that read those are behind the last tile's, which are over
        if (it > 0 && !wait_bar(&bars[BAR_O], (it - 1) & 1)) { ok = false; break; }
        qp.take(g.rows);
        if (!wait_bar(&bars[BAR_Q + qp.place], qp.fills() & 1) || !wait_bar(&bars[BAR_K_FULL + s], parity)) { ok = false; break; }
        tcgen05_fence_after();
        issue_s(it, s, g.tiles == 1);
        for (int t = 0; t < g.tiles; ++t, ++it) {
          const int s1 = s + 1 == STAGES ? 0 : s + 1;
          const uint32_t parity1 = s1 == 0 ? parity ^ 1u : parity;
          if (t + 1 < g.tiles) {
            if (it > 0 && !wait_bar(&bars[BAR_O], (it - 1) & 1)) { ok = false; break; }
            if (!wait_bar(&bars[BAR_K_FULL + s1], parity1)) { ok = false; break; }
            tcgen05_fence_after();
            issue_s(it + 1, s1, t + 2 == g.tiles);
          }
          if (!wait_bar(&bars[BAR_V_FULL + s], parity) || !wait_bar(&bars[BAR_P + (it & 1)], (it >> 1) & 1)) { ok = false; break; }
          if (t == 0 && seg > 0 && !wait_bar(&bars[BAR_O_FREE], (seg - 1) & 1)) { ok = false; break; }
          tcgen05_fence_after();
          const uint32_t low = v_low + s * (L::kStageBytes >> 4), p = tmem_s + (it & 1) * kKT;
#pragma unroll
          for (int kk = 0; kk < kKT / 16; ++kk) mma_ts(tmem_o, p + kk * 8, low + kk * (2048 >> 4), idesc_o, t > 0 || kk > 0 ? 1u : 0u);
#pragma unroll
          for (int kk = 0; kk < kKT / 16; ++kk) mma_ts(tmem_o, p + kKT / 2 + kk * 8, low + kk * (2048 >> 4), idesc_o, 1u);
          umma_commit(&bars[BAR_O]);
          umma_commit(&bars[BAR_V_EMPTY + s]);
          if (t == g.tiles - 1) umma_commit(&bars[BAR_END]);
          s = s1;
          parity = parity1;
        }
        qp.done();
        ++seg;
      }
      if (!ok && a.status) atomicExch(a.status, kStatusTimeoutMma);
    }
    __syncwarp();
  } else {
    // --------------------------------------------------------------------------------- softmax, one thread per row
    const int qw = warp & 3, r = qw * 32 + lane, G = a.N / a.Nk;
    const uint32_t lane_addr = static_cast<uint32_t>(qw * 32) << 16;
    const float scale_log2 = scale * 1.4426950408889634f;
    int seg = 0, it = 0, few_tiles = 0, few_segments = 0, stage = 0;
    uint32_t parity = 0;
    QueryPlace qp;
    while (walk.next(g)) {   // to the end even when a wait gave up: the four warps meet at barriers
      qp.take(g.rows);
      if (g.rows <= kFew) {
        few_rows<HD, BF16, CAP>(a, w, g, smem, bars, part, qp, scale, qw, lane, stage, parity, few_tiles, few_segments, ok);
        ++few_segments;
        qp.done();
        continue;
      }
      qp.done();
      const bool idle = qw * 32 >= g.rows;   // a warp without rows keeps the barriers going
      const int pos = g.seq < 0 ? 0x7fffffff : g.past + (g.in_seq + r) / G;
      const int first_pos = g.seq < 0 ? 0x7fffffff : g.past + g.in_seq / G;
      float m = -INFINITY, l = 0.f;
      for (int t = 0; t < g.tiles; ++t, ++it) {
        const int key0 = g.key0 + t * kKT;
        if (ok && !wait_warp(&bars[BAR_S + (it & 1)], (it >> 1) & 1)) ok = false;
        tcgen05_fence_after();
        if (!idle) {
          const uint32_t s_addr = tmem_s + (it & 1) * kKT + lane_addr;
          float sv[kKT];
          tmem_ld_x32(s_addr, sv);
          tmem_ld_x32(s_addr + 32, sv + 32);
          tmem_ld_wait();
          float fs = scale_log2;   // scores stay unscaled: the scale is part of the exponent's multiply-add; a cap leaves base-2 exponents
          if (CAP) {
            fs = 1.f;
            const Cap<CAP> cap(scale, a.softcap);
#pragma unroll
            for (int j = 0; j < kKT; ++j) sv[j] = cap(sv[j]);
          }
          if (key0 + kKT > g.end || key0 + kKT - 1 > first_pos) {
            const int hi = min(g.end - key0, pos - key0 + 1);   // keys of this tile that the row sees
#pragma unroll
            for (int j = 0; j < kKT; ++j) sv[j] = j < hi ? sv[j] : -INFINITY;
          }
          float m_raw = -INFINITY;
#pragma unroll
          for (int j = 0; j < kKT; j += 2) m_raw = fmax3(m_raw, sv[j], sv[j + 1]);
          const float m_tile = m_raw * fs;
          const bool raise = m_tile > m + kRaise;   // also the first finite maximum of a row
          if (__any_sync(0xffffffffu, raise)) {
            const float corr = raise ? (m == -INFINITY ? 0.f : ex2_approx(m - m_tile)) : 1.f;
            if (t > 0) {
              if (ok && !wait_warp(&bars[BAR_O], (it - 1) & 1)) ok = false;
              tcgen05_fence_after();
#pragma unroll 1
              for (int c = 0; c < HD; c += 32) {
                float v[32];
                tmem_ld_x32(tmem_o + lane_addr + c, v);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] *= corr;
                tmem_st_x32(tmem_o + lane_addr + c, v);
              }
            }
            l *= corr;
            if (raise) m = m_tile;
          }
          const float neg_m = m == -INFINITY ? 0.f : -m;
          f32x2 sum = pack2(0.f, 0.f);
          const f32x2 fs2 = pack2(fs, fs), neg2 = pack2(neg_m, neg_m), one = pack2(1.f, 1.f), minus = pack2(-1.f, -1.f);
#pragma unroll
          for (int c = 0; c < kKT; c += 32) {
            uint32_t packed[16], rest[16];
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              float p0, p1, h0, h1;
              unpack2(fma2(pack2(sv[c + j], sv[c + j + 1]), fs2, neg2), p0, p1);
              const f32x2 p = pack2(ex2_approx(p0), ex2_approx(p1));
              sum = fma2(p, one, sum);
              unpack2(p, p0, p1);
              if (BF16) {   // the upper halves of the two, not rounded, and what is left
                h0 = __uint_as_float(__float_as_uint(p0) & 0xffff0000u);
                h1 = __uint_as_float(__float_as_uint(p1) & 0xffff0000u);
                packed[j / 2] = __byte_perm(__float_as_uint(p0), __float_as_uint(p1), 0x7632);
              } else {
                const __half2 h = __floats2half2_rn(p0, p1);
                packed[j / 2] = *reinterpret_cast<const uint32_t*>(&h);
                h0 = __low2float(h);
                h1 = __high2float(h);
              }
              float d0, d1;
              unpack2(fma2(pack2(h0, h1), minus, p), d0, d1);
              rest[j / 2] = pack16<BF16>(d0, d1);
            }
            tmem_st_x16_u32(s_addr + c / 2, packed);
            tmem_st_x16_u32(s_addr + kKT / 2 + c / 2, rest);
          }
          float sum0, sum1;
          unpack2(sum, sum0, sum1);
          l += sum0 + sum1;
          tmem_st_wait();
        }
        const int live = g.end - key0;
        if (live < kKT && ok) {
          // what lies behind the last key may be anything, and 0 * NaN would reach the product: these rows of V become 0
          if (!wait_warp(&bars[BAR_V_FULL + stage], parity)) ok = false;
          uint8_t* v = smem + L::kOffKV + stage * L::kStageBytes + L::kBoxes * L::kBox + live * 128;
          for (int i = r; i < (kKT - live) * 8; i += 128)
#pragma unroll
            for (int bx = 0; bx < L::kBoxes; ++bx) *reinterpret_cast<uint4*>(v + bx * L::kBox + i * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async();
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[BAR_P + (it & 1)]);
        if (++stage == STAGES) {
          stage = 0;
          parity ^= 1u;
        }
      }
      if (ok && !wait_warp(&bars[BAR_END], seg & 1)) ok = false;
      tcgen05_fence_after();
      if (!idle) {
        const long long row = g.slot + static_cast<long long>(blockIdx.x) * kQT + r;
        const bool mine = ok && r < g.rows;
        if (mine) w.ml[row] = make_float2(m, l);
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          float v[32];
          tmem_ld_x32(tmem_o + lane_addr + c, v);
          tmem_ld_wait();
          if (mine)
#pragma unroll
            for (int j = 0; j < 32; j += 8) store8(w.o + row * HD + c + j, v + j);
        }
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[BAR_O_FREE]);
      ++seg;
    }
    if (!ok && lane == 0 && a.status) atomicExch(a.status, kStatusTimeoutEpilogue);
  }

  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc(tmem_s, kTmemCols);
  }
}

template <int E>
__device__ __forceinline__ void load_cg(const float* p, float* v) {
  if (E == 4) {
    const float4 x = __ldcg(reinterpret_cast<const float4*>(p));
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  } else {
    const float2 x = __ldcg(reinterpret_cast<const float2*>(p));
    v[0] = x.x; v[1] = x.y;
  }
}
// Step 3: a warp joins `per` neighbouring rows of a key head (32 at most).  Each lane looks one row's sequence up; where the
// segments of a unit are is worked out once for all of its rows.  SPLIT: few rows, whose segments may be hundreds; the four warps of
// a CTA share one row's.
template <typename T, int HD, bool SPLIT>
__global__ void __launch_bounds__(128) prefix_join_kernel(const ortb200_prefix_attn_args a, const int per) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31, G = a.N / a.Nk, all_rows = last_row(a);
  const int warp = threadIdx.x >> 5;
  __shared__ float part_o[SPLIT ? 4 : 1][HD];
  __shared__ float2 part_ml[4];
  const unsigned item = SPLIT ? blockIdx.x : blockIdx.x * 4 + warp, rows = static_cast<unsigned>(a.T) * G;
  const int kvh = static_cast<int>(item % a.Nk);
  const unsigned row0 = item / a.Nk * per;
  if (row0 >= rows) return;
  const int count = static_cast<int>(min(rows - row0, static_cast<unsigned>(per)));
  const Work w = work_of(a);
  // (step 1 has ended when this step begins: only the segments are waited for)
  const Plan plan = {__ldcg(&w.plan->total), __ldcg(&w.plan->prefix_tiles), 0};
  const int my_t = static_cast<int>((row0 + min(lane, count - 1)) / G);
  const int4 my_tok = __ldcg(&w.token[my_t]);
  const bool my_live = my_t < all_rows && my_t >= my_tok.y && my_t < my_tok.y + my_tok.z && plan.total > 0;   // lengths that start behind 0 leave rows to nobody
  // where the own units of the row's row tile start
  const int my_ort = my_live ? (static_cast<int>(row0) + min(lane, count - 1) - my_tok.y * G) / kQT : 0, my_tile = my_live ? __ldcg(&w.tile0[my_tok.x]) + my_ort : 0;
  const bool counted = my_live && my_tile < __ldcg(&w.tile0[my_tok.x + 1]);
  const long long my_start = counted ? prefix_places(a, G, all_rows, plan.prefix_tiles) + __ldcg(&w.first[my_tile]) : 0;
  // the units of a row, 0 of the prefix and 1 of its own keys: first tile in the numbering, tiles, first slot
  int prt = -1, ort = -1, seq = -1, tiles0 = 0, tiles1 = 0, first0 = 0, first1 = 0, count0 = 0, count1 = 0;
  long long from0 = 0, from1 = 0, slot0 = 0, slot1 = 0, start = 0;
  // segment k of the row, over both units: CTA first0 + k of the one or first1 + k - count0 of the other
  bool has = false, own = false;
  long long base = 0;
  auto segment = [&](int k) {
    own = k >= count0;
    const int i = own ? first1 + k - count0 : first0 + k;
    const long long from = own ? from1 : from0;
    has = k < count0 + count1 && max(from, share(plan.total, i)) < min(from + (own ? tiles1 : tiles0), share(plan.total, i + 1));
    base = (own ? slot1 : slot0) + static_cast<long long>(i) * kQT;
  };
  // rows of up to four segments, the usual ones: their places, the same in all lanes
  constexpr int kShort = 4;
  int n = 0, places4[kShort] = {0, 0, 0, 0};
  int t = -1;
  bool live = false;
  int4 tok = {0, 0, 0, 0};
  for (int r = 0; r < count; ++r) {
    const int pr = static_cast<int>(row0) + r;
    if (r == 0 || pr == (t + 1) * G) {
      t = __shfl_sync(0xffffffffu, my_t, r);
      live = __shfl_sync(0xffffffffu, counted, r);
      tok = {__shfl_sync(0xffffffffu, my_tok.x, r), __shfl_sync(0xffffffffu, my_tok.y, r), __shfl_sync(0xffffffffu, my_tok.z, r), __shfl_sync(0xffffffffu, my_tok.w, r)};
    }
    const int orow = pr - tok.y * G;
    if (!live) {
      count0 = count1 = n = 0;
      prt = -1;
    } else if (pr / kQT != prt || tok.x != seq || orow / kQT != ort) {
      const Span s = {tok.y, tok.z, tok.w};
      prt = pr / kQT;
      tiles0 = plan.prefix_tiles;
      const int before0 = extra(unit_rows(G, all_rows, 0));
      from0 = (static_cast<long long>(prt) * a.Nk + kvh) * (tiles0 + before0) + before0;
      slot0 = prefix_slot(a, prt, kvh, unit_rows(G, all_rows, prt));
      seq = tok.x;
      ort = orow / kQT;
      start = __shfl_sync(0xffffffffu, my_start, r);
      tiles1 = own_tiles(a, G, s, ort, tiles0);
      const int rows1 = unit_rows(G, s.rows, ort);
      from1 = start + static_cast<long long>(kvh) * places(tiles1, rows1) + extra(rows1);
      slot1 = own_slot(a, G, s.row0, ort, kvh, rows1);
      first0 = tiles0 > 0 ? owner(plan.total, from0) : 0;
      first1 = tiles1 > 0 ? owner(plan.total, from1) : 0;
      count0 = tiles0 > 0 ? owner(plan.total, from0 + tiles0 - 1) - first0 + 1 : 0;
      count1 = tiles1 > 0 ? owner(plan.total, from1 + tiles1 - 1) - first1 + 1 : 0;
      segment(lane);
      unsigned left = __ballot_sync(0xffffffffu, has);
      n = count0 + count1 > 32 ? kShort + 1 : __popc(left);
#pragma unroll
      for (int i = 0; i < kShort; ++i) {
        const int from = max(__ffs(left) - 1, 0);
        places4[i] = static_cast<int>(__shfl_sync(0xffffffffu, base, from)) * 2 + (from >= count0);
        left &= left - 1;
      }
    }
    if (r == 0) pdl_wait_prior_grids();
    float o[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    if (n <= kShort) {
      float2 ml[kShort];
      float v[kShort][E];
#pragma unroll
      for (int i = 0; i < kShort; ++i) {
        ml[i] = make_float2(-INFINITY, 0.f);
        if (i < n) {
          const unsigned row = (places4[i] >> 1) + static_cast<unsigned>(places4[i] & 1 ? orow : pr) % kQT;
          ml[i] = __ldcg(&w.ml[row]);
          load_cg<E>(w.o + static_cast<unsigned long long>(row) * HD + lane * E, v[i]);
        }
      }
      m = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
#pragma unroll
      for (int i = 0; i < kShort; ++i)
        if (i < n) {
          const float f = ml[i].x == -INFINITY ? 0.f : exp2f(ml[i].x - m);
          l += ml[i].x == -INFINITY ? ml[i].y : ml[i].y * f;   // a row whose scores are all NaN has no maximum; its sum carries the NaN on
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] += f * v[i][e];
        }
    }
    for (int k0 = SPLIT ? warp * 32 : 0; n > kShort && k0 < count0 + count1; k0 += SPLIT ? 128 : 32) {
      segment(k0 + lane);
      const long long row = base + (own ? orow : pr) % kQT;
      const float2 ml = has ? __ldcg(&w.ml[row]) : make_float2(-INFINITY, 0.f);
      unsigned left = __ballot_sync(0xffffffffu, has);
      const float mm = fmaxf(m, warp_max(ml.x));
      const float keep = m == -INFINITY ? 0.f : exp2f(m - mm), mine = ml.x == -INFINITY ? 0.f : exp2f(ml.x - mm);
      l = l * keep + warp_sum(ml.x == -INFINITY ? ml.y : ml.y * mine);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] *= keep;
      m = mm;
      while (left != 0) {   // R segments' values on their way at a time
        constexpr int R = 8;
        float v[R][E], f[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const bool some = left != 0;
          const int at = some ? __ffs(left) - 1 : 0;
          left &= left - 1;
          const long long from = __shfl_sync(0xffffffffu, row, at);
          f[i] = __shfl_sync(0xffffffffu, mine, at);
          if (some) {
            load_cg<E>(w.o + from * HD + lane * E, v[i]);
          } else {
            f[i] = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) v[i][e] = 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] += f[i] * v[i][e];
      }
    }
    if (SPLIT) {
      if (n > kShort) {
#pragma unroll
        for (int e = 0; e < E; ++e) part_o[warp][lane * E + e] = o[e];
        if (lane == 0) part_ml[warp] = make_float2(m, l);
        __syncthreads();
        m = fmaxf(fmaxf(part_ml[0].x, part_ml[1].x), fmaxf(part_ml[2].x, part_ml[3].x));
        l = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 ml = part_ml[i];
          const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - m);
          l += ml.x == -INFINITY ? ml.y : ml.y * f;
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] += f * part_o[i][lane * E + e];
        }
      }
      if (warp != 0) return;   // (a CTA has one row)
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* out = static_cast<T*>(a.out) + (static_cast<long long>(t) * a.N + kvh * G + (pr - t * G)) * HD + lane * E;
    __align__(8) T y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = from_float<T>(o[e] * inv);
    if (E == 4) *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(y);
    else *reinterpret_cast<uint32_t*>(out) = *reinterpret_cast<const uint32_t*>(y);
  }
}

template <typename T>
bool vectorised(const ortb200_prefix_attn_args* a) {
  if (a->cos_cache && (a->interleaved || a->rot_dim != a->H)) return false;
  uintptr_t p = reinterpret_cast<uintptr_t>(a->qkv) | reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v);
  if (a->cos_cache) p |= reinterpret_cast<uintptr_t>(a->cos_cache) | reinterpret_cast<uintptr_t>(a->sin_cache);
  return (p & 15) == 0;
}

template <typename T, int HD>
int launch_tc(const ortb200_prefix_attn_args* a, cudaStream_t stream) {
  using L = TcSmem<HD>;
  const CUtensorMapDataType dt = a->dtype == ORTB200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const int64_t rows = a->T * (a->N / a->Nk), entry = static_cast<int64_t>(a->Nk) * HD * 2;
  CUtensorMap tq, tk, tv;
  if (make_tensor_map_3d(&tq, work_of(*a).q, dt, 2, HD, rows, a->Nk, HD * 2, rows * HD * 2, 64, 16) != 0) return -6;
  const int64_t dims[4] = {HD, a->block_size, a->Nk, a->num_blocks}, strides[3] = {entry, HD * 2, entry * a->block_size};
  const int box = a->block_size < kKT ? a->block_size : kKT;
  if (make_tensor_map_4d(&tk, a->k_cache, dt, 2, dims, strides, 64, box) != 0) return -6;
  if (make_tensor_map_4d(&tv, a->v_cache, dt, 2, dims, strides, 64, box) != 0) return -6;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  auto kern = a->softcap > 64.f ? prefix_attn_kernel<HD, kBf16, 2> : a->softcap > 0.f ? prefix_attn_kernel<HD, kBf16, 1> : prefix_attn_kernel<HD, kBf16, 0>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal) != cudaSuccess) return -10;   // per device
  const int heads = a->N + 2 * a->Nk;
  const long long spread = 2 * kGrid / (a->T + 1), most = (heads + 15) / 16;   // few tokens: several CTAs per token, 16 heads at least to each
  const dim3 prep_grid(static_cast<unsigned>(a->T + 1), static_cast<unsigned>(spread < 1 ? 1 : spread > most ? most : spread));
  int rc = vectorised<T>(a) ? launch_kernel(prefix_prep_tc_kernel<T, true>, prep_grid, 128, 0, stream, a->use_pdl != 0, *a)
                            : launch_kernel(prefix_prep_tc_kernel<T, false>, prep_grid, 128, 0, stream, a->use_pdl != 0, *a);
  if (rc != 0) return rc;
  const float scale = a->scale != 0.f ? a->scale : 1.f / sqrtf(static_cast<float>(HD));
  // the two later steps may set up while the step before them ends: they wait for it before they read
  rc = launch_kernel(kern, dim3(kGrid), kThreads, L::kTotal, stream, true, tq, tk, tv, *a, scale);
  if (rc != 0) return rc;
  // Up to four rows per SM: a CTA each (one token of 32 heads over two key heads behind 18529 tokens: 23 us instead of 74 with one
  // warp a row).  Then one row per warp until there are rows for 16 warps on each SM, which is what fits at once: warps that come
  // later would look their segments up when the others have ended (24 prompts of up to 150 tokens: 37 us behind the product kernel
  // instead of 80).
  if (a->T * a->N <= 2 * kGrid) return launch_kernel(prefix_join_kernel<T, HD, true>, dim3(static_cast<unsigned>(a->T * a->N)), 128, 0, stream, true, *a, 1);
  const long long fit = 16 * kGrid / 2;
  const int per = static_cast<int>(std::min<long long>(32, (a->T * a->N + fit - 1) / fit));
  const long long warps = (rows + per - 1) / per * a->Nk;
  return launch_kernel(prefix_join_kernel<T, HD, false>, dim3(static_cast<unsigned>((warps + 3) / 4)), 128, 0, stream, true, *a, per);
}

template <typename T>
int launch_rows(const ortb200_prefix_attn_args* a, cudaStream_t stream) {
  T* q = static_cast<T*>(a->workspace);
  int rc = launch_kernel(prefix_prep_kernel<T>, dim3(static_cast<unsigned>(a->T + 1)), 128, 0, stream, a->use_pdl != 0, *a, q);
  if (rc != 0) return rc;
  const long long items = a->T * a->N;
  return launch_kernel(prefix_rows_kernel<T>, dim3(static_cast<unsigned>((items + 3) / 4)), 128, 0, stream, a->use_pdl != 0, *a, static_cast<const T*>(q));
}

}  // namespace
}  // namespace ortb200

using namespace ortb200;

extern "C" int64_t ortb200_prefix_attn_max_keys(void) { return kMaxKeys; }

extern "C" int64_t ortb200_prefix_attn_workspace_bytes(int64_t T, int B, int N, int Nk, int H, int tensor_cores) {
  if (T < 0 || B < 0 || N <= 0 || Nk <= 0 || H <= 0) return -1;
  if (!tensor_cores) return up256(T * N * H * 4);
  return plan_bytes(T, B, N, Nk) + up256(T * 16) + up256(T * N * H * 2) + up256(segment_rows(T, N) * 8) + segment_rows(T, N) * H * 4;
}

extern "C" int ortb200_prefix_attn(const ortb200_prefix_attn_args* a, ortb200_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!a || a->T < 0 || a->B < 0 || a->N <= 0 || a->Nk <= 0 || a->N % a->Nk != 0 || a->H <= 0) return -1;
  if (a->T == 0) return 0;
  if (!a->qkv || !a->k_cache || !a->v_cache || !a->cu_seqlens || !a->out || !a->shared_prefix || !a->workspace) return -1;
  if (a->B > 0 && (!a->past_seqlens || !a->block_table)) return -1;
  if ((a->k != nullptr) != (a->v != nullptr) || (a->positions != nullptr) != (a->slot_mapping != nullptr)) return -1;
  if (a->block_size <= 0 || a->max_blocks <= 0 || a->num_blocks <= 0) return -1;
  if (a->cos_cache && (!a->sin_cache || a->cos_rows <= 0 || a->rot_dim <= 0 || a->rot_dim % 2 != 0 || a->rot_dim > a->H)) return -1;
  if (a->H > kMaxHead || a->T * a->N > (a->tensor_cores ? 1ll << 29 : 0x7ffffffell)) return -2;   // (places of segment rows, doubled, pass in 32 bits)
  // what a sequence may hold, and the width of a token, pass in 32 bits
  if (static_cast<long long>(a->max_blocks) * a->block_size > kMaxKeys || (a->N + 2ll * a->Nk) * a->H > 0x7fffffffll) return -2;
  if (a->workspace_bytes < ortb200_prefix_attn_workspace_bytes(a->T, a->B, a->N, a->Nk, a->H, a->tensor_cores)) return -1;
  if (a->tensor_cores) {
    const bool blocks = a->block_size % kKT == 0 || a->block_size == 8 || a->block_size == 16 || a->block_size == 32;
    if ((a->H != 64 && a->H != 128) || !blocks || a->N / a->Nk > kQT) return -2;
    if ((reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache) | reinterpret_cast<uintptr_t>(a->out)) & 15) return -3;
    if (reinterpret_cast<uintptr_t>(a->workspace) & 255) return -3;
    if (a->dtype == ORTB200_BF16) return a->H == 128 ? launch_tc<__nv_bfloat16, 128>(a, stream) : launch_tc<__nv_bfloat16, 64>(a, stream);
    if (a->dtype == ORTB200_F16) return a->H == 128 ? launch_tc<__half, 128>(a, stream) : launch_tc<__half, 64>(a, stream);
    return -4;
  }
  switch (a->dtype) {
    case ORTB200_F16: return launch_rows<__half>(a, stream);
    case ORTB200_BF16: return launch_rows<__nv_bfloat16>(a, stream);
    case ORTB200_F32: return launch_rows<float>(a, stream);
  }
  return -4;
}
