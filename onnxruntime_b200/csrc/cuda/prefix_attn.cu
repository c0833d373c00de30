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
// (S = Q K^T into tensor memory, O += P V with P in tensor memory over the scores), warps 2 to 5 hold one row per thread.
#include <cuda.h>
#include <cuda_runtime.h>
#include <math.h>
#include <type_traits>
#include "attn_internal.h"
#include "launch_util.cuh"
#include "serving_ops.h"
#include "tensor_map.h"

namespace ortb200 {
namespace {

constexpr int kMaxHead = 256;

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
__device__ __forceinline__ int last_row(const ortb200_prefix_attn_args& a) { return min(max(a.cu_seqlens[a.B], 0), static_cast<int>(a.T)); }

// Row t: rotate its query heads into `q_out` [T, N, H], its key heads into the cache beside the values.
template <typename T>
__global__ void __launch_bounds__(128) prefix_prep_kernel(const ortb200_prefix_attn_args a, T* q_out) {
  const int t = blockIdx.x, H = a.H, heads = a.N + 2 * a.Nk, half = a.rot_dim / 2;
  pdl_wait_prior_grids();
  if (t >= last_row(a)) return;
  const int b = sequence_of(a.cu_seqlens, a.B, t);
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
  if (t < last_row(a)) {
    const int b = sequence_of(a.cu_seqlens, a.B, t);
    const Span s = span_of(a, b);   // (cumulative lengths that start behind 0 leave rows to nobody: no keys)
    const long long cap = static_cast<long long>(a.max_blocks) * a.block_size;
    const int keys = static_cast<int>(min(static_cast<long long>(s.past) + (t - s.row0) + 1, cap));
    const float scale = a.scale != 0.f ? a.scale : 1.f / sqrtf(static_cast<float>(H));
#pragma unroll
    for (int r = 0; r < R; ++r) qv[r] = r * 32 + lane < H ? to_float<T>(q[item * H + r * 32 + lane]) : 0.f;
    for (int j = 0; j < keys; ++j) {
      const int block = a.block_table[static_cast<long long>(b) * a.max_blocks + j / a.block_size];
      if (block < 0 || block >= a.num_blocks) continue;
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
constexpr bool kSplit = true;
constexpr int kQT = 128;          // query rows of a unit
constexpr int kKT = 64;           // keys of a tile
constexpr int kThreads = 192;
constexpr int kGrid = 296;        // two CTAs on each of 148 SMs
constexpr int kTmemCols = 256;    // two score buffers of 64 columns, O in up to 128
constexpr int kPlanInSmem = 1024; // sequences whose running sums a CTA keeps in shared memory

// What follows from the lengths.
struct Plan {
  long long total;       // length of the numbering
  int prefix_tiles;      // tiles of the prefix
  int prefix_row;        // row of the block table that the prefix is read from
};

struct Work {            // the workspace's parts
  Plan* plan;
  long long* first;      // [B + 1]: where the own units of each sequence start, behind the prefix's
  int4* token;           // [T]: the token's sequence, that sequence's first row, rows and past
  uint16_t* q;           // [Nk, T G, H]
  float2* ml;            // per row of a segment: m (in units of log 2) and l
  float* o;              // per row of a segment: H values
};
__host__ __device__ inline long long up256(long long n) { return (n + 255) / 256 * 256; }
__host__ __device__ inline long long segment_rows(long long T, int N) { return 2 * T * N + static_cast<long long>(kGrid) * kQT; }
__host__ __device__ inline Work work_of(const ortb200_prefix_attn_args& a) {
  char* p = static_cast<char*>(a.workspace);
  Work w;
  w.plan = reinterpret_cast<Plan*>(p);
  w.first = reinterpret_cast<long long*>(p + sizeof(Plan));
  p += up256(sizeof(Plan) + 8ll * (a.B + 1));
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
// costs a CTA as much time as some tiles, the more the more rows are written, and a share of many short units has to be worth as
// much as one of a long unit.
__device__ __forceinline__ int extra(int rows) { return rows > 32 ? 5 : 2; }
__device__ __forceinline__ int places(int tiles, int rows) { return tiles > 0 ? tiles + extra(rows) : 0; }
// The share of CTA i of `total` places starts at share(i); place x belongs to CTA owner(x).
__device__ __forceinline__ long long share(long long total, int i) { return total * i / kGrid; }
__device__ __forceinline__ int owner(long long total, long long x) { return static_cast<int>(((x + 1) * kGrid - 1) / total); }

// Unit `rt` (rows [128 rt, 128 rt + 128) of the sequence's rows x G) of a sequence: its keys [prefix keys, end) in tiles of 64.
__device__ __forceinline__ int own_end(const ortb200_prefix_attn_args& a, const Span& s, int rt) {
  const int G = a.N / a.Nk, last = min(rt * kQT + kQT, s.rows * G) - 1;
  return static_cast<int>(min(static_cast<long long>(s.past) + last / G + 1, static_cast<long long>(a.max_blocks) * a.block_size));
}
__device__ __forceinline__ int own_tiles(const ortb200_prefix_attn_args& a, const Span& s, int rt, int prefix_tiles) {
  return max((own_end(a, s, rt) + kKT - 1) / kKT - prefix_tiles, 0);
}
__device__ __forceinline__ int row_tiles(const ortb200_prefix_attn_args& a, int rows) { return (rows * (a.N / a.Nk) + kQT - 1) / kQT; }
__device__ __forceinline__ int unit_rows(const ortb200_prefix_attn_args& a, int rows, int rt) { return min(kQT, rows * (a.N / a.Nk) - rt * kQT); }
__device__ __forceinline__ int own_places(const ortb200_prefix_attn_args& a, const Span& s, int rt, int prefix_tiles) {
  return places(own_tiles(a, s, rt, prefix_tiles), unit_rows(a, s.rows, rt));
}
// all units of the prefix are numbered like the first
__device__ __forceinline__ long long prefix_places(const ortb200_prefix_attn_args& a, int all_rows, int prefix_tiles) {
  return static_cast<long long>(row_tiles(a, all_rows)) * a.Nk * places(prefix_tiles, unit_rows(a, all_rows, 0));
}
// first row that the segments of a unit may use, before 128 rows per CTA number: units follow one another without a gap
__device__ __forceinline__ long long prefix_slot(const ortb200_prefix_attn_args& a, int rt, int kvh, int rows) {
  return static_cast<long long>(rt) * kQT * a.Nk + static_cast<long long>(kvh) * rows;
}
__device__ __forceinline__ long long own_slot(const ortb200_prefix_attn_args& a, int row0, int rt, int kvh, int rows) {
  return a.T * a.N + static_cast<long long>(a.Nk) * (static_cast<long long>(row0) * (a.N / a.Nk) + static_cast<long long>(rt) * kQT) + static_cast<long long>(kvh) * rows;
}

// All THREADS of a CTA: how many tokens all sequences share, and where the own units of each sequence start (`first`, written
// for all to read after the next barrier).
template <int THREADS>
__device__ __forceinline__ Plan make_plan(const ortb200_prefix_attn_args& a, long long* first, int* status) {
  __shared__ int least_sm[THREADS / 32], row_sm[THREADS / 32];
  __shared__ long long sum_sm[THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int least = 0x7fffffff, row = 0x7fffffff;
  const int promised = *a.shared_prefix, all_rows = last_row(a);
  for (int b = threadIdx.x; b < a.B; b += THREADS) {
    const Span s = span_of(a, b);
    if (s.rows == 0) continue;
    least = min(least, s.past);
    row = min(row, b);
    if (status && (a.past_seqlens[b] != s.past || s.past + static_cast<long long>(s.rows) > static_cast<long long>(a.max_blocks) * a.block_size))
      atomicExch(status, kStatusBadLength);
  }
  least = __reduce_min_sync(0xffffffffu, least);
  row = __reduce_min_sync(0xffffffffu, row);
  if (lane == 0) {
    least_sm[warp] = least;
    row_sm[warp] = row;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) {
    least = min(least, least_sm[i]);
    row = min(row, row_sm[i]);
  }
  Plan p;
  p.prefix_tiles = least == 0x7fffffff ? 0 : max(min(promised, least), 0) / kKT;
  p.prefix_row = row == 0x7fffffff ? 0 : row;
  long long base = 0;
  for (int b0 = 0; b0 < a.B; b0 += THREADS) {
    const int b = b0 + threadIdx.x;
    long long n = 0;
    if (b < a.B) {
      const Span s = span_of(a, b);
      for (int rt = 0; rt < row_tiles(a, s.rows); ++rt) n += own_places(a, s, rt, p.prefix_tiles);
      n *= a.Nk;
    }
    long long sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    if (b0 > 0) __syncthreads();
    if (lane == 31) sum_sm[warp] = sum;
    __syncthreads();
    long long before = base;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
      if (i < warp) before += sum_sm[i];
      base += sum_sm[i];
    }
    if (b < a.B) first[b] = before + sum - n;
  }
  if (threadIdx.x == 0) first[a.B] = base;
  p.total = base + prefix_places(a, all_rows, p.prefix_tiles);
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
    const Plan p = make_plan<128>(a, w.first, a.status);
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
  static constexpr int kTotal = kOffFirst + 8 * (kPlanInSmem + 1) + 1024;
};
enum { BAR_Q = 0, BAR_Q_FREE = BAR_Q + 2, BAR_K_FULL = BAR_Q_FREE + 2, BAR_K_EMPTY = BAR_K_FULL + 3, BAR_V_FULL = BAR_K_EMPTY + 3, BAR_V_EMPTY = BAR_V_FULL + 3, BAR_S = BAR_V_EMPTY + 3,
       BAR_P = BAR_S + 2, BAR_O = BAR_P + 2, BAR_END, BAR_O_FREE, BAR_COUNT };
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
struct Walk {
  const ortb200_prefix_attn_args& a;
  const long long* first;
  Plan plan;
  int all_rows;
  long long prefix_total, cur, stop;
  __device__ Walk(const ortb200_prefix_attn_args& args, const long long* f, const Plan& p, int cta) : a(args), first(f), plan(p) {
    all_rows = last_row(a);
    prefix_total = prefix_places(a, all_rows, p.prefix_tiles);
    cur = share(p.total, cta);
    stop = share(p.total, cta + 1);
  }
  __device__ bool next(Segment& g) {
    const int G = a.N / a.Nk;
    while (cur < stop) {
      int n, at, before;    // the unit's tiles, the place within it, and the places in front of its tiles
      if (cur < prefix_total) {
        n = plan.prefix_tiles;
        before = extra(unit_rows(a, all_rows, 0));
        const long long u = cur / (n + before);
        at = static_cast<int>(cur - u * (n + before));
        const int rt = static_cast<int>(u / a.Nk);
        g.kvh = static_cast<int>(u % a.Nk);
        g.seq = -1;
        g.q_row = rt * kQT;
        g.rows = unit_rows(a, all_rows, rt);
        g.key0 = 0;
        g.end = n * kKT;
        g.past = g.in_seq = 0;
        g.table_row = plan.prefix_row;
        g.slot = prefix_slot(a, rt, g.kvh, g.rows);
      } else {
        long long x = cur - prefix_total;
        int lo = 0, hi = a.B;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (first[mid] <= x) lo = mid; else hi = mid;
        }
        x -= first[lo];
        const Span s = span_of(a, lo);
        int rt = 0, all = own_places(a, s, 0, plan.prefix_tiles);
        while (x >= static_cast<long long>(all) * a.Nk) {
          x -= static_cast<long long>(all) * a.Nk;
          all = own_places(a, s, ++rt, plan.prefix_tiles);
        }
        g.kvh = static_cast<int>(x) / all;
        at = static_cast<int>(x) % all;
        g.seq = lo;
        g.in_seq = rt * kQT;
        g.q_row = s.row0 * G + g.in_seq;
        g.rows = unit_rows(a, s.rows, rt);
        before = extra(g.rows);
        n = all - before;
        g.key0 = plan.prefix_tiles * kKT;
        g.end = own_end(a, s, rt);
        g.past = s.past;
        g.table_row = lo;
        g.slot = own_slot(a, s.row0, rt, g.kvh, g.rows);
      }
      const int upto = static_cast<int>(min(static_cast<long long>(n + before), at + (stop - cur)));
      cur += upto - at;
      const int t0 = max(at - before, 0);
      g.tiles = max(upto - before, 0) - t0;
      g.key0 += t0 * kKT;
      if (g.tiles > 0) return true;
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

__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait_bar(bar, parity)); }

template <int HD, bool BF16, bool CAP>
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
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    for (int i = 0; i < BAR_COUNT; ++i) mbar_init(&bars[i], i == BAR_P || i == BAR_P + 1 || i == BAR_O_FREE ? 4 : 1);
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
  const bool kept = a.B <= kPlanInSmem;
  if (kept) {
    plan = make_plan<kThreads>(a, first_sm, nullptr);
  } else {
    pdl_wait_prior_grids();
    plan = *w.plan;
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_s = __reduce_or_sync(0xffffffffu, *tmem_slot);   // S / P: two buffers of 64 columns; the same for all, and known to be
  const uint32_t tmem_o = tmem_s + 2 * kKT;

  Walk walk(a, kept ? first_sm : w.first, plan, blockIdx.x);
  Segment g;
  bool ok = true;

  if (warp == 0) {
    // ---------------------------------------------------------------------------------------------------- loads
    const int piece = min(a.block_size, kKT), pieces = kKT / piece;   // rows that one block gives a tile
    int s = 0, k_tiles = 0, v_tiles = 0;
    uint32_t parity = 1;   // the first round over the stages waits for nothing
    QueryPlace qp;
    bool waited = !kept;
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
      auto block_at = [&](int key) { return min(max(table[min(key / a.block_size, a.max_blocks - 1)], 0), a.num_blocks - 1); };
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
      while (ok && walk.next(g)) {
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
          if (kSplit)
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
    // The reference maximum of a row is raised only when a tile exceeds it by 2^8 (weights stay below 256), so that O in tensor
    // memory is rescaled a few times per row.
    constexpr float kRaise = 8.f;
    int seg = 0, it = 0;
    while (ok && walk.next(g)) {
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
#pragma unroll
            for (int j = 0; j < kKT; ++j) sv[j] = a.softcap * tanhf(sv[j] * scale / a.softcap) * 1.4426950408889634f;
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
          float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
          for (int c = 0; c < kKT; c += 32) {
            uint32_t packed[16], rest[16];
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float p0 = ex2_approx(fmaf(sv[c + j], fs, neg_m)), p1 = ex2_approx(fmaf(sv[c + j + 1], fs, neg_m));
              sum0 += p0;
              sum1 += p1;
              if (BF16) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(p0, p1);
                packed[j / 2] = *reinterpret_cast<const uint32_t*>(&h);
                if (kSplit) {
                  const __nv_bfloat162 d = __floats2bfloat162_rn(p0 - __low2float(h), p1 - __high2float(h));
                  rest[j / 2] = *reinterpret_cast<const uint32_t*>(&d);
                }
              } else {
                const __half2 h = __floats2half2_rn(p0, p1);
                packed[j / 2] = *reinterpret_cast<const uint32_t*>(&h);
                if (kSplit) {
                  const __half2 d = __floats2half2_rn(p0 - __low2float(h), p1 - __high2float(h));
                  rest[j / 2] = *reinterpret_cast<const uint32_t*>(&d);
                }
              }
            }
            tmem_st_x16_u32(s_addr + c / 2, packed);
            if (kSplit) tmem_st_x16_u32(s_addr + kKT / 2 + c / 2, rest);
          }
          l += sum0 + sum1;
          tmem_st_wait();
        }
        const int live = g.end - key0;
        if (live < kKT && ok) {
          // what lies behind the last key may be anything, and 0 * NaN would reach the product: these rows of V become 0
          if (!wait_warp(&bars[BAR_V_FULL + it % STAGES], (it / STAGES) & 1)) ok = false;
          uint8_t* v = smem + L::kOffKV + it % STAGES * L::kStageBytes + L::kBoxes * L::kBox + live * 128;
          for (int i = r; i < (kKT - live) * 8; i += 128)
#pragma unroll
            for (int bx = 0; bx < L::kBoxes; ++bx) *reinterpret_cast<uint4*>(v + bx * L::kBox + i * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async();
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[BAR_P + (it & 1)]);
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
// Step 3: one warp per token and query head.
template <typename T, int HD>
__global__ void __launch_bounds__(128) prefix_join_kernel(const ortb200_prefix_attn_args a) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (item >= a.T * a.N) return;
  const Work w = work_of(a);
  const int t = static_cast<int>(item / a.N), head = static_cast<int>(item % a.N), G = a.N / a.Nk, kvh = head / G, all_rows = last_row(a);
  float o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  // (step 1 has ended when this step begins: only the segments are waited for)
  const int4 tok = __ldcg(&w.token[t]);
  const Plan plan = {__ldcg(&w.plan->total), __ldcg(&w.plan->prefix_tiles), 0};
  const bool live = t < all_rows && t >= tok.y && t < tok.y + tok.z && plan.total > 0;   // lengths that start behind 0 leave rows to nobody
  // the row's two units, 0 of the prefix and 1 of its own keys: first tile in the numbering, tiles, first slot
  long long from0 = 0, from1 = 0, slot0 = 0, slot1 = 0;
  int tiles0 = 0, tiles1 = 0;
  if (live) {
    const Span s = {tok.y, tok.z, tok.w};
    const int pr = t * G + head % G, prt = pr / kQT, orow = (t - s.row0) * G + head % G, ort = orow / kQT;
    tiles0 = plan.prefix_tiles;
    const int before0 = extra(unit_rows(a, all_rows, 0));
    from0 = (static_cast<long long>(prt) * a.Nk + kvh) * (tiles0 + before0) + before0;
    slot0 = prefix_slot(a, prt, kvh, unit_rows(a, all_rows, prt)) + pr % kQT;
    long long start = prefix_places(a, all_rows, tiles0) + __ldcg(&w.first[tok.x]);
    for (int rt = 0; rt < ort; ++rt) start += static_cast<long long>(own_places(a, s, rt, tiles0)) * a.Nk;
    tiles1 = own_tiles(a, s, ort, tiles0);
    const int rows1 = unit_rows(a, s.rows, ort);
    from1 = start + static_cast<long long>(kvh) * places(tiles1, rows1) + extra(rows1);
    slot1 = own_slot(a, s.row0, ort, kvh, rows1) + orow % kQT;
  }
  // segment k of the row, over both units: CTA first0 + k of the one or first1 + k - count0 of the other
  const int first0 = tiles0 > 0 ? owner(plan.total, from0) : 0, count0 = tiles0 > 0 ? owner(plan.total, from0 + tiles0 - 1) - first0 + 1 : 0;
  const int first1 = tiles1 > 0 ? owner(plan.total, from1) : 0, count1 = tiles1 > 0 ? owner(plan.total, from1 + tiles1 - 1) - first1 + 1 : 0;
  pdl_wait_prior_grids();
  for (int k0 = 0; k0 < count0 + count1; k0 += 32) {
    const int k = k0 + lane;
    const bool own = k >= count0;
    const int i = own ? first1 + k - count0 : first0 + k;
    const long long from = own ? from1 : from0;
    const bool has = k < count0 + count1 && max(from, share(plan.total, i)) < min(from + (own ? tiles1 : tiles0), share(plan.total, i + 1));
    const long long row = (own ? slot1 : slot0) + static_cast<long long>(i) * kQT;
    const float2 ml = has ? __ldcg(&w.ml[row]) : make_float2(-INFINITY, 0.f);
    unsigned left = __ballot_sync(0xffffffffu, has);
    // the segments' values are on their way while the weights are formed
    constexpr int R = 8;
    float v[R][E];
    int at[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      at[r] = left != 0 ? __ffs(left) - 1 : -1;
      left &= left - 1;
      const long long rw = __shfl_sync(0xffffffffu, row, max(at[r], 0));
      if (at[r] >= 0) load_cg<E>(w.o + rw * HD + lane * E, v[r]);
    }
    const float mm = fmaxf(m, warp_max(ml.x));
    const float keep = m == -INFINITY ? 0.f : exp2f(m - mm), mine = ml.x == -INFINITY ? 0.f : exp2f(ml.x - mm);
    // a row whose scores are all NaN has no maximum; its sum carries the NaN on
    l = l * keep + warp_sum(ml.x == -INFINITY ? ml.y : ml.y * mine);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= keep;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float f = __shfl_sync(0xffffffffu, mine, max(at[r], 0));
      if (at[r] >= 0)
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += f * v[r][e];
    }
    for (; left != 0; left &= left - 1) {
      const int j = __ffs(left) - 1;
      const float f = __shfl_sync(0xffffffffu, mine, j);
      float x[E];
      load_cg<E>(w.o + __shfl_sync(0xffffffffu, row, j) * HD + lane * E, x);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] += f * x[e];
    }
    m = mm;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* out = static_cast<T*>(a.out) + item * HD + lane * E;
  __align__(8) T y[E];
#pragma unroll
  for (int e = 0; e < E; ++e) y[e] = from_float<T>(o[e] * inv);
  if (E == 4) *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(y);
  else *reinterpret_cast<uint32_t*>(out) = *reinterpret_cast<const uint32_t*>(y);
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
  auto kern = a->softcap > 0.f ? prefix_attn_kernel<HD, kBf16, true> : prefix_attn_kernel<HD, kBf16, false>;
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
  return launch_kernel(prefix_join_kernel<T, HD>, dim3(static_cast<unsigned>((a->T * a->N + 3) / 4)), 128, 0, stream, true, *a);
}

template <typename T>
int launch_rows(const ortb200_prefix_attn_args* a, cudaStream_t stream) {
  T* q = static_cast<T*>(a->workspace);
  int rc = launch_kernel(prefix_prep_kernel<T>, dim3(static_cast<unsigned>(a->T)), 128, 0, stream, a->use_pdl != 0, *a, q);
  if (rc != 0) return rc;
  const long long items = a->T * a->N;
  return launch_kernel(prefix_rows_kernel<T>, dim3(static_cast<unsigned>((items + 3) / 4)), 128, 0, stream, a->use_pdl != 0, *a, static_cast<const T*>(q));
}

}  // namespace
}  // namespace ortb200

using namespace ortb200;

extern "C" int64_t ortb200_prefix_attn_workspace_bytes(int64_t T, int B, int N, int Nk, int H, int tensor_cores) {
  if (!tensor_cores) return up256(T * N * H * 4);
  return up256(sizeof(Plan) + 8ll * (B + 1)) + up256(T * 16) + up256(T * N * H * 2) + up256(segment_rows(T, N) * 8) + segment_rows(T, N) * H * 4;
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
  if (a->H > kMaxHead || a->T * a->N > 0x7fffffffll) return -2;
  if (a->workspace_bytes < ortb200_prefix_attn_workspace_bytes(a->T, a->B, a->N, a->Nk, a->H, a->tensor_cores)) return -1;
  if (a->tensor_cores) {
    const bool blocks = a->block_size % kKT == 0 || a->block_size == 8 || a->block_size == 16 || a->block_size == 32;
    if ((a->H != 64 && a->H != 128) || !blocks || a->N / a->Nk > kQT) return -2;
    if (((reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache)) & 15) || (reinterpret_cast<uintptr_t>(a->workspace) & 255)) return -3;
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
