// Log probabilities of given tokens, entropy and the best alternatives out of logits (com.ortb200.TokenLogProbs), and their
// gradient (com.ortb200.TokenLogProbsGrad).
//
// One pass over a row.  A thread keeps a running maximum m, S = sum exp(x - m) and W = sum exp(x - m) (x - m) of the logits it has
// seen; when the maximum moves from m to m', W becomes (W + S (m - m')) c and S becomes S c with c = exp(m - m').  Joined over
// the row: log_sum_exp = m + log S and entropy = log S - W / S.  All of it is held in 32 bits; m is a logit as it is, exponents
// and W are to the base 2.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <math.h>
#include "launch_util.cuh"
#include "serving_ops.h"

namespace ortb200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kMaxTop = 32, kMaxParts = 16;
constexpr int kMaxVocab = 0x7fff0000;   // an index plus the threads of a CTA fits 31 bits
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_fast(float t) {   // relative error 2^-22
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}
__device__ __forceinline__ float exp_fast(float d) { return exp2_fast(d * kLog2e); }   // and |d| 2^-23: what is far below 1 weighs little

// A row as its first elements up to a 16-byte boundary, whole vectors, and the rest.
template <typename T>
struct Row {
  static constexpr int E = 16 / sizeof(T);
  const T* x;
  int head, vectors, n;
  __device__ Row(const T* p, int vocab) : x(p), n(vocab) {
    head = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / static_cast<int>(sizeof(T)), vocab);
    vectors = (vocab - head) / E;
  }
  __device__ const uint4* body() const { return reinterpret_cast<const uint4*>(x + head); }
  __device__ int tail() const { return head + vectors * E; }
};
template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float* f) {
  const T* t = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < Row<T>::E; ++i) f[i] = to_float<T>(t[i]);
}

__device__ __forceinline__ float max3(float a, float b, float c) {   // NaN if one of them is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

constexpr float kFar = -1e30f;   // an exponent below all that count: 0 times it is 0, where 0 times -inf would be NaN

// m the largest logit, s = sum 2^t, w = sum 2^t t with t = (x - m) log2(e).  The difference comes first: the maximum's own exponent is
// 0 whatever its size.  (One multiply-add x log2(e) - m log2(e) is off by 2^-24 of |m|, which for masks of -1e10 and beyond is more
// than a 32-bit exponent holds; it took 592 us instead of 601 in a call for 4096 rows of 128256 bf16 logits and their gradient.)  Two logits go
// through one instruction.
struct Stats {
  float m, s, w;
  static __device__ __forceinline__ Stats none() { return {-INFINITY, 0.f, 0.f}; }
  __device__ __forceinline__ void raise(float to) {   // to >= m
    if (s != 0.f) {
      const float d = fmaxf((m - to) * kLog2e, kFar), c = exp2f(d);
      w = d == 0.f ? w : (w + s * d) * c;
      s *= c;
    }
    m = to;
  }
  // N logits whose largest is `top` (NaN if one of them is)
  template <int N>
  __device__ __forceinline__ void add(const float* x, float top) {
    if (top > m) raise(top);
    const float ref = m == -INFINITY ? 0.f : -m;
    if (N == 1) {
      const float t = max_nan((x[0] + ref) * kLog2e, kFar), e = exp2_fast(t);
      s += e;
      w = fmaf(e, t, w);
      return;
    }
    const f32x2 scale = pack2(kLog2e, kLog2e), ref2 = pack2(ref, ref), one = pack2(1.f, 1.f);
    f32x2 s2 = pack2(0.f, 0.f), w2 = s2;
#pragma unroll
    for (int i = 0; i + 1 < N; i += 2) {
      float t0, t1;
      unpack2(mul2(fma2(pack2(x[i], x[i + 1]), one, ref2), scale), t0, t1);
      t0 = max_nan(t0, kFar);   // (an impossible token has -inf, and so has one beyond 32 bits below the largest)
      t1 = max_nan(t1, kFar);
      const f32x2 e = pack2(exp2_fast(t0), exp2_fast(t1));
      s2 = fma2(e, one, s2);
      w2 = fma2(e, pack2(t0, t1), w2);
    }
    float a, b;
    unpack2(s2, a, b);
    s += a + b;
    unpack2(w2, a, b);
    w += a + b;
  }
  __device__ __forceinline__ void join(Stats b) {
    const float to = fmaxf(m, b.m);
    raise(to);
    b.raise(to);
    s += b.s;
    w += b.w;
  }
  __device__ __forceinline__ Stats shuffle_xor(int o) const {
    Stats r;
    r.m = __shfl_xor_sync(0xffffffffu, m, o);
    r.s = __shfl_xor_sync(0xffffffffu, s, o);
    r.w = __shfl_xor_sync(0xffffffffu, w, o);
    return r;
  }
};

// A key orders (value, index) pairs by value, then by lower index; zeros of both signs are equal, NaN is the largest.
__device__ __forceinline__ unsigned order_of(float f) {
  f += 0.f;
  const unsigned u = __float_as_uint(f);
  return f != f ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float ordered(unsigned order) { return __uint_as_float((order & 0x80000000u) ? order & 0x7fffffffu : ~order); }
__device__ __forceinline__ unsigned long long key_of(float f, int index) { return (static_cast<unsigned long long>(order_of(f)) << 32) | (0xffffffffu - static_cast<unsigned>(index)); }
__device__ __forceinline__ float value_of(unsigned long long key) { return ordered(static_cast<unsigned>(key >> 32)); }

// The 32 best pairs a warp has seen, lane i the i-th best.
struct Best {
  unsigned long long mine = 0;     // this lane's pair; 0: none
  unsigned long long last = 0;     // the top_k-th: what is not above it is no alternative
  __device__ __forceinline__ void insert(unsigned long long key, int lane, int top_k) {
    const int above = __popc(__ballot_sync(0xffffffffu, mine > key));
    const unsigned long long up = __shfl_up_sync(0xffffffffu, mine, 1);
    if (lane > above) mine = up;
    if (lane == above) mine = key;
    last = __shfl_sync(0xffffffffu, mine, top_k - 1);
  }
  // one pair of every lane (0: none)
  __device__ __forceinline__ void offer(unsigned long long key, int lane, int top_k) {
    for (unsigned left = __ballot_sync(0xffffffffu, key > last); left != 0; left &= left - 1) {
      const unsigned long long k = __shfl_sync(0xffffffffu, key, __ffs(left) - 1);
      if (k > last) insert(k, lane, top_k);
    }
  }
  __device__ __forceinline__ void offer_one(bool has, float x, int index, int lane, int top_k) { offer(has ? key_of(x, index) : 0, lane, top_k); }
};
// The k largest of n different keys (0: none) in shared memory, in order, to out[0 .. k), which holds zeros: a key's place is the
// number of larger ones.
__device__ __forceinline__ void select_best(const unsigned long long* keys, int n, unsigned long long* out, int k) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const unsigned long long mine = keys[i];
    if (mine == 0) continue;
    int larger = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) larger += keys[j] > mine;
    if (larger < k) out[larger] = mine;
  }
}

struct Shared {
  Stats stats[kThreads / 32];
  Stats part_stats[kMaxParts];                            // the first CTA's: what the cluster's CTAs found
  unsigned bound, kth[2];                                 // values (order_of) that top_k of the CTA's reach: of a warp's list, of the threads' largest
  __align__(16) unsigned tops[kThreads];
  unsigned long long best[kThreads / 32 * kMaxTop];
  unsigned long long part_best[kMaxParts * kMaxTop];      // the first CTA's
  unsigned long long chosen[kMaxTop];
};

// order_of the top_k-th largest of what the threads hold.  `turn` counts the calls: what the last call found may still be read.
__device__ __forceinline__ unsigned kth_of_threads(Shared& sm, float top, int turn, int lane, int top_k) {
  unsigned sorted = order_of(top);
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int o = size / 2; o > 0; o >>= 1) {   // a bitonic sort of the warp's, the largest first
      const unsigned other = __shfl_xor_sync(0xffffffffu, sorted, o);
      sorted = ((lane & o) == 0) == ((lane & size) == 0) ? max(sorted, other) : min(sorted, other);
    }
  if (lane < top_k) sm.tops[(threadIdx.x >> 5) * top_k + lane] = sorted;
  if (threadIdx.x == 0) {
    sm.kth[turn & 1] = 0xffffffffu;
    if (turn == 0) sm.bound = 0;
  }
  __syncthreads();
  const int n = kThreads / 32 * top_k;
  if (static_cast<int>(threadIdx.x & ~31u) >= n) {   // (whole warps)
    __syncthreads();
    return sm.kth[turn & 1];
  }
  const unsigned mine = static_cast<int>(threadIdx.x) < n ? sm.tops[threadIdx.x] : 0;
  int larger = static_cast<int>(threadIdx.x) < n ? 0 : top_k;
  for (int i = 0; i < n; i += 4) {   // (8 lists: a multiple of 4)
    const uint4 t = *reinterpret_cast<const uint4*>(sm.tops + i);
    larger += (t.x > mine) + (t.y > mine) + (t.z > mine) + (t.w > mine);
  }
  const unsigned least = __reduce_min_sync(0xffffffffu, larger < top_k ? mine : 0xffffffffu);
  if (lane == 0) atomicMin(&sm.kth[turn & 1], least);
  __syncthreads();
  return sm.kth[turn & 1];
}

// A cluster of CTAs per row, each with a share of its vectors; the first CTA puts the shares together over distributed shared memory.
//
// Without alternatives the row is one stream: 2000 rows of 50257 fp32 logits take 70 us (402 MB, 61 at the copy rate), 2000 of bf16
// 52 (201 MB, 31: the exponentials, 16 a clock and SM, take 27 by themselves), 6 rows of 128256 bf16 4.8, which is latency: begin, one
// round of loads, two barriers of the cluster.  With the best 1 / 5 / 20: 84 / 98 / 139, 71 / 88 / 125 and 7.6 / 9.1 / 16 us.  What costs
// there is not the insertions alone: bounds from one warp each (110 us for bf16 with one alternative), lists merged one by
// one (13 us for 6 rows with five) and ranks counted among all 256 threads' values (120) were slower.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, TOP && sizeof(T) == 4 ? 3 : 4) token_log_probs_kernel(const ortb200_token_log_probs_args a) {
  constexpr int E = Row<T>::E, U = TOP && E == 8 ? 2 : 4;
  __shared__ Shared sm;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, top_k = a.top_k;
  const long long row = blockIdx.x / parts;
  pdl_wait_prior_grids();
  const Row<T> x(static_cast<const T*>(a.logits) + row * a.vocab, a.vocab);
  long long token = -1;
  float chosen = 0.f;
  if (part == 0 && threadIdx.x == 0) {
    token = a.tokens[row];
    if (token >= 0 && token < a.vocab) chosen = to_float<T>(x.x[token]);
  }
  Stats st = Stats::none();
  Best best;
  if (parts > 1) cluster.barrier_arrive();   // (waited for before anything goes to another CTA's memory: that one has begun then)
  if (part == 0) {   // the elements in front of the first vector: fewer than a warp
    const bool has = static_cast<int>(threadIdx.x) < x.head;
    const float f = has ? to_float<T>(x.x[threadIdx.x]) : 0.f;
    if (has) st.add<1>(&f, f);
    if (TOP && warp == 0) best.offer_one(has, f, threadIdx.x, lane, top_k);
  }
  const int from = static_cast<int>(static_cast<long long>(x.vectors) * part / parts), to = static_cast<int>(static_cast<long long>(x.vectors) * (part + 1) / parts);
  const uint4* body = x.body();
  // U vectors at a time, the next ones on their way; behind the share's end stand impossible tokens that are no alternatives
  const int rounds = (to - from + kThreads * U - 1) / (kThreads * U);
  uint4 raw[U];
  float highest = -INFINITY;
  unsigned bound = 0;
  int turn = 0;
  auto fetch = [&](int v) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * kThreads < to) raw[u] = __ldcs(body + v + u * kThreads);
  };
  int v = from + threadIdx.x;
  fetch(v);
  for (int i = 0; i < rounds; ++i, v += kThreads * U) {
    const int count = min(U, (to - v + kThreads - 1) / kThreads);   // vectors of this thread (may be negative: none)
    float f[U * E];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      unpack<T>(raw[u], f + u * E);
      if (u >= count)
#pragma unroll
        for (int j = 0; j < E; ++j) f[u * E + j] = -INFINITY;
    }
    if (i + 1 < rounds) fetch(v + kThreads * U);
    float top = max_nan(f[0], f[1]);
#pragma unroll
    for (int j = 2; j < U * E; j += 2) top = max3(top, f[j], f[j + 1]);
    st.add<U * E>(f, top);
    if (TOP) {
      // what is below the top_k-th of the threads' largest so far is no alternative; it is found anew when the number of rounds
      // has become fourfold: by then some 3 top_k values have passed the old one
      highest = max_nan(highest, top);
      if ((i & (i + 1)) == 0 && ((i + 1) & 0x55555555)) bound = max(bound, kth_of_threads(sm, highest, turn++, lane, top_k));
      const float limit = ordered(max(bound, *static_cast<volatile unsigned*>(&sm.bound)));
      if (__any_sync(0xffffffffu, !(top < limit))) {   // (NaN is the largest)
        unsigned may = 0;
#pragma unroll
        for (int j = 0; j < U * E; ++j) may |= j / E < count && !(f[j] < limit) ? 1u << j : 0u;
        const unsigned any = __reduce_or_sync(0xffffffffu, may);
        const unsigned long long before = best.last;
#pragma unroll
        for (int j = 0; j < U * E; ++j)
          if (any >> j & 1) best.offer_one(may >> j & 1, f[j], x.head + (v + j / E * kThreads) * E + j % E, lane, top_k);
        if (best.last != before && lane == 0) atomicMax(&sm.bound, static_cast<unsigned>(best.last >> 32));
      }
    }
  }
  if (part == parts - 1) {
    const int i = x.tail() + threadIdx.x;
    const float f = i < x.n ? to_float<T>(x.x[i]) : 0.f;
    if (i < x.n) st.add<1>(&f, f);
    if (TOP && warp == 0) best.offer_one(i < x.n, f, i, lane, top_k);
  }
  // the warp's, the CTA's, the cluster's
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) st.join(st.shuffle_xor(o));
  if (lane == 0) sm.stats[warp] = st;
  if (TOP) {
    if (lane < top_k) sm.best[warp * top_k + lane] = best.mine;
    if (warp == 0) sm.chosen[lane] = 0;
  }
  __syncthreads();
  if (TOP) {
    select_best(sm.best, kThreads / 32 * top_k, sm.chosen, top_k);
    __syncthreads();
  }
  if (warp == 0) {
    st = lane < kThreads / 32 ? sm.stats[lane] : Stats::none();
#pragma unroll
    for (int o = kThreads / 64; o > 0; o >>= 1) st.join(st.shuffle_xor(o));
  }
  if (parts > 1) {
    cluster.barrier_wait();
    Shared* to_first = cluster.map_shared_rank(&sm, 0);
    if (threadIdx.x == 0) to_first->part_stats[part] = st;
    if (TOP && static_cast<int>(threadIdx.x) < top_k) to_first->part_best[part * top_k + threadIdx.x] = sm.chosen[threadIdx.x];
    cluster.sync();
    if (part != 0) return;
    if (TOP) {
      if (warp == 0) sm.chosen[lane] = 0;
      __syncthreads();
      select_best(sm.part_best, parts * top_k, sm.chosen, top_k);
      __syncthreads();
    }
    if (warp == 0) {
      st = lane < parts ? sm.part_stats[lane] : Stats::none();
#pragma unroll
      for (int o = kMaxParts / 2; o > 0; o >>= 1) st.join(st.shuffle_xor(o));
    }
  }
  if (warp == 0) {   // (lane 0 has the sums of all)
    st.m = __shfl_sync(0xffffffffu, st.m, 0);
    st.s = __shfl_sync(0xffffffffu, st.s, 0);
    st.w = __shfl_sync(0xffffffffu, st.w, 0);
    const bool empty = st.s == 0.f;   // nothing in the row is possible
    const float log_s = log2f(st.s), ln_s = __fmul_rn(log_s, kLn2), lse = empty ? -INFINITY : st.m + ln_s;
    // from the largest logit, not from m + log S, whose rounding is 2^-24 of m: log S is never below 0, so this is never above it
    auto log_prob_of = [&](float f) { return empty ? -INFINITY : (f - st.m) - ln_s; };
    if (lane == 0) {
      if (a.log_sum_exp) a.log_sum_exp[row] = lse;
      if (a.log_sum_exp_rest) {   // the error of the sum m + ln_s, exact
        const float added = lse - st.m;
        a.log_sum_exp_rest[row] = isfinite(lse) ? (st.m - (lse - added)) + (ln_s - added) : 0.f;
      }
      if (a.entropy) a.entropy[row] = empty ? 0.f : (log_s - st.w / st.s) * kLn2;
      if (a.log_prob) a.log_prob[row] = token < 0 || token >= a.vocab ? 0.f : log_prob_of(chosen);
    }
    if (TOP && lane < top_k) {
      const unsigned long long key = sm.chosen[lane];
      if (a.top_tokens) a.top_tokens[row * top_k + lane] = 0xffffffffu - static_cast<unsigned>(key);
      if (a.top_log_probs) a.top_log_probs[row * top_k + lane] = log_prob_of(value_of(key));
    }
  }
}

// One CTA per share of a row.  The token and the alternatives are few: their logits are read before anything is written (the
// gradient may lie over the logits), and their elements written once more at the end.
//
// d x_i = p_i (sum of what does not go to single tokens - d_entropy (log p_i + entropy)) + what goes to token i.  A stream of one read
// and one write: 4096 rows of 128256 bf16 logits take 356 us (2.1 GB, 321 at the copy rate), 300 of 32000 fp16 10 us, of
// which beginning and ending are half.  Both kernels together 561 us, 1673 when they went element by element.
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) token_log_probs_grad_kernel(const ortb200_token_log_probs_grad_args a, int parts) {
  constexpr int E = Row<T>::E, U = 2;
  __shared__ long long at[kMaxTop + 1];
  __shared__ float gain[kMaxTop + 1];
  const long long row = blockIdx.x / parts;
  const int part = static_cast<int>(blockIdx.x % parts);
  pdl_wait_prior_grids();
  const Row<T> x(static_cast<const T*>(a.logits) + row * a.vocab, a.vocab);
  T* dx = static_cast<T*>(a.d_logits) + row * a.vocab;
  const float lse = a.log_sum_exp[row], rest = a.log_sum_exp_rest ? a.log_sum_exp_rest[row] : 0.f;
  const float g_h = a.d_entropy ? a.d_entropy[row] : 0.f, h = a.d_entropy ? a.entropy[row] : 0.f;
  const int special = 1 + a.top_k;
  if (static_cast<int>(threadIdx.x) < special) {
    const int k = static_cast<int>(threadIdx.x) - 1;
    const long long i = k < 0 ? a.tokens[row] : a.top_tokens[row * a.top_k + k];
    const bool in = i >= 0 && i < a.vocab;
    at[threadIdx.x] = in ? i : -1;
    gain[threadIdx.x] = !in ? 0.f : k < 0 ? (a.d_log_prob ? a.d_log_prob[row] : 0.f) : a.d_top_log_probs[row * a.top_k + k];
  }
  __syncthreads();
  float all = a.d_log_sum_exp ? a.d_log_sum_exp[row] : 0.f;
  for (int k = 0; k < special; ++k) all -= gain[k];
  const bool empty = lse == -INFINITY;   // nothing in the row is possible, and nothing changes that
  auto slope = [&](float v) {
    const float lp = (v - lse) - rest;
    // exp(-200) is 0 in 32 bits: below, the factor needs no more than a finite value (an impossible token has lp = -inf)
    return empty ? 0.f : exp_fast(lp) * (all - g_h * (fmaxf(lp, -200.f) + h));
  };
  // this share's elements: vectors [from, to), the head in the first and the tail in the last
  const int from = static_cast<int>(static_cast<long long>(x.vectors) * part / parts), to = static_cast<int>(static_cast<long long>(x.vectors) * (part + 1) / parts);
  const int first = part == 0 ? 0 : x.head + from * E, end = part == parts - 1 ? x.n : x.head + to * E;
  float kept = 0.f;
  bool own = false;
  if (static_cast<int>(threadIdx.x) < special) {
    const long long i = at[threadIdx.x];
    own = i >= first && i < end;
    if (own) {
      kept = slope(to_float<T>(x.x[i]));
      if (!empty)
        for (int k = 0; k < special; ++k)
          if (at[k] == i) kept += gain[k];
    }
  }
  __syncthreads();
  if (((reinterpret_cast<uintptr_t>(dx) ^ reinterpret_cast<uintptr_t>(x.x)) & 15) == 0) {
    const uint4* body = x.body();
    uint4* out = reinterpret_cast<uint4*>(dx + x.head);
    auto turn = [&](const uint4& raw) {
      float f[E];
      unpack<T>(raw, f);
      uint4 y;
      T* t = reinterpret_cast<T*>(&y);
#pragma unroll
      for (int e = 0; e < E; ++e) t[e] = from_float<T>(slope(f[e]));
      return y;
    };
    int v = from + threadIdx.x;
    for (; v + kThreads * (U - 1) < to; v += kThreads * U) {
      uint4 raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = __ldcs(body + v + u * kThreads);
#pragma unroll
      for (int u = 0; u < U; ++u) __stcs(out + v + u * kThreads, turn(raw[u]));
    }
    for (; v < to; v += kThreads) __stcs(out + v, turn(__ldcs(body + v)));
    if (part == 0 && static_cast<int>(threadIdx.x) < x.head) dx[threadIdx.x] = from_float<T>(slope(to_float<T>(x.x[threadIdx.x])));
    if (part == parts - 1 && x.tail() + static_cast<int>(threadIdx.x) < x.n) {
      const int i = x.tail() + threadIdx.x;
      dx[i] = from_float<T>(slope(to_float<T>(x.x[i])));
    }
  } else {   // the two rows start at different places between 16-byte boundaries
    for (int i = first + threadIdx.x; i < end; i += kThreads) dx[i] = from_float<T>(slope(to_float<T>(x.x[i])));
  }
  __syncthreads();
  if (own) dx[at[threadIdx.x]] = from_float<T>(kept);
}

// CTAs per row, a power of two: the least of waves x (3 us to begin and to join + the share at 16 KB a microsecond), which is what a
// CTA with its loads in flight reads when four of them share an SM.
int parts_of(int64_t rows, int64_t row_bytes) {
  int best = 1;
  double least = 1e30;
  for (int parts = 1; parts <= kMaxParts; parts *= 2) {
    const double waves = static_cast<double>((rows * parts + 4 * 148 - 1) / (4 * 148));
    const double t = waves * (3.0 + static_cast<double>(row_bytes) / parts / 16384.0);
    if (t < 0.98 * least) {
      least = t;
      best = parts;
    }
  }
  return best;
}

template <typename T, bool TOP>
int launch_log_probs(const ortb200_token_log_probs_args* a, cudaStream_t stream) {
  const int parts = parts_of(a->rows, static_cast<int64_t>(a->vocab) * sizeof(T));
  if (parts > 8 && cudaFuncSetAttribute(token_log_probs_kernel<T, TOP>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return -10;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a->rows * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = parts;
  attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = a->use_pdl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, token_log_probs_kernel<T, TOP>, *a) == cudaSuccess ? 0 : -11;
}

template <typename T>
int launch_log_probs(const ortb200_token_log_probs_args* a, cudaStream_t stream) {
  return a->top_k > 0 ? launch_log_probs<T, true>(a, stream) : launch_log_probs<T, false>(a, stream);
}

}  // namespace
}  // namespace ortb200

using namespace ortb200;

extern "C" int ortb200_token_log_probs_max_vocab(void) { return kMaxVocab; }

extern "C" int ortb200_token_log_probs(const ortb200_token_log_probs_args* a, ortb200_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!a || a->rows < 0 || a->vocab <= 0 || a->top_k < 0 || a->top_k > a->vocab) return -1;
  if (a->top_k > kMaxTop || a->rows > 0x0fffffffll || a->vocab > kMaxVocab) return -2;
  if (a->rows == 0) return 0;
  if (!a->logits || !a->tokens) return -1;
  switch (a->dtype) {
    case ORTB200_F16: return launch_log_probs<__half>(a, stream);
    case ORTB200_BF16: return launch_log_probs<__nv_bfloat16>(a, stream);
    case ORTB200_F32: return launch_log_probs<float>(a, stream);
  }
  return -4;
}

extern "C" int ortb200_token_log_probs_grad(const ortb200_token_log_probs_grad_args* a_, ortb200_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!a_) return -1;
  ortb200_token_log_probs_grad_args a = *a_;
  if (a.rows < 0 || a.vocab <= 0 || a.top_k < 0 || a.top_k > a.vocab) return -1;
  if (a.top_k > kMaxTop || a.rows > 0x0fffffffll || a.vocab > kMaxVocab) return -2;
  if (a.rows == 0) return 0;
  if (!a.logits || !a.tokens || !a.log_sum_exp || !a.d_logits || (a.d_entropy && !a.entropy) || (a.d_top_log_probs && !a.top_tokens)) return -1;
  if (!a.d_top_log_probs) a.top_k = 0;
  // shares of 8 KB at least, until there are eight CTAs for each SM
  const int64_t row_bytes = static_cast<int64_t>(a.vocab) * (a.dtype == ORTB200_F32 ? 4 : 2);
  const int64_t most = row_bytes / 8192 < 1 ? 1 : row_bytes / 8192, wanted = (8 * 148 + a.rows - 1) / a.rows;
  const int parts = static_cast<int>(wanted < most ? wanted : most);
  const dim3 grid(static_cast<unsigned>(a.rows * parts));
  switch (a.dtype) {
    case ORTB200_F16: return launch_kernel(token_log_probs_grad_kernel<__half>, grid, kThreads, 0, stream, a.use_pdl != 0, a, parts);
    case ORTB200_BF16: return launch_kernel(token_log_probs_grad_kernel<__nv_bfloat16>, grid, kThreads, 0, stream, a.use_pdl != 0, a, parts);
    case ORTB200_F32: return launch_kernel(token_log_probs_grad_kernel<float>, grid, kThreads, 0, stream, a.use_pdl != 0, a, parts);
  }
  return -4;
}
