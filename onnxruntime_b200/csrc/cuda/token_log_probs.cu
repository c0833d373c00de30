// Log probabilities of given tokens, entropy and the best alternatives out of logits (com.ortb200.TokenLogProbs), and their
// gradient (com.ortb200.TokenLogProbsGrad).
//
// One pass over a row.  A thread keeps a running maximum m, S = sum exp(x - m) and W = sum exp(x - m) (x - m) of the logits it has
// seen; when the maximum moves from m to m', W becomes (W + S (m - m')) c and S becomes S c with c = exp(m - m').  Joined over
// the row: log_sum_exp = m + log S and entropy = log S - W / S.  All of it is held in 32 bits.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <math.h>
#include "launch_util.cuh"
#include "serving_ops.h"

namespace ortb200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kMaxTop = 32;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp_fast(float d) {   // relative error 2^-22 + |d| 2^-23: what is far below the maximum weighs little
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(d * kLog2e));
  return e;
}

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

struct Stats {
  float m, s, w;
  __device__ __forceinline__ void raise(float to) {   // to >= m
    if (s != 0.f) {
      const float d = m - to, c = expf(d);
      w = d == 0.f ? w : (w + s * d) * c;
      s *= c;
    }
    m = to;
  }
  template <int N>
  __device__ __forceinline__ void add(const float* x) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
    if (top > m) raise(top);
    const float ref = m == -INFINITY ? 0.f : m;
    float s0 = 0.f, s1 = 0.f, w0 = 0.f, w1 = 0.f;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float d0 = x[i] - ref, e0 = exp_fast(d0);
      s0 += e0;
      w0 = fmaf(e0, fmaxf(d0, -1e30f), w0);   // an impossible token: 0 times -inf counts as 0
      if (i + 1 < N) {
        const float d1 = x[i + 1] - ref, e1 = exp_fast(d1);
        s1 += e1;
        w1 = fmaf(e1, fmaxf(d1, -1e30f), w1);
      }
    }
    s += s0 + s1;
    w += w0 + w1;
  }
  __device__ __forceinline__ void join(Stats b) {
    const float to = fmaxf(m, b.m);
    raise(to);
    b.raise(to);
    s += b.s;
    w += b.w;
  }
};

// The 32 best (value, index) pairs a warp has seen, lane i the i-th best.  A key orders by value, then by lower index; zeros of both
// signs are equal, NaN is the largest.
__device__ __forceinline__ unsigned long long key_of(float f, int index) {
  f += 0.f;
  const unsigned u = __float_as_uint(f);
  const unsigned order = f != f ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return (static_cast<unsigned long long>(order) << 32) | (0xffffffffu - static_cast<unsigned>(index));
}
__device__ __forceinline__ float value_of(unsigned long long key) {
  const unsigned order = static_cast<unsigned>(key >> 32);
  return __uint_as_float((order & 0x80000000u) ? order & 0x7fffffffu : ~order);
}
struct Best {
  unsigned long long mine = 0;     // this lane's pair; 0: none
  unsigned long long last = 0;     // the top_k-th: what is not above it is no alternative
  float limit = -INFINITY;         // its value
  __device__ __forceinline__ void insert(unsigned long long key, int lane, int top_k) {
    const int above = __popc(__ballot_sync(0xffffffffu, mine > key));
    const unsigned long long up = __shfl_up_sync(0xffffffffu, mine, 1);
    if (lane > above) mine = up;
    if (lane == above) mine = key;
    last = __shfl_sync(0xffffffffu, mine, top_k - 1);
    limit = value_of(last);
  }
  // one pair of every lane (0: none)
  __device__ __forceinline__ void offer(unsigned long long key, int lane, int top_k) {
    for (unsigned left = __ballot_sync(0xffffffffu, key > last); left != 0; left &= left - 1) {
      const unsigned long long k = __shfl_sync(0xffffffffu, key, __ffs(left) - 1);
      if (k > last) insert(k, lane, top_k);
    }
  }
  // x[0 .. N) of every lane, of which those below `count` exist, at index, index + 1 ...; all of them come behind what was offered before, so that a
  // value equal to the limit is no alternative
  template <int N>
  __device__ __forceinline__ void offer_all(const float* x, int index, int count, int lane, int top_k) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < N; ++i) any |= i < count && !(x[i] <= limit);
    if (!__any_sync(0xffffffffu, any || (last == 0 && count > 0))) return;
#pragma unroll
    for (int i = 0; i < N; ++i) offer(i < count ? key_of(x[i], index + i) : 0, lane, top_k);
  }
};

struct Shared {
  Stats stats[kThreads / 32];
  unsigned long long best[kThreads / 32][kMaxTop];
  Stats joined;                        // of the CTA
  unsigned long long joined_best[kMaxTop];
};

// A cluster of CTAs per row, each with a share of its vectors; the first CTA puts the shares together over distributed shared memory.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, TOP ? 3 : 4) token_log_probs_kernel(const ortb200_token_log_probs_args a) {
  constexpr int E = Row<T>::E, U = TOP ? 2 : 4;
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
  Stats st = {-INFINITY, 0.f, 0.f};
  Best best;
  if (part == 0) {   // the elements in front of the first vector: fewer than a warp
    const bool has = static_cast<int>(threadIdx.x) < x.head;
    const float f = has ? to_float<T>(x.x[threadIdx.x]) : 0.f;
    if (has) st.add<1>(&f);
    if (TOP && warp == 0) best.offer_all<1>(&f, threadIdx.x, has ? 1 : 0, lane, top_k);
  }
  const int from = static_cast<int>(static_cast<long long>(x.vectors) * part / parts), to = static_cast<int>(static_cast<long long>(x.vectors) * (part + 1) / parts);
  const uint4* body = x.body();
  int v = from + threadIdx.x;
  const int whole = from + (to - from) / (kThreads * U) * (kThreads * U);
  for (; v < whole; v += kThreads * U) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = __ldcs(body + v + u * kThreads);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[E];
      unpack<T>(raw[u], f);
      st.add<E>(f);
      if (TOP) best.offer_all<E>(f, x.head + (v + u * kThreads) * E, E, lane, top_k);
    }
  }
  for (int v0 = whole; v0 < to; v0 += kThreads) {   // (all threads: alternatives are offered by whole warps)
    v = v0 + threadIdx.x;
    float f[E];
    if (v < to) {
      unpack<T>(__ldcs(body + v), f);
      st.add<E>(f);
    }
    if (TOP) best.offer_all<E>(f, x.head + v * E, v < to ? E : 0, lane, top_k);
  }
  if (part == parts - 1) {
    const int i = x.tail() + threadIdx.x;
    const float f = i < x.n ? to_float<T>(x.x[i]) : 0.f;
    if (i < x.n) st.add<1>(&f);
    if (TOP && warp == 0) best.offer_all<1>(&f, i, i < x.n ? 1 : 0, lane, top_k);
  }
  // the warp's, the CTA's, the cluster's
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) st.join({__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.w, o)});
  if (lane == 0) sm.stats[warp] = st;
  if (TOP) sm.best[warp][lane] = lane < top_k ? best.mine : 0;
  __syncthreads();
  if (warp == 0) {
    st = sm.stats[0];
    for (int i = 1; i < kThreads / 32; ++i) st.join(sm.stats[i]);
    if (TOP)
      for (int i = 1; i < kThreads / 32; ++i) best.offer(sm.best[i][lane], lane, top_k);
    if (parts > 1) {
      if (lane == 0) sm.joined = st;
      if (TOP) sm.joined_best[lane] = lane < top_k ? best.mine : 0;
    }
  }
  if (parts > 1) {
    cluster.sync();
    if (part == 0 && warp == 0) {
      for (int c = 1; c < parts; ++c) {
        const Shared* other = cluster.map_shared_rank(&sm, c);
        st.join(other->joined);
        if (TOP) best.offer(other->joined_best[lane], lane, top_k);
      }
    }
  }
  if (part == 0 && warp == 0) {
    const bool empty = st.s == 0.f;   // nothing in the row is possible
    const float log_s = logf(st.s), lse = empty ? -INFINITY : st.m + log_s;
    if (lane == 0) {
      if (a.log_sum_exp) a.log_sum_exp[row] = lse;
      if (a.entropy) a.entropy[row] = empty ? 0.f : log_s - st.w / st.s;
      if (a.log_prob) a.log_prob[row] = token < 0 || token >= a.vocab ? 0.f : empty ? -INFINITY : chosen - lse;
    }
    if (TOP && lane < top_k) {
      const unsigned index = 0xffffffffu - static_cast<unsigned>(best.mine);
      if (a.top_tokens) a.top_tokens[row * top_k + lane] = index;
      if (a.top_log_probs) a.top_log_probs[row * top_k + lane] = empty ? -INFINITY : value_of(best.mine) - lse;
    }
  }
  if (parts > 1) cluster.sync();   // no CTA leaves while its shared memory is read
}

// One CTA per share of a row.  The token and the alternatives are few: their logits are read before anything is written (the
// gradient may lie over the logits), and their elements written once more at the end.
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
  const float lse = a.log_sum_exp[row];
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
    const float lp = v - lse;
    return empty ? 0.f : exp_fast(lp) * (all - g_h * (fmaxf(lp, -1e30f) + h));   // an impossible token: 0 times -inf counts as 0
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

// CTAs per row: enough for four on each SM while a share keeps some thousand logits
int parts_of(int64_t rows, int vocab, int most) {
  int parts = 1;
  while (parts < most && rows * parts < 4 * 148 && vocab / (2 * parts) >= 2048) parts *= 2;
  return parts;
}

template <typename T, bool TOP>
int launch_log_probs(const ortb200_token_log_probs_args* a, cudaStream_t stream) {
  const int parts = parts_of(a->rows, a->vocab, 8);
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

extern "C" int ortb200_token_log_probs(const ortb200_token_log_probs_args* a, ortb200_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!a || a->rows < 0 || a->vocab <= 0 || a->top_k < 0 || a->top_k > a->vocab) return -1;
  if (a->top_k > kMaxTop || a->rows > 0x0fffffffll) return -2;
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
  if (a.top_k > kMaxTop || a.rows > 0x0fffffffll) return -2;
  if (a.rows == 0) return 0;
  if (!a.logits || !a.tokens || !a.log_sum_exp || !a.d_logits || (a.d_entropy && !a.entropy) || (a.d_top_log_probs && !a.top_tokens)) return -1;
  if (!a.d_top_log_probs) a.top_k = 0;
  const int parts = parts_of(a.rows, a.vocab, 8);
  const dim3 grid(static_cast<unsigned>(a.rows * parts));
  switch (a.dtype) {
    case ORTB200_F16: return launch_kernel(token_log_probs_grad_kernel<__half>, grid, kThreads, 0, stream, a.use_pdl != 0, a, parts);
    case ORTB200_BF16: return launch_kernel(token_log_probs_grad_kernel<__nv_bfloat16>, grid, kThreads, 0, stream, a.use_pdl != 0, a, parts);
    case ORTB200_F32: return launch_kernel(token_log_probs_grad_kernel<float>, grid, kThreads, 0, stream, a.use_pdl != 0, a, parts);
  }
  return -4;
}
