// Log probabilities of given tokens, entropy and the best alternatives out of logits (com.ortb200.TokenLogProbs), and their
// gradient (com.ortb200.TokenLogProbsGrad).
//
// One CTA per row.  A thread keeps a running maximum m, S = sum exp(x - m) and W = sum exp(x - m) (x - m) of the logits it has
// seen; when the maximum moves from m to m', W becomes (W + S (m - m')) c and S becomes S c with c = exp(m - m').  Joined over
// the row: log_sum_exp = m + log S and entropy = log S - W / S.  All of it is held in 32 bits.
#include <cuda_runtime.h>
#include <math.h>
#include "launch_util.cuh"
#include "serving_ops.h"

namespace ortb200 {
namespace {

constexpr int kThreads = 256;

struct Stats {
  float m, s, w;
};
__device__ __forceinline__ void rescale(Stats& a, float m) {   // m >= a.m
  if (a.s == 0.f) {
    a.m = m;
    return;
  }
  const float d = a.m - m, c = expf(d);
  a.w = d == 0.f ? a.w : (a.w + a.s * d) * c;
  a.s *= c;
  a.m = m;
}
__device__ __forceinline__ void join(Stats& a, Stats b) {
  const float m = fmaxf(a.m, b.m);
  rescale(a, m);
  rescale(b, m);
  a.s += b.s;
  a.w += b.w;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_log_probs_kernel(const ortb200_token_log_probs_args a) {
  __shared__ Stats sm[kThreads / 32];
  __shared__ unsigned long long best[kThreads / 32];
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + row * a.vocab;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait_prior_grids();
  Stats st = {-INFINITY, 0.f, 0.f};
  for (int v = threadIdx.x; v < a.vocab; v += kThreads) {
    const float f = to_float<T>(x[v]);
    if (f > st.m) rescale(st, f);
    if (f != -INFINITY) {
      const float d = f - st.m, e = expf(d);
      st.s += e;
      st.w += e * d;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stats other = {__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.w, o)};
    join(st, other);
  }
  if (lane == 0) sm[warp] = st;
  __syncthreads();
  st = sm[0];
  for (int i = 1; i < kThreads / 32; ++i) join(st, sm[i]);
  const float log_s = logf(st.s), lse = st.s == 0.f ? -INFINITY : st.m + log_s;
  if (threadIdx.x == 0) {
    const long long tok = a.tokens[row];
    if (a.log_sum_exp) a.log_sum_exp[row] = lse;
    if (a.entropy) a.entropy[row] = st.s == 0.f ? 0.f : log_s - st.w / st.s;
    if (a.log_prob) {
      const bool in = tok >= 0 && tok < a.vocab;
      a.log_prob[row] = !in ? 0.f : st.s == 0.f ? -INFINITY : to_float<T>(x[tok]) - lse;
    }
  }
  // the alternatives one after another: the largest key below the last one; a key orders by value, then by lower index
  unsigned long long last = ~0ull;
  for (int k = 0; k < a.top_k; ++k) {
    unsigned long long top = 0;
    for (int v = threadIdx.x; v < a.vocab; v += kThreads) {
      const float f = to_float<T>(x[v]) + 0.f;   // -0 becomes 0: they are equal
      unsigned u = __float_as_uint(f);
      u = f != f ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
      const unsigned long long key = (static_cast<unsigned long long>(u) << 32) | (0xffffffffu - static_cast<unsigned>(v));
      if (key < last && key > top) top = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, top, o);
      top = other > top ? other : top;
    }
    __syncthreads();
    if (lane == 0) best[warp] = top;
    __syncthreads();
    for (int i = 0; i < kThreads / 32; ++i) top = best[i] > top ? best[i] : top;
    last = top;
    if (threadIdx.x == 0) {
      const unsigned v = 0xffffffffu - static_cast<unsigned>(top);
      if (a.top_tokens) a.top_tokens[row * a.top_k + k] = v;
      if (a.top_log_probs) a.top_log_probs[row * a.top_k + k] = st.s == 0.f ? -INFINITY : to_float<T>(x[v]) - lse;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_log_probs_grad_kernel(const ortb200_token_log_probs_grad_args a) {
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + row * a.vocab;
  T* dx = static_cast<T*>(a.d_logits) + row * a.vocab;
  pdl_wait_prior_grids();
  const long long tok = a.tokens[row];
  const float lse = a.log_sum_exp[row];
  const float g_lp = a.d_log_prob && tok >= 0 && tok < a.vocab ? a.d_log_prob[row] : 0.f;
  const float g_h = a.d_entropy ? a.d_entropy[row] : 0.f, h = a.d_entropy ? a.entropy[row] : 0.f;
  float top = 0.f;
  if (a.d_top_log_probs)
    for (int k = 0; k < a.top_k; ++k) top += a.d_top_log_probs[row * a.top_k + k];
  const float all = (a.d_log_sum_exp ? a.d_log_sum_exp[row] : 0.f) - g_lp - top;
  for (int v = threadIdx.x; v < a.vocab; v += kThreads) {
    const float lp = to_float<T>(x[v]) - lse;
    float d = 0.f;
    if (lse != -INFINITY) {
      if (lp != -INFINITY) d = expf(lp) * (all - g_h * (lp + h));
      if (v == tok) d += g_lp;
      if (a.d_top_log_probs)
        for (int k = 0; k < a.top_k; ++k)
          if (a.top_tokens[row * a.top_k + k] == v) d += a.d_top_log_probs[row * a.top_k + k];
    }
    dx[v] = from_float<T>(d);
  }
}

}  // namespace
}  // namespace ortb200

using namespace ortb200;

extern "C" int ortb200_token_log_probs(const ortb200_token_log_probs_args* a, ortb200_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!a || a->rows < 0 || a->vocab <= 0 || a->top_k < 0 || a->top_k > a->vocab) return -1;
  if (a->top_k > 32 || a->rows > 0x7fffffffll) return -2;
  if (a->rows == 0) return 0;
  if (!a->logits || !a->tokens) return -1;
  const dim3 grid(static_cast<unsigned>(a->rows));
  switch (a->dtype) {
    case ORTB200_F16: return launch_kernel(token_log_probs_kernel<__half>, grid, kThreads, 0, stream, a->use_pdl != 0, *a);
    case ORTB200_BF16: return launch_kernel(token_log_probs_kernel<__nv_bfloat16>, grid, kThreads, 0, stream, a->use_pdl != 0, *a);
    case ORTB200_F32: return launch_kernel(token_log_probs_kernel<float>, grid, kThreads, 0, stream, a->use_pdl != 0, *a);
  }
  return -4;
}

extern "C" int ortb200_token_log_probs_grad(const ortb200_token_log_probs_grad_args* a, ortb200_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!a || a->rows < 0 || a->vocab <= 0 || a->top_k < 0 || a->top_k > a->vocab) return -1;
  if (a->top_k > 32 || a->rows > 0x7fffffffll) return -2;
  if (a->rows == 0) return 0;
  if (!a->logits || !a->tokens || !a->log_sum_exp || !a->d_logits || (a->d_entropy && !a->entropy) || (a->d_top_log_probs && !a->top_tokens)) return -1;
  const dim3 grid(static_cast<unsigned>(a->rows));
  switch (a->dtype) {
    case ORTB200_F16: return launch_kernel(token_log_probs_grad_kernel<__half>, grid, kThreads, 0, stream, a->use_pdl != 0, *a);
    case ORTB200_BF16: return launch_kernel(token_log_probs_grad_kernel<__nv_bfloat16>, grid, kThreads, 0, stream, a->use_pdl != 0, *a);
    case ORTB200_F32: return launch_kernel(token_log_probs_grad_kernel<float>, grid, kThreads, 0, stream, a->use_pdl != 0, *a);
  }
  return -4;
}
