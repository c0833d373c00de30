// Penalties for repeated tokens, biases, masks and temperatures on logits (com.ortb200.ProcessLogits).
//
// Every logit is read once and every score written once.  A CTA has a chunk of a row's vocabulary, with a counter per token in shared
// memory, and three passes: it reads the row's whole text and counts the tokens of its chunk; it streams the chunk through
// mask and temperature, which asks nothing of the counters; then it works the counted tokens out again, few of the chunk, and
// last the biased ones.  No CTA waits for another, and counting commutes: no result depends on an order of arrival.
#include <cuda_runtime.h>
#include <math.h>
#include "draft_ops.h"
#include "launch_util.cuh"

namespace ortb200 {
namespace {

constexpr int kThreads = 512;
constexpr int kMaxChunk = 16384;      // counters of a CTA: 64 KB, three CTAs to an SM
constexpr int kMaxVocab = 0x7fff0000; // an index plus the tokens of a pass fits 31 bits
constexpr unsigned kSeen = 0x80000000u, kBiased = 0x40000000u, kCount = 0x3fffffffu;

// What a row asks for besides its text.
struct RowRules {
  float repetition, presence, frequency, temperature;
  const unsigned* mask;
  long long bias0, bias1;
};
__device__ __forceinline__ RowRules rules_of(const ortb200_process_logits_args& a, long long r, bool report) {
  RowRules q;
  q.repetition = a.repetition ? a.repetition[r] : 1.f;
  q.presence = a.presence ? a.presence[r] : 0.f;
  q.frequency = a.frequency ? a.frequency[r] : 0.f;
  q.temperature = a.temperature ? a.temperature[r] : 1.f;
  if (!(q.temperature > 0.f)) q.temperature = 1.f;
  q.mask = nullptr;
  bool bad = false;
  if (a.allowed) {
    const int m = a.row_mask[r];
    if (m >= a.masks) bad = true;
    else if (m >= 0) q.mask = reinterpret_cast<const unsigned*>(a.allowed) + static_cast<long long>(m) * a.mask_words;
  }
  q.bias0 = q.bias1 = 0;
  if (a.bias_tokens) {
    q.bias0 = a.bias_starts[r];
    q.bias1 = a.bias_starts[r + 1];
    if (q.bias0 < 0 || q.bias1 < q.bias0 || q.bias1 > a.bias_len) {
      bad = true;
      q.bias0 = q.bias1 = 0;
    }
  }
  if (bad && report && a.status) atomicExch(a.status, kStatusBadArgument);
  return q;
}
__device__ __forceinline__ float penalised(const RowRules& q, float x, unsigned word) {
  if (word & ~kBiased) {   // somewhere in the text
    x = x < 0.f ? x * q.repetition : x / q.repetition;
    const unsigned c = word & kCount;
    if (c) x -= q.frequency * static_cast<float>(c) + q.presence;
  }
  return x;
}
__device__ __forceinline__ float finished(const RowRules& q, float x, bool allowed) {
  if (q.temperature != 1.f) x = x / q.temperature;
  return allowed ? x : -INFINITY;
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float* f) {
  const T* t = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < 16 / static_cast<int>(sizeof(T)); ++i) f[i] = to_float<T>(t[i]);
}

// E: logits of a vector (1: any alignment).  TEXT: rows may have texts.
template <typename T, int E, bool TEXT>
__global__ void __launch_bounds__(kThreads, 3) process_logits_kernel(const ortb200_process_logits_args a, const int chunk, const int parts) {
  extern __shared__ __align__(16) unsigned counts[];   // [chunk + 2 E]: a row's first tokens may lie in front of the first vector, its last ones behind the last
  const int part = static_cast<int>(blockIdx.x % parts);
  const long long r = blockIdx.x / parts;
  pdl_wait_prior_grids();
  const T* x = static_cast<const T*>(a.logits) + r * a.vocab;
  float* y = a.scores + r * a.vocab;
  // the row's vectors start at the first token whose place in the tensor E divides; what is in front of them is the first CTA's
  const int lead = E == 1 ? 0 : min(static_cast<int>((E - r * a.vocab % E) % E), a.vocab);
  const int tail = lead + (a.vocab - lead) / E * E;                   // the last tokens, fewer than a vector: the CTA's that has what is in front of them
  const int tail_part = tail > lead ? (tail - lead - 1) / chunk : 0;
  const int body0 = lead + part * chunk, body1 = min(body0 + chunk, tail), vectors = max(body1 - body0, 0) / E;   // the chunk
  const int first = part == 0 ? 0 : body0, end = part == tail_part ? a.vocab : part < tail_part ? body1 : first;  // with what is left over
  const int base = body0 - E;                                         // the token of counter 0
  const RowRules q = rules_of(a, r, part == 0 && threadIdx.x == 0);

  bool text = false;
  if constexpr (TEXT) {
    long long h0 = 0, h1 = 0, counted = 0;
    const bool asks = q.repetition != 1.f || q.presence != 0.f || q.frequency != 0.f;
    if (asks && a.history) {
      const long long l = a.row_list ? a.row_list[r] : r;
      bool bad = l >= a.lists;
      if (l >= 0 && !bad) {
        h0 = a.history_starts[l];
        h1 = a.history_starts[l + 1];
        bad = h0 < 0 || h1 < h0 || h1 > a.history_len;
        if (bad) h0 = h1 = 0;
        counted = a.generated_starts ? a.generated_starts[l] : h0;
      }
      if (bad && part == 0 && threadIdx.x == 0 && a.status) atomicExch(a.status, kStatusBadArgument);
    }
    const int drafted = asks && a.drafted ? a.drafted_width : 0;
    text = h1 > h0 || drafted > 0;
    if (text) {
      for (int i = threadIdx.x; i < (chunk + 2 * E + 3) / 4; i += kThreads) reinterpret_cast<uint4*>(counts)[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      const unsigned size = static_cast<unsigned>(end - first);
      auto add = [&](long long v, bool count) {
        const unsigned long long at = static_cast<unsigned long long>(v - first);
        if (at >= size) return;
        unsigned* to = counts + (first - base) + static_cast<unsigned>(at);
        if (count) atomicAdd(to, 1u);
        else atomicOr(to, kSeen);
      };
      // two tokens to a load, four loads of a thread on their way
      constexpr int kAhead = 4;
      const long long odd = min(h0 + static_cast<long long>((reinterpret_cast<uintptr_t>(a.history + h0) >> 3) & 1), h1), pairs = (h1 - odd) / 2;
      if (threadIdx.x == 0 && odd > h0) add(a.history[h0], h0 >= counted);
      if (threadIdx.x == 32 && odd + 2 * pairs < h1) add(a.history[h1 - 1], h1 - 1 >= counted);
      const longlong2* two = reinterpret_cast<const longlong2*>(a.history + odd);
      long long i = threadIdx.x;
      for (; i + (kAhead - 1) * kThreads < pairs; i += kAhead * kThreads) {
        longlong2 v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) v[k] = __ldg(two + i + k * kThreads);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const long long at = odd + 2 * (i + k * kThreads);
          add(v[k].x, at >= counted);
          add(v[k].y, at + 1 >= counted);
        }
      }
      for (; i < pairs; i += kThreads) {
        const longlong2 v = __ldg(two + i);
        add(v.x, odd + 2 * i >= counted);
        add(v.y, odd + 2 * i + 1 >= counted);
      }
      for (int d = threadIdx.x; d < drafted; d += kThreads) add(a.drafted[r * a.drafted_width + d], true);
    }
  }

  // ------------------------------------------------------------------------------------------------------ the chunk's vectors
  auto allowed = [&](int v) { return !q.mask || (__ldg(q.mask + (v >> 5)) >> (v & 31) & 1); };
  constexpr int kAhead = E == 1 ? 8 : 4;
  for (int i0 = 0; i0 < vectors; i0 += kAhead * kThreads) {
    T one[E == 1 ? kAhead : 1];
    uint4 many[E == 1 ? 1 : kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int at = i0 + i * kThreads + threadIdx.x;
      if (at < vectors) {
        if constexpr (E == 1) one[i] = x[body0 + at];
        else many[i] = __ldg(reinterpret_cast<const uint4*>(x + body0) + at);
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int at = i0 + i * kThreads + threadIdx.x, v = body0 + at * E;
      if (at >= vectors) continue;
      if constexpr (E == 1) {
        y[v] = finished(q, to_float<T>(one[i]), allowed(v));
      } else {
        float f[E];
        unpack<T>(many[i], f);
        if (q.temperature != 1.f)   // in front of the mask: infinities take the long way through a division (18 instead of 5 us for 150 rows of 32000)
#pragma unroll
          for (int e = 0; e < E; ++e) f[e] = f[e] / q.temperature;
        if (q.mask) {   // E bits from bit v on; they may lie in two words
          const int w0 = v >> 5, w1 = (v + E - 1) >> 5;
          const unsigned lo = __ldg(q.mask + w0), hi = w1 != w0 ? __ldg(q.mask + w1) : 0u, bits = __funnelshift_r(lo, hi, v & 31);
#pragma unroll
          for (int e = 0; e < E; ++e) f[e] = bits >> e & 1 ? f[e] : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < E; e += 4) __stcs(reinterpret_cast<float4*>(y + v + e), make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]));
      }
    }
  }
  auto whole = [&](int v, unsigned word, float bias) { y[v] = finished(q, penalised(q, to_float<T>(x[v]), word) + bias, allowed(v)); };
  if (E > 1) {
    if (part == 0 && static_cast<int>(threadIdx.x) < lead) whole(threadIdx.x, 0u, 0.f);
    if (part == tail_part && static_cast<int>(threadIdx.x) < a.vocab - tail) whole(tail + threadIdx.x, 0u, 0.f);
  }
  if (text) {   // ----------------------------------------------------------------------------------------------------- the text's tokens
    __syncthreads();
    const int last = end - base;
    for (int i = 4 * threadIdx.x; i < last; i += 4 * kThreads) {
      const uint4 w = *reinterpret_cast<const uint4*>(counts + i);
      if (w.x) whole(base + i, w.x, 0.f);
      if (w.y) whole(base + i + 1, w.y, 0.f);
      if (w.z) whole(base + i + 2, w.z, 0.f);
      if (w.w) whole(base + i + 3, w.w, 0.f);
    }
  }

  // --------------------------------------------------------------------------------------------------------------- biases
  // A token's flag tells whether it has several: who finds it set has come second.  Without a text only the counters of biased tokens
  // are in use.
  if (q.bias1 > q.bias0) {
    __shared__ int twice;
    auto mine = [&](long long b) -> int {   // the counter of a bias's token, -1 where it is another CTA's or none
      const long long v = a.bias_tokens[b];
      return v >= first && v < end ? static_cast<int>(v) - base : -1;
    };
    if (threadIdx.x == 0) twice = 0;
    if (!text)
      for (long long b = q.bias0 + threadIdx.x; b < q.bias1; b += kThreads) {
        const int at = mine(b);
        if (at >= 0) counts[at] = 0;
      }
    __syncthreads();   // also: the passes above have written what is written again here
    for (long long b = q.bias0 + threadIdx.x; b < q.bias1; b += kThreads) {
      const int at = mine(b);
      if (at < 0) continue;
      const unsigned word = atomicOr(&counts[at], kBiased);
      if (word & kBiased) twice = 1;   // (whoever writes, writes the same)
      else whole(base + at, word, a.bias_values[b]);
    }
    __syncthreads();
    if (twice)   // rare: every bias looks for others of its token, and the first of several sums them up in their order
      for (long long b = q.bias0 + threadIdx.x; b < q.bias1; b += kThreads) {
        const int at = mine(b);
        if (at < 0) continue;
        const long long t = base + at;
        bool leads = true, several = false;
        for (long long o = q.bias0; o < b && leads; ++o) leads = a.bias_tokens[o] != t;
        if (!leads) continue;
        float sum = a.bias_values[b];
        for (long long o = b + 1; o < q.bias1; ++o)
          if (a.bias_tokens[o] == t) {
            sum += a.bias_values[o];
            several = true;
          }
        if (several) whole(base + at, counts[at], sum);
      }
  }
}

template <typename T, int E, bool TEXT>
int launch(const ortb200_process_logits_args* a, cudaStream_t stream) {
  // Short chunks where rows are few, so that every SM has some; but a text is read once for each chunk, so not beyond where the usual text
  // is as many bytes as the chunk.
  const int64_t text = TEXT && a->history && a->lists > 0 ? 8 * (a->history_len / a->lists) : 0;
  int chunk = kMaxChunk;
  while (chunk > 2048 && a->rows * ((a->vocab + chunk - 1) / chunk) < 3 * 148 && text <= chunk / 2 * static_cast<int64_t>(sizeof(T) + 4)) chunk /= 2;
  const long long parts = (a->vocab + chunk - 1) / chunk;
  if (a->rows * parts > 0x7fffffffll) return -2;
  const int smem = TEXT || a->bias_tokens ? (chunk + 2 * E + 4) * 4 : 0;
  auto kern = process_logits_kernel<T, E, TEXT>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (kMaxChunk + 64) * 4) != cudaSuccess) return -10;   // per device
  return launch_kernel(kern, dim3(static_cast<unsigned>(a->rows * parts)), kThreads, smem, stream, a->use_pdl != 0, *a, chunk, static_cast<int>(parts));
}

template <typename T>
int launch_type(const ortb200_process_logits_args* a, cudaStream_t stream) {
  constexpr int E = 16 / sizeof(T);
  const bool aligned = ((reinterpret_cast<uintptr_t>(a->logits) | reinterpret_cast<uintptr_t>(a->scores)) & 15) == 0;
  const bool text = a->history || a->drafted;
  if (aligned) return text ? launch<T, E, true>(a, stream) : launch<T, E, false>(a, stream);
  return text ? launch<T, 1, true>(a, stream) : launch<T, 1, false>(a, stream);
}

}  // namespace
}  // namespace ortb200

using namespace ortb200;

extern "C" int ortb200_process_logits_max_vocab(void) { return kMaxVocab; }

extern "C" int ortb200_process_logits(const ortb200_process_logits_args* a, ortb200_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!a || a->rows < 0 || a->vocab <= 0 || a->history_len < 0 || a->bias_len < 0 || a->lists < 0 || a->drafted_width < 0 || a->masks < 0) return -1;
  if (a->rows == 0) return 0;
  if (!a->logits || !a->scores) return -1;
  if (a->history && !a->history_starts) return -1;
  if (a->bias_tokens && (!a->bias_values || !a->bias_starts)) return -1;
  if (a->allowed && (!a->row_mask || a->mask_words < (a->vocab + 31) / 32)) return -1;
  if (a->vocab > kMaxVocab || a->history_len + a->drafted_width > kCount) return -2;   // (a count has 30 bits)
  switch (a->dtype) {
    case ORTB200_F16: return launch_type<__half>(a, stream);
    case ORTB200_BF16: return launch_type<__nv_bfloat16>(a, stream);
    case ORTB200_F32: return launch_type<float>(a, stream);
  }
  return -4;
}
