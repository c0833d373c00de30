// Penalties for repeated tokens, biases, masks and temperatures on logits (com.ortb200.ProcessLogits).
//
// Every logit is read once and every score written once; what a row's text asks of them has to be known by then.  A cluster of
// CTAs has a row, each CTA a chunk of the vocabulary with a counter per token in shared memory.  The CTAs share the row's text among
// them, too: each reads a part and adds to the counters of whichever CTA has the token (a text of 60,000 tokens, read by all eight, would
// be as many bytes as the row's logits seven times over).  Counting commutes: no result depends on the order.
// The first logits of every thread are on their way while the text is counted.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <math.h>
#include "draft_ops.h"
#include "launch_util.cuh"

namespace ortb200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kChunk = 16384;         // tokens of a CTA where eight CTAs hold the vocabulary
constexpr int kMaxChunk = 56 * 1024;  // where they do not: counters that fit shared memory
constexpr int kMaxCluster = 8;
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
  if (!allowed) x = -INFINITY;
  return q.temperature != 1.f ? x / q.temperature : x;
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float* f) {
  const T* t = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < 16 / static_cast<int>(sizeof(T)); ++i) f[i] = to_float<T>(t[i]);
}

// E: logits of a vector (1: any alignment).  COUNTS: rows may have texts or biases; without, nothing but masks and temperatures.
template <typename T, int E, bool COUNTS>
__global__ void __launch_bounds__(kThreads) process_logits_kernel(const ortb200_process_logits_args a, const int chunk) {
  extern __shared__ unsigned counts[];   // [chunk + E]: of the chunk's tokens; a row's first tokens may lie in front of the first vector
  constexpr int kAhead = E == 1 ? 8 : 4;
  const cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const long long r = blockIdx.x / parts;
  pdl_wait_prior_grids();
  const T* x = static_cast<const T*>(a.logits) + r * a.vocab;
  float* y = a.scores + r * a.vocab;
  // the row's vectors start at the first token whose place in the tensor E divides: the tokens in front of it are the first CTA's
  const int lead = E == 1 ? 0 : min(static_cast<int>((E - r * a.vocab % E) % E), a.vocab);
  const int body0 = lead + part * chunk;                              // the chunk: tokens [body0, body1) in vectors, and what is left over
  const int body1 = static_cast<int>(min(static_cast<long long>(body0) + chunk, static_cast<long long>(lead + (a.vocab - lead) / E * E)));
  const int vectors = body1 > body0 ? (body1 - body0) / E : 0;
  const int tail = lead + (a.vocab - lead) / E * E;                   // the last tokens, fewer than a vector: the CTA's that has what is in front of them
  const int tail_part = tail > lead ? (tail - lead - 1) / chunk : 0;
  auto word_at = [&](int v) -> unsigned { return COUNTS ? counts[v - body0 + E] : 0u; };

  T ahead1[E == 1 ? kAhead : 1];
  uint4 ahead[E == 1 ? 1 : kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int at = i * kThreads + threadIdx.x;
    if (at < vectors) {
      if constexpr (E == 1) ahead1[i] = x[body0 + at];
      else ahead[i] = __ldcs(reinterpret_cast<const uint4*>(x + body0) + at);
    }
  }
  const RowRules q = rules_of(a, r, part == 0 && threadIdx.x == 0);
  bool listed = false;
  __shared__ int twice;
  if constexpr (COUNTS) {
    // ------------------------------------------------------------------------------------------ the row's text and biases
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
    listed = h1 > h0 || drafted > 0 || q.bias1 > q.bias0;
    if (threadIdx.x == 0) twice = 0;
    if (listed) {   // the same for all of a cluster
      for (int i = threadIdx.x; i < chunk + 2 * E; i += kThreads) counts[i] = 0;
      cluster.sync();
      const unsigned mine = smem_u32(counts);
      auto place = [&](long long v) -> unsigned {   // of a token's counter, in whichever CTA has it
        const int t = static_cast<int>(v), owner = t < lead ? 0 : t >= tail ? tail_part : (t - lead) / chunk;
        unsigned there;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(mine + static_cast<unsigned>(t - (lead + owner * chunk) + E) * 4u), "r"(owner));
        return there;
      };
      auto add = [&](long long v, bool count) {
        if (v < 0 || v >= a.vocab) return;
        if (count) asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(place(v)), "r"(1u) : "memory");
        else asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(place(v)), "r"(kSeen) : "memory");
      };
      const long long all = static_cast<long long>(parts) * kThreads;
      long long i = h0 + static_cast<long long>(part) * kThreads + threadIdx.x;
      for (; i + 3 * all < h1; i += 4 * all) {
        long long v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = a.history[i + k * all];
#pragma unroll
        for (int k = 0; k < 4; ++k) add(v[k], i + k * all >= counted);
      }
      for (; i < h1; i += all) add(a.history[i], i >= counted);
      if (part == 0)
        for (int d = threadIdx.x; d < drafted; d += kThreads) add(a.drafted[r * a.drafted_width + d], true);
      for (long long b = q.bias0 + static_cast<long long>(part) * kThreads + threadIdx.x; b < q.bias1; b += all) {
        const long long v = a.bias_tokens[b];
        if (v >= 0 && v < a.vocab) asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(place(v)), "r"(kBiased) : "memory");
      }
      cluster.sync();
    }
  }

  // ------------------------------------------------------------------------------------------------------ the chunk's vectors
  for (int i0 = 0; i0 * kThreads < vectors; i0 += kAhead) {
    if (i0 > 0) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int at = (i0 + i) * kThreads + threadIdx.x;
        if (at < vectors) {
          if constexpr (E == 1) ahead1[i] = x[body0 + at];
          else ahead[i] = __ldcs(reinterpret_cast<const uint4*>(x + body0) + at);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int at = (i0 + i) * kThreads + threadIdx.x, v = body0 + at * E;
      if (at >= vectors) continue;
      float f[E];
      if constexpr (E == 1) f[0] = to_float<T>(ahead1[i]);
      else unpack<T>(ahead[i], f);
      if (COUNTS && listed) {
        unsigned w[E], any = 0;
        if constexpr (E == 1) {
          w[0] = word_at(v);
        } else {
#pragma unroll
          for (int e = 0; e < E; e += 4) *reinterpret_cast<uint4*>(w + e) = *reinterpret_cast<const uint4*>(counts + v - body0 + E + e);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) any |= w[e];
        if (any)
#pragma unroll
          for (int e = 0; e < E; ++e) f[e] = penalised(q, f[e], w[e]);
      }
      unsigned bits = 0xffffffffu;
      if (q.mask) {   // E bits from bit v on; they may lie in two words
        const int first = v >> 5, last = (v + E - 1) >> 5;
        const unsigned lo = __ldg(q.mask + first), hi = last != first ? __ldg(q.mask + last) : 0u;
        bits = __funnelshift_r(lo, hi, v & 31);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = finished(q, f[e], bits >> e & 1);
      if constexpr (E == 1) {
        y[v] = f[0];
      } else {
#pragma unroll
        for (int e = 0; e < E; e += 4) __stcs(reinterpret_cast<float4*>(y + v + e), make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]));
      }
    }
  }
  auto single = [&](int v, float x_, float bias) {
    float f = penalised(q, x_, listed ? word_at(v) : 0u) + bias;
    y[v] = finished(q, f, !q.mask || (__ldg(q.mask + (v >> 5)) >> (v & 31) & 1));
  };
  if (E > 1) {
    if (part == 0 && threadIdx.x < lead) single(threadIdx.x, to_float<T>(x[threadIdx.x]), 0.f);
    if (part == tail_part && static_cast<int>(threadIdx.x) < a.vocab - tail) single(tail + threadIdx.x, to_float<T>(x[tail + threadIdx.x]), 0.f);
  }

  // --------------------------------------------------------------------------------------------------------------- biases
  // Few tokens of a row have one: each is worked out again, behind everything else of this CTA.  Whoever finds a token's flag set takes
  // it down and looks for the token's other biases, which count in their order; of a token with several the first to arrive does it for
  // all of them.
  if (COUNTS && q.bias1 > q.bias0) {
    __syncthreads();
    for (long long b = q.bias0 + threadIdx.x; b < q.bias1; b += kThreads) {
      const long long t = a.bias_tokens[b];
      if (t < 0 || t >= a.vocab) continue;
      const int v = static_cast<int>(t), owner = v < lead ? 0 : v >= tail ? tail_part : (v - lead) / chunk;
      if (owner != part) continue;
      if (!(atomicAnd(&counts[v - body0 + E], ~kBiased) & kBiased)) {
        twice = 1;   // (several threads write the same)
        continue;
      }
      single(v, to_float<T>(x[v]), a.bias_values[b]);
    }
    __syncthreads();
    if (twice)   // rare: every bias of the row looks for others of its token, and the first of several sums them up
      for (long long b = q.bias0 + threadIdx.x; b < q.bias1; b += kThreads) {
        const long long t = a.bias_tokens[b];
        if (t < 0 || t >= a.vocab) continue;
        const int v = static_cast<int>(t), owner = v < lead ? 0 : v >= tail ? tail_part : (v - lead) / chunk;
        if (owner != part) continue;
        bool first = true, several = false;
        for (long long o = q.bias0; o < b && first; ++o) first = a.bias_tokens[o] != t;
        if (!first) continue;
        float sum = a.bias_values[b];
        for (long long o = b + 1; o < q.bias1; ++o)
          if (a.bias_tokens[o] == t) {
            sum += a.bias_values[o];
            several = true;
          }
        if (several) single(v, to_float<T>(x[v]), sum);
      }
  }
}

template <typename T, int E, bool COUNTS>
int launch(const ortb200_process_logits_args* a, int parts, int chunk, cudaStream_t stream) {
  const int smem = COUNTS ? (chunk + 2 * E) * 4 : 0;
  auto kern = process_logits_kernel<T, E, COUNTS>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (kMaxChunk + 64) * 4) != cudaSuccess) return -10;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a->rows * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = parts;
  attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = a->use_pdl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, *a, chunk) == cudaSuccess ? 0 : -11;
}

template <typename T>
int launch_type(const ortb200_process_logits_args* a, cudaStream_t stream) {
  constexpr int E = 16 / sizeof(T);
  const bool aligned = ((reinterpret_cast<uintptr_t>(a->logits) | reinterpret_cast<uintptr_t>(a->scores)) & 15) == 0;
  const bool counts = (a->history || a->drafted || a->bias_tokens) != 0;
  // as many CTAs to a row as hold its counters, and up to eight where there are few rows
  int parts = 1;
  while (parts < kMaxCluster && (static_cast<long long>(parts) * kChunk < a->vocab || a->rows * parts < 148)) parts *= 2;
  const int chunk = ((a->vocab + parts - 1) / parts + E - 1) / E * E;
  if (a->rows * parts > 0x7fffffffll) return -2;
  if (aligned) return counts ? launch<T, E, true>(a, parts, chunk, stream) : launch<T, E, false>(a, parts, chunk, stream);
  return counts ? launch<T, 1, true>(a, parts, chunk, stream) : launch<T, 1, false>(a, parts, chunk, stream);
}

}  // namespace
}  // namespace ortb200

using namespace ortb200;

extern "C" int ortb200_process_logits_max_vocab(void) { return kMaxCluster * kMaxChunk; }

extern "C" int ortb200_process_logits(const ortb200_process_logits_args* a, ortb200_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!a || a->rows < 0 || a->vocab <= 0 || a->history_len < 0 || a->bias_len < 0 || a->lists < 0 || a->drafted_width < 0 || a->masks < 0) return -1;
  if (a->rows == 0) return 0;
  if (!a->logits || !a->scores) return -1;
  if (a->history && !a->history_starts) return -1;
  if (a->bias_tokens && (!a->bias_values || !a->bias_starts)) return -1;
  if (a->allowed && (!a->row_mask || a->mask_words < (a->vocab + 31) / 32)) return -1;
  if (a->vocab > kMaxCluster * kMaxChunk || a->history_len + a->drafted_width > kCount) return -2;   // (a count has 30 bits)
  switch (a->dtype) {
    case ORTB200_F16: return launch_type<__half>(a, stream);
    case ORTB200_BF16: return launch_type<__nv_bfloat16>(a, stream);
    case ORTB200_F32: return launch_type<float>(a, stream);
  }
  return -4;
}
