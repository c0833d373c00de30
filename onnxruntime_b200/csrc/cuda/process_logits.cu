// Penalties for repeated tokens, biases, masks and temperatures on logits (com.ortb200.ProcessLogits).
//
// Every logit is read once and every score written once.  A CTA has a chunk of a row's vocabulary, with a counter per token in shared
// memory.  It asks its logits into L2, reads the row's whole text and biases and counts and flags the tokens of its chunk, and streams the
// chunk through temperature and mask.  The few tokens that are touched are listed, and worked out again behind the stream; where
// they are more than the list holds, the stream looks at every counter.  No CTA waits for another, and counting commutes: no result
// depends on an order of arrival.
//
// What bounds it: without texts the stream (384 rows of 128256 bf16 logits 55 us, 295 MB; the bytes need 45).  With a text of 2250 tokens to a
// row 108 us: reading and counting it in each of 16 chunks, 112 MB out of L2 and half of the instructions; issue slots are 67 % busy.  A text of
// 45000 tokens and 50257 32-bit logits, 40 rows: 24 us, nearly all of it the text: four parts of a row read it, the last of which has 1105 tokens, and with
// one CTA of 1024 threads to an SM 160 CTAs are two rounds.  Slower, for the same 384 rows: a text read once by a cluster of
// the row's CTAs, which add to each other's counters, 212 us; a kernel that gathers what a row touches in a hash table, behind the stream or
// in front of it, 105 to 111 and a second launch; a warp's tokens of the chunk queued and counted 32 at a time 123.
#include <cuda_runtime.h>
#include <math.h>
#include "draft_ops.h"
#include "launch_util.cuh"

namespace ortb200 {
namespace {

constexpr int kMaxChunk = 16384;      // counters of a CTA: 64 KB
constexpr int kList = 1024;           // touched tokens of a chunk that are listed
constexpr int kBiases = 256;          // biases of a chunk that are
constexpr int kMaxVocab = 0x7fff0000; // an index plus the tokens of a pass fits 31 bits
constexpr unsigned kSeen = 0x80000000u, kBiased = 0x40000000u, kCount = 0x3fffffffu;

// Quotients by one divisor of a whole row: with its rounded reciprocal r, q = x r is off by a unit or so, the remainder x - q d is exact in
// a fused multiply-add, and q + r (x - q d) is the quotient rounded once (P. Markstein, IBM Journal of Research and Development 34, 1990;
// numbers below 2^-100, whose remainders 32 bits do not hold, are within 3 times that).
// A division takes some twenty instructions, and the long way for infinities: with one for every logit the kernel had 48 instructions to a logit.
struct Divisor {
  float d, r;   // r: NaN where the reciprocal's exponent leaves no room for the remainder
  __device__ __forceinline__ explicit Divisor(float by) : d(by), r(fabsf(by) > 0x1p-100f && fabsf(by) < 0x1p100f ? 1.f / by : NAN) {}
  __device__ __forceinline__ float special(float x, float q) const { return r == r ? q : x / d; }   // infinities, and what overflows
  __device__ __forceinline__ float operator()(float x) const {
    const float q = x * r, y = fmaf(fmaf(-q, d, x), r, q);
    return y == y ? y : special(x, q);
  }
  template <int N>
  __device__ __forceinline__ void all(float* f) const {
    const f32x2 r2 = pack2(r, r), minus = pack2(-d, -d), one = pack2(1.f, 1.f);
    f32x2 x[N / 2], q[N / 2], y[N / 2], sum = pack2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      x[i] = pack2(f[2 * i], f[2 * i + 1]);
      q[i] = mul2(x[i], r2);
      y[i] = fma2(fma2(q[i], minus, x[i]), r2, q[i]);
      sum = fma2(y[i], one, sum);
    }
    float s0, s1;
    unpack2(sum, s0, s1);
    if (s0 + s1 == s0 + s1) {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) unpack2(y[i], f[2 * i], f[2 * i + 1]);
    } else {   // one of them is no number, or the sum of two infinities
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = (*this)(f[i]);
    }
  }
};

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
  if (a.bias_starts) {
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
__device__ __forceinline__ float penalised(const RowRules& q, const Divisor& repeated, float x, unsigned word) {
  if (word & ~kBiased) {   // somewhere in the text
    x = x < 0.f ? x * q.repetition : repeated(x);
    const unsigned c = word & kCount;
    if (c) x -= q.frequency * static_cast<float>(c) + q.presence;
  }
  return x;
}

// The text of a row: history [begin, end), of which what lies from `counted` on counts, and its row of drafted tokens.
struct Text {
  long long begin, end, counted;
  int drafted;
  bool bad;
  // (Asked for beside the row's rules: every load that waits for another adds most of a microsecond to a CTA that has some eight.)
  __device__ __forceinline__ Text(const ortb200_process_logits_args& a, long long r) : begin(0), end(0), counted(0), drafted(a.drafted ? a.drafted_width : 0), bad(false) {
    if (!a.history) return;
    const long long l = a.row_list ? a.row_list[r] : r;
    bad = l >= a.lists;
    if (l < 0 || bad) return;
    begin = a.history_starts[l];
    end = a.history_starts[l + 1];
    counted = a.generated_starts ? a.generated_starts[l] : 0;
    bad = begin < 0 || end < begin || end > a.history_len;
    if (bad) begin = end = 0;
  }
  __device__ __forceinline__ bool any() const { return end > begin || drafted > 0; }
};
// add(token) for tokens [begin, end) of the history, by all threads: two tokens to a load, AHEAD loads of a thread on their way
template <int THREADS, int AHEAD, typename F>
__device__ __forceinline__ void for_tokens(const int64_t* history, long long begin, long long end, F add) {
  if (begin >= end) return;
  const int64_t* p = history + begin;
  const int len = static_cast<int>(end - begin), odd = static_cast<int>((reinterpret_cast<uintptr_t>(p) >> 3) & 1), pairs = (len - odd) / 2;   // (a history has fewer than 2^30 tokens)
  if (threadIdx.x == 0 && odd) add(p[0]);
  if (threadIdx.x == 32 && odd + 2 * pairs < len) add(p[len - 1]);
  const longlong2* two = reinterpret_cast<const longlong2*>(p + odd);
  for (int i = threadIdx.x; i < pairs; i += AHEAD * THREADS) {
    longlong2 v[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (i + k * THREADS < pairs) v[k] = __ldg(two + i + k * THREADS);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (i + k * THREADS < pairs) {
        add(v[k].x);
        add(v[k].y);
      }
  }
}
// seen(token) for what does not count of a text, count(token) for what does
template <int THREADS, int AHEAD, typename S, typename C>
__device__ __forceinline__ void for_text(const ortb200_process_logits_args& a, const Text& t, long long r, S seen, C count) {
  const long long counts_from = min(max(t.counted, t.begin), t.end);
  for_tokens<THREADS, AHEAD>(a.history, t.begin, counts_from, seen);
  for_tokens<THREADS, AHEAD>(a.history, counts_from, t.end, count);
  for (int d = threadIdx.x; d < t.drafted; d += THREADS) count(a.drafted[r * a.drafted_width + d]);
}
// (as an instruction of its own: the compiler makes one addition for a warp out of atomicAdd to one place, which costs more than the two
// lanes that usually come)
__device__ __forceinline__ int next_place(int* counter) {
  int n;
  asm volatile("atom.shared.add.u32 %0, [%1], 1;" : "=r"(n) : "r"(smem_u32(counter)) : "memory");
  return n;
}

// A score from its logit: penalties by the token's counter, its bias, the temperature, the mask.
template <typename T>
struct Scorer {
  const T* x;
  float* y;
  const RowRules& q;
  const Divisor &warmth, &repeated;
  __device__ __forceinline__ bool allowed(int v) const { return !q.mask || (__ldg(q.mask + (v >> 5)) >> (v & 31) & 1); }
  __device__ __forceinline__ float finished(int v, float f) const {
    if (q.temperature != 1.f) f = warmth(f);
    return allowed(v) ? f : -INFINITY;
  }
  // (a bias of -inf is a ban: added to an infinite logit, or to one that is no number, it would leave a NaN, which a search for the largest takes)
  __device__ __forceinline__ void whole(int v, unsigned word, float bias) const {
    y[v] = bias == -INFINITY ? bias : finished(v, penalised(q, repeated, to_float<T>(x[v]), word) + bias);
  }
};

// How a row is divided: its vectors start at the first token whose place in the tensor E divides; what is in front of them is the first
// CTA's, and the last tokens, fewer than a vector, belong to whoever has what is in front of those.
struct Chunks {
  int vocab, chunk, lead, tail, tail_part;
  __device__ __forceinline__ Chunks(int vocabulary, long long r, int E, int size) : vocab(vocabulary), chunk(size) {
    lead = E == 1 ? 0 : min(static_cast<int>((E - r * vocab % E) % E), vocab);
    tail = lead + (vocab - lead) / E * E;
    tail_part = tail > lead ? (tail - lead - 1) / chunk : 0;
  }
};

template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float* f) {
  const T* t = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < 16 / static_cast<int>(sizeof(T)); ++i) f[i] = to_float<T>(t[i]);
}

// Where a CTA is: tokens [first, end) of row r, the vectors among them, and the token of counter 0 (a row's first tokens may lie in front of
// the first vector, its last ones behind the last).
struct Place {
  int body0, vectors, first, end, base;
  __device__ __forceinline__ Place(const Chunks& c, int part, int E) {
    body0 = c.lead + part * c.chunk;
    const int body1 = min(body0 + c.chunk, c.tail);
    vectors = max(body1 - body0, 0) / E;
    first = part == 0 ? 0 : body0;
    end = part == c.tail_part ? c.vocab : part < c.tail_part ? body1 : first;
    base = body0 - E;
  }
};

// E: logits of a vector (1: any alignment).  TOUCHED: rows may have texts or biases; else the stream alone.
template <typename T, int E, bool TOUCHED, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 6 : 1) process_logits_kernel(const ortb200_process_logits_args a, const int chunk, const int parts) {
  extern __shared__ __align__(16) unsigned counts[];            // [chunk + 2 E + 4]
  __shared__ int listed, biases, twice;
  __shared__ uint16_t list[TOUCHED ? kList : 1], biased[TOUCHED ? kBiases : 1];   // of counters
  __shared__ float bias_of[TOUCHED ? kBiases : 1];
  const int part = static_cast<int>(blockIdx.x % parts);
  const long long r = blockIdx.x / parts;
  pdl_wait_prior_grids();
  const T* x = static_cast<const T*>(a.logits) + r * a.vocab;
  float* y = a.scores + r * a.vocab;
  const Chunks c(a.vocab, r, E, chunk);
  const Place at(c, part, E);
  for (int i = threadIdx.x; i * 128 < at.vectors * E * static_cast<int>(sizeof(T)); i += THREADS)   // on their way while the row's rules and text come
    asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(x + at.body0) + i * 128));
  const Text t(a, r);
  const RowRules q = rules_of(a, r, part == 0 && threadIdx.x == 0);
  const Divisor warmth(q.temperature), repeated(q.repetition);
  const Scorer<T> s = {x, y, q, warmth, repeated};

  bool touched = false, dense = false;   // dense: the stream looks at the counters, and there is no list
  if constexpr (TOUCHED) {
    const bool asks = q.repetition != 1.f || q.presence != 0.f || q.frequency != 0.f, text = asks && t.any();   // (a row without penalties has no use for its text)
    if (asks && t.bad && part == 0 && threadIdx.x == 0 && a.status) atomicExch(a.status, kStatusBadArgument);
    touched = text || q.bias1 > q.bias0;
    if (touched) {
      if (threadIdx.x == 0) listed = biases = twice = 0;
      for (int i = threadIdx.x; i < (chunk + 2 * E + 4) / 4; i += THREADS) reinterpret_cast<uint4*>(counts)[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      const unsigned size = static_cast<unsigned>(at.end - at.first);
      auto counter_of = [&](long long v) -> int {   // -1: another CTA's token, or none
        const unsigned u = static_cast<unsigned>(v) - static_cast<unsigned>(at.first);
        return u >= size || static_cast<unsigned long long>(v) >> 32 ? -1 : at.first - at.base + static_cast<int>(u);
      };
      auto to_list = [&](int i) {
        const int n = next_place(&listed);
        if (n < kList) list[n] = static_cast<uint16_t>(i);
      };
      dense = text && t.end - t.begin > static_cast<long long>(parts) * kList;   // too many to be listed, most likely
      for (long long b = q.bias0 + threadIdx.x; b < q.bias1; b += THREADS) {
        const int i = counter_of(a.bias_tokens[b]);
        if (i < 0) continue;
        const unsigned was = atomicOr(&counts[i], kBiased);
        if (was & kBiased) twice = 1;   // (whoever writes, writes the same)
        if (was == 0) to_list(i);
        const int n = atomicAdd(&biases, 1);
        if (n < kBiases) {
          biased[n] = static_cast<uint16_t>(i);
          bias_of[n] = a.bias_values[b];
        }
      }
      if (text && dense) {
        for_text<THREADS, 4>(
            a, t, r,
            [&](long long v) {
              const int i = counter_of(v);
              if (i >= 0) atomicOr(&counts[i], kSeen);
            },
            [&](long long v) {
              const int i = counter_of(v);
              if (i >= 0) atomicAdd(&counts[i], 1u);
            });
      } else if (text) {
        for_text<THREADS, 4>(
            a, t, r,
            [&](long long v) {
              const int i = counter_of(v);
              if (i >= 0 && atomicOr(&counts[i], kSeen) == 0) to_list(i);
            },
            [&](long long v) {
              const int i = counter_of(v);
              if (i >= 0 && atomicAdd(&counts[i], 1u) == 0) to_list(i);
            });
      }
      __syncthreads();
      dense = dense || listed > kList;
    }
  }

  // ------------------------------------------------------------------------------------------------------ the chunk's vectors
  constexpr int kAhead = E == 1 ? 8 : 4;
  for (int i0 = 0; i0 < at.vectors; i0 += kAhead * THREADS) {
    T one[E == 1 ? kAhead : 1];
    uint4 many[E == 1 ? 1 : kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int n = i0 + i * THREADS + threadIdx.x;
      if (n < at.vectors) {
        if constexpr (E == 1) one[i] = x[at.body0 + n];
        else many[i] = __ldg(reinterpret_cast<const uint4*>(x + at.body0) + n);
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int n = i0 + i * THREADS + threadIdx.x, v = at.body0 + n * E;
      if (n >= at.vectors) continue;
      if constexpr (E == 1) {
        y[v] = s.finished(v, penalised(q, repeated, to_float<T>(one[i]), TOUCHED && dense ? counts[v - at.base] : 0u));
      } else {
        float f[E];
        unpack<T>(many[i], f);
        if (TOUCHED && dense) {
          unsigned w[E];
#pragma unroll
          for (int e = 0; e < E; e += 4) *reinterpret_cast<uint4*>(w + e) = *reinterpret_cast<const uint4*>(counts + v - at.base + e);
#pragma unroll
          for (int e = 0; e < E; ++e) f[e] = penalised(q, repeated, f[e], w[e]);
        }
        if (q.temperature != 1.f) warmth.all<E>(f);
        if (q.mask) {   // E bits from bit v on; they may lie in two words
          const int w0 = v >> 5, w1 = (v + E - 1) >> 5;
          const unsigned lo = __ldg(q.mask + w0), hi = w1 != w0 ? __ldg(q.mask + w1) : 0u, bits = __funnelshift_r(lo, hi, v & 31);
#pragma unroll
          for (int e = 0; e < E; ++e) f[e] = bits & 1u << e ? f[e] : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < E; e += 4) __stcs(reinterpret_cast<float4*>(y + v + e), make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]));
      }
    }
  }
  if (E > 1) {
    const int t = static_cast<int>(threadIdx.x), v = t < E ? t : c.tail + t - E;
    if (t < E ? part == 0 && v < c.lead : part == c.tail_part && v < a.vocab) s.whole(v, touched ? counts[v - at.base] : 0u, 0.f);
  }

  // -------------------------------------------------------------------------------------------------------- what is touched
  if constexpr (TOUCHED) {
    if (!touched) return;
    __syncthreads();   // the stream's scores have been written
    const bool apart = dense || twice || biases > kBiases;   // biases are worked out by themselves
    if (!dense)
      for (int i = threadIdx.x; i < listed; i += THREADS) {
        const int n = list[i];
        const unsigned word = counts[n];
        float bias = 0.f;
        if (word & kBiased) {
          if (apart) continue;
          for (int k = 0; k < biases; ++k)
            if (biased[k] == n) bias = bias_of[k];
        }
        s.whole(at.base + n, word, bias);
      }
    if (!apart) return;
    auto here = [&](long long v) { return v >= at.first && v < at.end; };
    if (!twice) {   // many biases, or a long text
      for (long long b = q.bias0 + threadIdx.x; b < q.bias1; b += THREADS) {
        const long long v = a.bias_tokens[b];
        if (here(v)) s.whole(static_cast<int>(v), counts[static_cast<int>(v) - at.base], a.bias_values[b]);
      }
      return;
    }
    // Rare: a token has several biases.  One warp goes through all of them in their order, 32 at a time, and keeps the sums where the scores go; a
    // counter's flag tells whether its token has no sum yet.  Then whoever sets the flag again makes the score of the sum.  (A search for each bias
    // among all others would take the square of their number.)
    __syncthreads();
    if (threadIdx.x < 32) {
      const int lane = static_cast<int>(threadIdx.x);
      for (long long b0 = q.bias0; b0 < q.bias1; b0 += 32) {
        const long long v = b0 + lane < q.bias1 ? a.bias_tokens[b0 + lane] : -1;
        const bool mine = here(v);
        if (!__any_sync(0xffffffffu, mine)) continue;
        const float value = mine ? a.bias_values[b0 + lane] : 0.f;
        const unsigned same = __match_any_sync(0xffffffffu, mine ? static_cast<int>(v) : -1 - lane);   // of a token the first lane sums up
        const bool leads = mine && __ffs(same) - 1 == lane;
        float sum = value;
        if (leads) {
          unsigned& word = counts[static_cast<int>(v) - at.base];
          if (!(word & kBiased)) sum = y[v] + value;
          word &= ~kBiased;
        }
        for (unsigned rest = leads ? same & (same - 1) : 0; __any_sync(0xffffffffu, rest != 0); rest &= rest - 1) {
          const float next = __shfl_sync(0xffffffffu, value, rest ? __ffs(rest) - 1 : lane);
          if (rest) sum += next;
        }
        if (leads) y[v] = sum;
        __syncwarp();
      }
    }
    __syncthreads();
    for (long long b = q.bias0 + threadIdx.x; b < q.bias1; b += THREADS) {
      const long long v = a.bias_tokens[b];
      if (!here(v)) continue;
      const unsigned word = atomicOr(&counts[static_cast<int>(v) - at.base], kBiased);
      if (!(word & kBiased)) s.whole(static_cast<int>(v), word, y[v]);
    }
  }
}

template <typename T, int E, bool TOUCHED, int THREADS>
int launch(const ortb200_process_logits_args* a, int64_t text_bytes, cudaStream_t stream) {
  // Usually four vectors of logits to a thread.  Shorter chunks where rows are few, so that every SM has some, but, as a text is read once
  // for each chunk, none that are fewer bytes than the usual text.
  int chunk = THREADS == 256 ? 8192 : kMaxChunk;
  while (chunk > 2048 && a->rows * ((a->vocab + chunk - 1) / chunk) < 3 * 148 && text_bytes <= chunk / 2 * static_cast<int64_t>(sizeof(T) + 4)) chunk /= 2;
  const long long parts = (a->vocab + static_cast<long long>(chunk) - 1) / chunk;
  if (a->rows * parts > 0x7fffffffll) return -2;
  const int smem = TOUCHED ? (chunk + 2 * E + 4) * 4 : 0;
  auto kern = process_logits_kernel<T, E, TOUCHED, THREADS>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (kMaxChunk + 64) * 4) != cudaSuccess) return -10;   // per device
  return launch_kernel(kern, dim3(static_cast<unsigned>(a->rows * parts)), THREADS, smem, stream, a->use_pdl != 0, *a, chunk, static_cast<int>(parts));
}

template <typename T, int E>
int launch_rows(const ortb200_process_logits_args* a, cudaStream_t stream) {
  if (!a->history && !a->drafted && !a->bias_tokens) return launch<T, E, false, 256>(a, 0, stream);
  // Every chunk reads the row's text.  Texts of up to 64 KB: chunks of 8192 and CTAs of 256 threads, six to an SM (384 rows of 128256 with 2250
  // tokens 108 us, with 10 tokens 70; chunks of 16384 and three CTAs of 512 threads 104 and 80, two of them 122 and 92).  Longer ones: chunks of 16384,
  // half as many bytes of text, and 1024 threads that read them (40 rows of 50257 with 45000 tokens 24 us; before a text's two parts had loops of their own 27, 512 threads 32, the short texts' way 45).
  const int64_t text_bytes = a->history && a->lists > 0 ? 8 * (a->history_len / a->lists) : 0;
  return text_bytes > 64 * 1024 ? launch<T, E, true, 1024>(a, text_bytes, stream) : launch<T, E, true, 256>(a, text_bytes, stream);
}

template <typename T>
int launch_type(const ortb200_process_logits_args* a, cudaStream_t stream) {
  const bool aligned = ((reinterpret_cast<uintptr_t>(a->logits) | reinterpret_cast<uintptr_t>(a->scores)) & 15) == 0;
  return aligned ? launch_rows<T, 16 / sizeof(T)>(a, stream) : launch_rows<T, 1>(a, stream);
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
