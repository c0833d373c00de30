// Attention of a batch whose sequences begin with the same tokens (com.ortb200.SharedPrefixPagedAttention).
//
// softmax(q K^T) V splits over any partition of the keys: with m the largest score of a part, l = sum exp(s - m) and
// o = sum exp(s - m) v, two parts join as m = max(m1, m2), l = l1 e^(m1 - m) + l2 e^(m2 - m), o likewise; the result is o / l.
//
// Step 1 rotates the queries and the new keys and appends keys and values to the cache; step 2 attends.
#include <cuda_runtime.h>
#include <math.h>
#include "launch_util.cuh"
#include "serving_ops.h"

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
  pos = pos < 0 ? 0 : pos >= a.cos_rows ? a.cos_rows - 1 : pos;   // never past the rotary tables
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
    const Span s = span_of(a, b);
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
  return T * N * H * 4;
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
  switch (a->dtype) {
    case ORTB200_F16: return launch_rows<__half>(a, stream);
    case ORTB200_BF16: return launch_rows<__nv_bfloat16>(a, stream);
    case ORTB200_F32: return launch_rows<float>(a, stream);
  }
  return -4;
}
