// Moves units of a cache - the entry of a token, or a block - to other places of the same cache, in all of a model's caches at once
// (com.ortb200.PagedCacheMove).
//
// A target may be another move's source (a path of accepted tokens closes up, beams change places), so all sources are read before
// any target is written.  No CTA needs another for that: a CTA owns a range of bytes within the unit, of one cache, for ALL moves, and
// what lies there nobody else touches.  It reads the range of every source into shared memory, meets its own barrier, and writes.
//
// What bounds it: the bytes where they are many (40 blocks of 256 tokens in 24 caches of 8 heads of 128, 1 GB there and back: 145 to 150 us, 6.7 to
// 6.9 TB/s), the latency of a read behind a read of its place and a write behind it where they are few (200 tokens in 32 caches 8 us, 6 tokens in 64
// caches 5 us; the host's part of such a call is 12 and 18 us, most of it for the caches' names and tensors).  The range is as wide as lets four
// CTAs stay on an SM: each has up to 48 KB on its way.
#include <cuda_runtime.h>
#include "draft_ops.h"
#include "launch_util.cuh"

namespace ortb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kCaches = 128;        // caches of one launch: their addresses are kernel arguments
constexpr int kMaxMoves = 3000;     // times the narrowest range, 64 bytes, fits shared memory

struct Caches {
  uint8_t* at[kCaches];
  long long bytes[kCaches];
};

template <typename V>
__device__ __forceinline__ void fetch(V* to, const V* from) {
  if constexpr (sizeof(V) == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
  } else {
    *to = *from;
  }
}
__device__ __forceinline__ bool moved(long long source, long long target, long long units) {
  return target >= 0 && target < units && source >= 0 && source < units;
}

// What is wrong with the moves: places outside the cache, targets that are named twice.  One CTA looks, beside the others; its table
// of targets has at least twice as many places as there are moves, so that a search ends.
__device__ __forceinline__ void check_moves(const ortb200_cache_move_args& a, unsigned long long* seen, int slots_log2) {
  const unsigned slots = 1u << slots_log2;
  for (unsigned i = threadIdx.x; i < slots; i += kThreads) seen[i] = ~0ull;
  __syncthreads();
  bool bad = false;
  for (int m = threadIdx.x; m < static_cast<int>(a.moves); m += kThreads) {
    const long long s = a.sources[m], t = a.targets[m];
    if (t < 0) continue;
    if (!moved(s, t, a.units)) {
      bad = true;
      continue;
    }
    unsigned h = static_cast<unsigned>((static_cast<unsigned long long>(t) * 0x9e3779b97f4a7c15ull) >> (64 - slots_log2));
    while (true) {
      const unsigned long long was = atomicCAS(&seen[h], ~0ull, static_cast<unsigned long long>(t));
      if (was == ~0ull) break;
      if (was == static_cast<unsigned long long>(t)) {
        bad = true;
        break;
      }
      h = (h + 1) & (slots - 1);
    }
  }
  if (bad) atomicExch(a.status, kStatusBadArgument);
}

// V: the widest vector that divides all units and addresses.  cols: vectors of a CTA's range (a power of two).  The last CTA of a
// grid's first row checks the moves.
template <typename V>
__global__ void __launch_bounds__(kThreads) cache_move_kernel(const __grid_constant__ Caches caches, const ortb200_cache_move_args a, const int cols, const int slots_log2) {
  extern __shared__ __align__(16) uint8_t smem[];
  V* held = reinterpret_cast<V*>(smem);
  const int col = threadIdx.x & (cols - 1), moves = static_cast<int>(a.moves), step = kThreads / cols;
  const long long unit = caches.bytes[blockIdx.y] / static_cast<long long>(sizeof(V)), at = static_cast<long long>(blockIdx.x) * cols + col;
  pdl_wait_prior_grids();
  if (blockIdx.x == gridDim.x - 1) {
    if (blockIdx.y == 0 && a.status) check_moves(a, reinterpret_cast<unsigned long long*>(smem), slots_log2);
    return;
  }
  if (static_cast<long long>(blockIdx.x) * cols >= unit) return;
  V* base = reinterpret_cast<V*>(caches.at[blockIdx.y]) + at;
  const bool mine = at < unit;
  for (int m = threadIdx.x / cols; m < moves; m += step) {
    const long long s = a.sources[m], t = a.targets[m];
    if (mine && moved(s, t, a.units)) fetch(held + m * cols + col, static_cast<const V*>(base + s * unit));
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  for (int m = threadIdx.x / cols; m < moves; m += step) {
    const long long s = a.sources[m], t = a.targets[m];
    if (mine && moved(s, t, a.units)) base[t * unit] = held[m * cols + col];
  }
}

template <typename V>
int launch_move(const ortb200_cache_move_args* a, int64_t widest, cudaStream_t stream) {
  constexpr int kMaxSmem = 200 * 1024;
  // the widest range whose sources fit 48 KB (four CTAs and more to an SM)
  int cols = 64;
  while (cols > 1 && (cols * sizeof(V) * a->moves > 48 * 1024 || cols / 2 >= (widest + static_cast<int64_t>(sizeof(V)) - 1) / static_cast<int64_t>(sizeof(V))) &&
         cols * sizeof(V) > 64)
    cols /= 2;
  const int smem = static_cast<int>(cols * sizeof(V) * a->moves);
  int slots_log2 = 1;
  while ((1 << slots_log2) < 2 * a->moves) ++slots_log2;   // 8 bytes each, fewer than 32 a move: no more than the narrowest range takes
  if (smem > kMaxSmem) return -2;
  if (cudaFuncSetAttribute(cache_move_kernel<V>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem) != cudaSuccess) return -10;
  for (int c0 = 0; c0 < a->num_caches; c0 += kCaches) {
    Caches c = {};
    const int n = a->num_caches - c0 < kCaches ? a->num_caches - c0 : kCaches;
    int64_t most = 0;
    for (int i = 0; i < n; ++i) {
      c.at[i] = static_cast<uint8_t*>(a->caches[c0 + i]);
      c.bytes[i] = a->unit_bytes[c0 + i];
      most = c.bytes[i] > most ? c.bytes[i] : most;
    }
    const int64_t ranges = (most / static_cast<int64_t>(sizeof(V)) + cols - 1) / cols;
    if (ranges >= 0x7fffffff) return -2;
    ortb200_cache_move_args mine = *a;
    if (c0 > 0) mine.status = nullptr;   // checked by the first launch
    const int rc = launch_kernel(cache_move_kernel<V>, dim3(static_cast<unsigned>(ranges + 1), n), kThreads, smem, stream, a->use_pdl != 0, c, mine, cols, slots_log2);
    if (rc != 0) return rc;
  }
  return 0;
}

}  // namespace
}  // namespace ortb200

using namespace ortb200;

extern "C" int64_t ortb200_cache_move_max_moves(void) { return kMaxMoves; }

extern "C" int ortb200_cache_move(const ortb200_cache_move_args* a, ortb200_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!a || a->num_caches < 0 || a->moves < 0 || a->units < 0) return -1;
  if (a->moves == 0 || a->num_caches == 0) return 0;
  if (!a->caches || !a->unit_bytes || !a->sources || !a->targets) return -1;
  if (a->moves > kMaxMoves) return -2;
  uint64_t all = 0;
  int64_t widest = 0;
  for (int i = 0; i < a->num_caches; ++i) {
    if (a->unit_bytes[i] < 0 || (a->unit_bytes[i] > 0 && !a->caches[i])) return -1;
    all |= reinterpret_cast<uintptr_t>(a->caches[i]) | static_cast<uint64_t>(a->unit_bytes[i]);
    widest = a->unit_bytes[i] > widest ? a->unit_bytes[i] : widest;
  }
  if (all % 16 == 0) return launch_move<uint4>(a, widest, stream);
  if (all % 4 == 0) return launch_move<uint32_t>(a, widest, stream);
  if (all % 2 == 0) return launch_move<uint16_t>(a, widest, stream);
  return launch_move<uint8_t>(a, widest, stream);
}
