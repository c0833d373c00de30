// Layout of a serving batch out of the lengths of its requests (com.ortb200.PagedBatchLayout): block table, cumulative lengths,
// positions and cache slots.
//
// Two running sums over the requests (tokens, blocks to hand out) decide everything; every CTA forms them for itself in shared
// memory, so that one launch does it all and no CTA waits for another.
//
// What bounds it: the launch where requests are few (24 requests 3.5 us on the device, 160 with 27000 rows 4.1), the table where
// it is large: 1000 requests of 4096 blocks, 33 MB there and back, take 10.3 us, 5.1 at the copy rate.  Slower per call: one 64-bit
// atomic in shared memory per request for the totals (14 and 27 us instead of 9 and 13), and an entry of the table per thread
// instead of four times 16 bytes (45).
#include <cuda_runtime.h>
#include "launch_util.cuh"
#include "serving_ops.h"

namespace ortb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxRequests = 16384;   // 8 bytes of shared memory each
constexpr long long kMaxRows = 0x7ff00000;   // a row or block plus the threads of the grid fits 31 bits

// (past and new each fit 31 bits: their sum fits 32)
__device__ __forceinline__ long long blocks_of(long long tokens, int s) {
  const unsigned t = static_cast<unsigned>(tokens), q = t / static_cast<unsigned>(s);
  return static_cast<long long>(q) + (q * static_cast<unsigned>(s) != t);
}

// What a warp knows of its requests: tokens, blocks to hand out, the largest refusal code.
struct Totals {
  long long tokens, blocks;
  int worst;
};

__global__ void __launch_bounds__(kThreads) batch_layout_kernel(const ortb200_batch_layout_args a) {
  extern __shared__ int sums[];
  int* cum = sums;              // [B + 1]
  int* first = sums + a.B + 1;  // [B + 1]
  __shared__ Totals sm[kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int s = a.block_size, each = (a.B + kThreads - 1) / kThreads;
  // a thread's requests follow one another: their sums first, the running sums of the threads, then every request's
  const int b0 = min(static_cast<int>(threadIdx.x) * each, a.B), b1 = min(b0 + each, a.B);
  int worst = 0;
  long long sum_a = 0, sum_b = 0;   // 64 bits: what would overflow the 32 of the outputs is refused
  auto request = [&](int b, int& n, int& need) {
    const int past = a.past_seqlens[b];
    n = a.new_tokens[b];
    need = 0;
    if (past < 0 || n < 0) {
      worst = 4;
      n = 0;
      return;
    }
    const long long held = blocks_of(past, s), all = blocks_of(static_cast<long long>(past) + n, s);
    need = static_cast<int>(all - held);
    if (n > 0 && all > a.max_blocks && worst < 2) worst = 2;
  };
#pragma unroll 4
  for (int b = b0; b < b1; ++b) {
    int n, need;
    request(b, n, need);
    sum_a += n;
    sum_b += need;
  }
  long long up_a = sum_a, up_b = sum_b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, up_a, o), y = __shfl_up_sync(0xffffffffu, up_b, o);
    if (lane >= o) {
      up_a += x;
      up_b += y;
    }
  }
  worst = __reduce_max_sync(0xffffffffu, worst);
  if (lane == 31) sm[warp] = {up_a, up_b, worst};
  __syncthreads();
  long long run_a = up_a - sum_a, run_b = up_b - sum_b, all_a = 0, all_b = 0;
  int refused = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) {
      run_a += sm[w].tokens;
      run_b += sm[w].blocks;
    }
    all_a += sm[w].tokens;
    all_b += sm[w].blocks;
    refused = max(refused, sm[w].worst);
  }
  if (refused < 4 && all_a > a.rows) refused = 3;
  if (refused < 2 && all_b > a.num_free) refused = 1;
#pragma unroll 4
  for (int b = b0; b < b1; ++b) {
    int n, need;
    request(b, n, need);
    cum[b] = static_cast<int>(run_a);
    first[b] = static_cast<int>(run_b);
    run_a += n;
    run_b += need;
  }
  if (threadIdx.x == 0) {
    cum[a.B] = static_cast<int>(all_a);
    first[a.B] = static_cast<int>(all_b);
  }
  __syncthreads();

  const long long tid = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x, stride = static_cast<long long>(gridDim.x) * kThreads;
  if (tid == 0) {
    a.blocks_used[0] = refused ? -refused : static_cast<int>(all_b);
    if (refused && a.status) atomicExch(a.status, kStatusBadLength);
  }
  for (long long b = tid; b <= a.B; b += stride) a.cum[b] = refused ? 0 : cum[b];
  const int end = refused ? 0 : cum[a.B];
  for (long long t = tid; t < a.rows; t += stride) {
    long long pos = -1, slot = -1;
    if (t < end) {
      int lo = 0, hi = a.B;   // the last request that starts at or before t and has tokens
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cum[mid] <= t) lo = mid; else hi = mid;
      }
      const int past = a.past_seqlens[lo];
      const long long held = blocks_of(past, s);
      pos = static_cast<long long>(past) + (t - cum[lo]);
      const unsigned j = static_cast<unsigned>(pos) / static_cast<unsigned>(s), offset = static_cast<unsigned>(pos) - j * static_cast<unsigned>(s);
      // a block that this call hands out is not read from the table, which another CTA may be writing
      const int block = j < held ? a.table_in[static_cast<long long>(lo) * a.max_blocks + j] : a.free_blocks[first[lo] + j - held];
      slot = static_cast<long long>(block) * s + offset;
    }
    a.positions[t] = pos;
    a.slot_mapping[t] = slot;
  }
  // the table: what the requests hold, and the blocks that they are given
  const int used = refused ? 0 : static_cast<int>(all_b);
  if (a.table_out == a.table_in) {
    for (int i = static_cast<int>(tid); i < used; i += static_cast<int>(stride)) {
      int lo = 0, hi = a.B;   // the request that block i goes to
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= i) lo = mid; else hi = mid;
      }
      a.table_out[static_cast<long long>(lo) * a.max_blocks + blocks_of(a.past_seqlens[lo], s) + i - first[lo]] = a.free_blocks[i];
    }
    return;
  }
  const long long entries = static_cast<long long>(a.B) * a.max_blocks;
  auto entry = [&](int old, int b, int j) {
    const int fresh = refused ? 0 : first[b + 1] - first[b];
    if (fresh == 0) return old;
    const long long k = j - blocks_of(a.past_seqlens[b], s);
    return k >= 0 && k < fresh ? a.free_blocks[first[b] + k] : old;
  };
  if (((reinterpret_cast<uintptr_t>(a.table_in) | reinterpret_cast<uintptr_t>(a.table_out)) & 15) == 0 && a.max_blocks % 4 == 0) {
    // rows of whole vectors; four of them on their way per thread
    const unsigned per_row = static_cast<unsigned>(a.max_blocks) / 4;
    const long long vectors = entries / 4;
    const int4* in = reinterpret_cast<const int4*>(a.table_in);
    int4* out = reinterpret_cast<int4*>(a.table_out);
    for (long long i = tid; i < vectors; i += 4 * stride) {
      int4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i + u * stride < vectors) v[u] = __ldcs(in + i + u * stride);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const long long at = i + u * stride;
        if (at >= vectors) break;
        const int b = static_cast<int>(at <= 0xffffffffll ? static_cast<unsigned>(at) / per_row : at / per_row), j = 4 * static_cast<int>(at - static_cast<long long>(b) * per_row);
        const int fresh = refused ? 0 : first[b + 1] - first[b];
        if (fresh > 0) {
          const long long k = j - blocks_of(a.past_seqlens[b], s);
          if (k > -4 && k < fresh) {
            int* e = reinterpret_cast<int*>(&v[u]);
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (k + c >= 0 && k + c < fresh) e[c] = a.free_blocks[first[b] + k + c];
          }
        }
        __stcs(out + at, v[u]);
      }
    }
    return;
  }
  for (long long i = tid; i < entries; i += stride) {
    const int b = static_cast<int>(i / a.max_blocks), j = static_cast<int>(i % a.max_blocks);
    a.table_out[i] = entry(a.table_in[i], b, j);
  }
}

}  // namespace
}  // namespace ortb200

using namespace ortb200;

extern "C" int ortb200_batch_layout_max_requests(void) { return kMaxRequests; }
extern "C" int64_t ortb200_batch_layout_max_rows(void) { return kMaxRows; }

extern "C" int ortb200_batch_layout(const ortb200_batch_layout_args* a, ortb200_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!a || !a->cum || !a->blocks_used || a->B < 0 || a->max_blocks < 0 || a->block_size <= 0 || a->rows < 0 || a->num_free < 0) return -1;
  if (a->B > 0 && (!a->past_seqlens || !a->new_tokens || (a->max_blocks > 0 && (!a->table_in || !a->table_out)))) return -1;
  if (a->rows > 0 && (!a->positions || !a->slot_mapping)) return -1;
  if (a->num_free > 0 && !a->free_blocks) return -1;
  if (a->B > kMaxRequests || a->rows > kMaxRows) return -2;
  const int smem = 8 * (a->B + 1);
  if (smem > 47 * 1024) {   // (the kernel has some shared memory of its own, which counts towards the 48 KB that need no leave)
    if (cudaFuncSetAttribute(batch_layout_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * (kMaxRequests + 1)) != cudaSuccess) return -10;
  }
  const long long most = a->rows > static_cast<long long>(a->B) * a->max_blocks ? a->rows : static_cast<long long>(a->B) * a->max_blocks;
  const long long want = (most + kThreads - 1) / kThreads;
  const int grid = static_cast<int>(want < 1 ? 1 : want > 592 ? 592 : want);
  batch_layout_kernel<<<grid, kThreads, smem, stream>>>(*a);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}
