// Layout of a serving batch out of the lengths of its requests (com.ortb200.PagedBatchLayout): block table, cumulative lengths,
// positions and cache slots.
//
// Two running sums over the requests (tokens, blocks to hand out) decide everything; every CTA forms them for itself in shared
// memory, so that one launch does it all and no CTA waits for another.
#include <cuda_runtime.h>
#include "launch_util.cuh"
#include "serving_ops.h"

namespace ortb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxRequests = 16384;   // 8 bytes of shared memory each

__device__ __forceinline__ int blocks_of(long long tokens, int s) { return static_cast<int>((tokens + s - 1) / s); }

// exclusive running sums over the block of two values per thread; the totals of all threads in tot_a, tot_b
__device__ __forceinline__ void scan2(int& a, int& b, int& tot_a, int& tot_b, int (*sm)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int own_a = a, own_b = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) { a += x; b += y; }
  }
  __syncthreads();
  if (lane == 31) { sm[warp][0] = a; sm[warp][1] = b; }
  __syncthreads();
  tot_a = tot_b = 0;
  int before_a = 0, before_b = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w == warp) { before_a = tot_a; before_b = tot_b; }
    tot_a += sm[w][0];
    tot_b += sm[w][1];
  }
  a += before_a - own_a;
  b += before_b - own_b;
}

__global__ void __launch_bounds__(kThreads) batch_layout_kernel(const ortb200_batch_layout_args a) {
  extern __shared__ int sums[];
  int* cum = sums;              // [B + 1]
  int* first = sums + a.B + 1;  // [B + 1]
  __shared__ int sm[kThreads / 32][2];
  __shared__ int refused_sm;
  __shared__ unsigned long long totals[2];
  if (threadIdx.x == 0) {
    refused_sm = 0;
    totals[0] = totals[1] = 0;
  }
  __syncthreads();
  const int s = a.block_size;
  int base_a = 0, base_b = 0, worst = 0;
  unsigned long long sum_a = 0, sum_b = 0;
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    int n = 0, need = 0;
    if (b < a.B) {
      const int past = a.past_seqlens[b];
      n = a.new_tokens[b];
      if (past < 0 || n < 0) {
        worst = 4;
        n = 0;
      } else {
        const int held = blocks_of(past, s), all = blocks_of(static_cast<long long>(past) + n, s);
        need = all - held;
        if (need > 0 && all > a.max_blocks && worst < 2) worst = 2;
        if (n > 0 && held > a.max_blocks && worst < 2) worst = 2;
      }
    }
    sum_a += n;
    sum_b += need;
    int ta, tb;
    scan2(n, need, ta, tb, sm);
    if (b < a.B) {
      cum[b] = base_a + n;
      first[b] = base_b + need;
    }
    base_a += ta;
    base_b += tb;
  }
  // 64-bit totals: what overflows 32 bits in the running sums is refused here
  atomicAdd(&totals[0], sum_a);
  atomicAdd(&totals[1], sum_b);
  atomicMax(&refused_sm, worst);
  if (threadIdx.x == 0) {
    cum[a.B] = base_a;
    first[a.B] = base_b;
  }
  __syncthreads();
  int refused = refused_sm;
  if (refused < 4 && totals[0] > static_cast<unsigned long long>(a.rows)) refused = 3;
  if (refused < 2 && totals[1] > static_cast<unsigned long long>(a.num_free)) refused = 1;

  const long long tid = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x, stride = static_cast<long long>(gridDim.x) * kThreads;
  if (tid == 0) a.blocks_used[0] = refused ? -refused : base_b;
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
      const int past = a.past_seqlens[lo], held = blocks_of(past, s);
      pos = static_cast<long long>(past) + (t - cum[lo]);
      const int j = static_cast<int>(pos / s);
      // a block that this call hands out is not read from the table, which another CTA may be writing
      const int block = j < held ? a.table_in[static_cast<long long>(lo) * a.max_blocks + j] : a.free_blocks[first[lo] + j - held];
      slot = static_cast<long long>(block) * s + pos % s;
    }
    a.positions[t] = pos;
    a.slot_mapping[t] = slot;
  }
  const long long entries = static_cast<long long>(a.B) * a.max_blocks;
  for (long long i = tid; i < entries; i += stride) {
    const int b = static_cast<int>(i / a.max_blocks), j = static_cast<int>(i % a.max_blocks);
    const int fresh = refused ? 0 : first[b + 1] - first[b];
    const int held = fresh > 0 ? blocks_of(a.past_seqlens[b], s) : 0;
    if (j >= held && j < held + fresh) a.table_out[i] = a.free_blocks[first[b] + j - held];
    else if (a.table_out != a.table_in) a.table_out[i] = a.table_in[i];
  }
}

}  // namespace
}  // namespace ortb200

using namespace ortb200;

extern "C" int ortb200_batch_layout_max_requests(void) { return kMaxRequests; }

extern "C" int ortb200_batch_layout(const ortb200_batch_layout_args* a, ortb200_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!a || !a->cum || !a->blocks_used || a->B < 0 || a->max_blocks < 0 || a->block_size <= 0 || a->rows < 0 || a->num_free < 0) return -1;
  if (a->B > 0 && (!a->past_seqlens || !a->new_tokens || (a->max_blocks > 0 && (!a->table_in || !a->table_out)))) return -1;
  if (a->rows > 0 && (!a->positions || !a->slot_mapping)) return -1;
  if (a->num_free > 0 && !a->free_blocks) return -1;
  if (a->B > kMaxRequests || a->rows > 0x7fffffffll) return -2;
  const int smem = 8 * (a->B + 1);
  if (smem > 48 * 1024) {
    if (cudaFuncSetAttribute(batch_layout_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * (kMaxRequests + 1)) != cudaSuccess) return -10;
  }
  const long long most = a->rows > static_cast<long long>(a->B) * a->max_blocks ? a->rows : static_cast<long long>(a->B) * a->max_blocks;
  const long long want = (most + kThreads - 1) / kThreads;
  const int grid = static_cast<int>(want < 1 ? 1 : want > 592 ? 592 : want);
  batch_layout_kernel<<<grid, kThreads, smem, stream>>>(*a);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}
