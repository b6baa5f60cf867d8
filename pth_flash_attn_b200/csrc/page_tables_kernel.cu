// Block tables, slots, positions and offsets of a step from the requests' lengths, in one launch.
//
//   seq_r = c_r + q_r;  start_r = sum_{i<r} q_i;  pages of r that are new: ceil(c_r/BS) .. ceil(seq_r/BS), whose ids
//   are the entries first_r = sum_{i<r} new_i onwards of the free list.
//
// Every CTA sums the lengths of all requests up for itself (a thread takes a run of requests, then one scan over the
// CTA) and keeps the two running sums in shared memory, so nothing is passed between CTAs and no second launch is
// needed: 8 bytes of lengths a request, 128 KB at the 16,384 that a call takes, out of the L2 cache.  Tokens and new pages are then
// two flat lists that the CTAs deal out evenly however the lengths are spread; the request of an entry is found by
// bisection.  A token's page is taken from the free list itself where it is new, so no CTA reads what
// another writes.
//
// What bounds it is latency: alone and cold the kernel runs 4.8 us for 64 requests of one token each, 6.6 for 4 x 2,048 tokens and 8.1
// for 128 prompts of up to 2,500 tokens (3 MB written); launches that wait in the stream behind one another take 2.5, 2.8 and
// 4.2.  A call takes the host 6.2 us, so eager calls behind one another take 8.0 us each.
#include "kv16.cuh"
#include "pdl.cuh"

namespace pthb200 {
namespace {

constexpr int kTableThreads = 256;
constexpr int kTableWarps = kTableThreads / 32;
constexpr int kMostCtas = 592;        // four per SM

__device__ __forceinline__ int pages_of(int64_t tokens, int block_size) {
  if (tokens <= 0) return 0;
  if (tokens + block_size <= 0xffffffffll) return (int)(((uint32_t)tokens + (uint32_t)(block_size - 1)) / (uint32_t)block_size);
  return (int)((tokens + block_size - 1) / block_size);
}

// Largest r in [0, n) with first[r] <= i.
__device__ __forceinline__ int owner(const int32_t* first, int n, int i) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= i) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kTableThreads) page_tables_kernel(const __grid_constant__ PthB200TablesArgs a) {
  extern __shared__ int32_t sums[];  // start [num_reqs + 1], first [num_reqs + 1], context [num_reqs]
  __shared__ int32_t warp_q[kTableWarps], warp_n[kTableWarps];
  const int R = a.num_reqs, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int32_t* const start = sums;
  int32_t* const first = sums + R + 1;
  int32_t* const context = first + R + 1;
  pdl_wait();
  const int per = (R + kTableThreads - 1) / kTableThreads, r0 = min(R, tid * per), r1 = min(R, r0 + per);
  int q_sum = 0, n_sum = 0;
  for (int r = r0; r < r1; ++r) {
    const int c = max(0, __ldg(a.context_lens + r)), q = max(0, __ldg(a.query_lens + r));
    start[r] = q_sum;
    first[r] = n_sum;
    context[r] = c;
    q_sum += q;
    n_sum += pages_of((int64_t)c + q, a.block_size) - pages_of(c, a.block_size);
  }
  int q_inc = q_sum, n_inc = n_sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, q_inc, o), y = __shfl_up_sync(0xffffffffu, n_inc, o);
    if (lane >= o) {
      q_inc += x;
      n_inc += y;
    }
  }
  if (lane == 31) {
    warp_q[warp] = q_inc;
    warp_n[warp] = n_inc;
  }
  __syncthreads();
  int q_base = q_inc - q_sum, n_base = n_inc - n_sum;
  for (int w = 0; w < warp; ++w) {
    q_base += warp_q[w];
    n_base += warp_n[w];
  }
  for (int r = r0; r < r1; ++r) {
    start[r] += q_base;
    first[r] += n_base;
  }
  if (tid == kTableThreads - 1) {
    start[R] = q_base + q_sum;
    first[R] = n_base + n_sum;
  }
  __syncthreads();
  const int total = start[R], pages = first[R];

  const int stride = gridDim.x * kTableThreads, at = blockIdx.x * kTableThreads + tid;
  for (int r = at; r <= R; r += stride) {
    a.query_start_loc[r] = start[r];
    if (r < R) a.seq_lens[r] = context[r] + (start[r + 1] - start[r]);
  }
  if (at == 0) *a.pages_taken = pages;
  for (int i = at; i < pages; i += stride) {
    const int r = owner(first, R, i);
    const int64_t col = (int64_t)pages_of(context[r], a.block_size) + (i - first[r]);
    if (col >= 0 && col < a.num_pages) a.block_table[(int64_t)r * a.block_table_row_stride + col] = i < a.num_free ? __ldg(a.free_blocks + i) : -1;
  }
  for (int t = at; t < a.num_tokens; t += stride) {
    int64_t slot = -1;
    int pos = 0;
    if (t < total) {
      const int r = owner(start, R, t);
      const int c = context[r];
      pos = c + (t - start[r]);
      const int col = (int)((uint32_t)pos / (uint32_t)a.block_size), old = pages_of(c, a.block_size);
      if ((uint32_t)col < (uint32_t)a.num_pages) {
        int block;
        if (col < old) {
          block = __ldg(a.block_table + (int64_t)r * a.block_table_row_stride + col);
        } else {
          const int i = first[r] + (col - old);
          block = (uint32_t)i < (uint32_t)a.num_free ? __ldg(a.free_blocks + i) : -1;
        }
        if (block >= 0) slot = (int64_t)block * a.block_size + (pos - col * a.block_size);
      }
    }
    a.slot_mapping[t] = slot;
    if (a.positions != nullptr) a.positions[t] = pos;
  }
}

}  // namespace

cudaError_t launch_page_tables(const PthB200TablesArgs& a, cudaStream_t stream) {
  const int smem = (3 * a.num_reqs + 2) * 4;  // 197 KB at the most requests
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    err = cudaFuncSetAttribute(page_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (3 * 16384 + 2) * 4);
    if (err != cudaSuccess) return err;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  // a thread per token as far as the SMs hold them at once: what a token waits for are two loads, one after the other
  const int ctas = (a.num_tokens + kTableThreads - 1) / kTableThreads;
  return pdl_launch(page_tables_kernel, dim3((unsigned)(ctas < 1 ? 1 : ctas > kMostCtas ? kMostCtas : ctas)), dim3(kTableThreads), smem, stream, a);
}

}  // namespace pthb200
