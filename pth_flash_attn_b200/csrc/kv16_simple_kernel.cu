// Attention over the 16-bit paged cache, one CTA per (query token, query head): the formula, on CUDA cores.
//
// A thread takes one of 128 keys at a time, the CTA keeps the running maximum m and sum l of the row's exponentials,
//   out = sum_j exp2(s_j - m) v_j / sum_j exp2(s_j - m),   s_j = scale log2(e) q . k_j,
// and thread d accumulates the columns d, d + 128 of the output.
#include "kv16.cuh"
#include "pdl.cuh"

namespace pthb200 {
namespace {

constexpr int kSimpleThreads = 128;

__device__ __forceinline__ float load16(const uint8_t* row, int d, int dtype) { return load_q_elem(row, d, dtype); }

__global__ void __launch_bounds__(kSimpleThreads) kv16_simple_kernel(const __grid_constant__ Kv16Params p) {
  __shared__ float q_s[256], p_s[kSimpleThreads], red[4];
  __shared__ int64_t off_s[kSimpleThreads];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = blockIdx.z, head = blockIdx.y, D = p.head_size, kvh = head / p.group;
  pdl_wait();
  int first, lo, hi;
  const int tokens = kv16_tokens(p, r, &first);
  if ((int)blockIdx.x >= tokens) return;
  const int token = first + blockIdx.x;
  kv16_visible(p, r, &lo, &hi);
  const uint8_t* q_row = p.q + (int64_t)token * p.q_stride_token + (int64_t)head * p.q_stride_head;
  for (int d = tid; d < D; d += kSimpleThreads) q_s[d] = load16(q_row, d, p.dtype) * p.scale_log2;
  __syncthreads();
  const int32_t* bt = p.block_table + (int64_t)r * p.block_table_row_stride;
  float m = -INFINITY, l = 0.f, acc[2] = {0.f, 0.f};
  for (int j0 = lo; j0 < hi; j0 += kSimpleThreads) {
    const int j = j0 + tid;
    float s = -INFINITY;
    if (j < hi) {
      const int64_t off = (int64_t)__ldg(bt + j / p.block_size) * p.stride_block + (int64_t)(j % p.block_size) * p.stride_slot +
                          (int64_t)kvh * p.stride_head;
      off_s[tid] = off;
      s = 0.f;
      for (int d = 0; d < D; ++d) s = fmaf(q_s[d], load16(p.k + off, d, p.dtype), s);
    }
    float mx = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) red[warp] = mx;
    __syncthreads();
    const float m_new = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = exp2f(m - m_use);
    p_s[tid] = exp2f(s - m_use);
    __syncthreads();
    l *= alpha;
    acc[0] *= alpha;
    acc[1] *= alpha;
    m = m_new;
    const int n = min(kSimpleThreads, hi - j0);
    for (int i = 0; i < n; ++i) {
      const float w = p_s[i];
      l += w;
      for (int c = 0; c < 2; ++c) {
        const int d = tid + c * kSimpleThreads;
        if (d < D) acc[c] = fmaf(w, load16(p.v + off_s[i], d, p.dtype), acc[c]);
      }
    }
    __syncthreads();
  }
  uint8_t* out = p.out + (int64_t)token * p.out_stride_token + (int64_t)head * p.out_stride_head;
  for (int c = 0; c < 2; ++c) {
    const int d = tid + c * kSimpleThreads;
    if (d < D) store_out_elem(out, d, p.dtype, l > 0.f || l != l ? acc[c] / l : 0.f);
  }
  if (tid == 0 && p.lse != nullptr) p.lse[(int64_t)token * p.num_q_heads + head] = l > 0.f || l != l ? (m + log2f(l)) * kLn2 : -INFINITY;
}

}  // namespace

int64_t kv16_workspace_bytes(int head_size, int num_sms) {
  (void)head_size;
  (void)num_sms;
  return 0;
}

cudaError_t launch_kv16_attention(const Kv16Params& p, cudaStream_t stream) {
  if (p.num_reqs > 65535 || p.num_q_heads > 65535) return cudaErrorInvalidConfiguration;
  return pdl_launch(kv16_simple_kernel, dim3(p.max_query_len, p.num_q_heads, p.num_reqs), dim3(kSimpleThreads), 0, stream, p);
}

}  // namespace pthb200
