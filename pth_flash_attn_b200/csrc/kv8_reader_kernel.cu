// Reader of the 8-bit paged cache: a run of positions of each request back into rows of 32 or 16 bits, c x scale rounded once.
// Bytes bound it: Hkv D (1 + size) x 2 per row.
//
// A CTA takes kRows rows.  A warp finds their requests and blocks first, a row a lane; then all threads move pieces of 16 cells,
// kBatch of them in flight, neighbours side by side in memory.  16 requests' 161,568 rows of 8 heads, 128 dims, to fp16, 0.99 GB: 163 us, 0.93 of
// the copy bandwidth.
#include "kv8.cuh"

#include "page_copy.cuh"
#include "pdl.cuh"

namespace pthb200 {
namespace {

constexpr int kThreads = 256, kBatch = 4;

struct Read8Params {
  uint8_t* dst[2];
  int64_t dst_stride_token[2], dst_stride_head[2];
  const uint8_t* cache[2];
  int64_t stride_block[2], stride_slot[2], stride_head[2];
  const float* scale[2];
  int64_t scale_stride_block[2], scale_stride_group[2], scale_stride_head[2];   // in elements
  const int32_t* block_table;
  int64_t block_table_row_stride;
  const int32_t* first;
  const int32_t* row_start_loc;
  int32_t num_blocks, block_size, scale_tokens, num_kv_heads, num_reqs, num_rows, num_pages, max_rows;
  bool wide;   // destination rows lie on 32-byte boundaries
};

// Where a row comes from.
struct Place {
  int block, slot;   // block -1: there is no such cell; -2: the row belongs to no request
};
// Of the lane's row; the warp's rows are row0 + lane.
__device__ __forceinline__ Place place_of(const Read8Params& p, int row0, int rows) {
  // the last request that begins at or in front of the first row, 32 at a time; the others' follow close behind
  const int lane = threadIdx.x & 31, row = row0 + lane;
  int lo = 0, hi = p.num_reqs;
#pragma unroll 1
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    const uint32_t before = __ballot_sync(0xffffffffu, at < hi && __ldg(p.row_start_loc + at) <= row0);
    const int last = before == 0 ? 0 : 31 - __clz(before);
    hi = min(hi, lo + (last + 1) * step);
    lo += last * step;
  }
  if (lane >= rows) return Place{-2, 0};
  // (steps that grow, then halves: requests without rows may lie between)
  int r = lo, above = lo + 1;
#pragma unroll 1
  for (int step = 1; above < p.num_reqs && __ldg(p.row_start_loc + above) <= row; step *= 2) {
    r = above;
    above = step < p.num_reqs - above ? above + step : p.num_reqs;
  }
#pragma unroll 1
  while (above - r > 1) {
    const int middle = r + (above - r) / 2;
    if (__ldg(p.row_start_loc + middle) <= row) r = middle; else above = middle;
  }
  const int start = __ldg(p.row_start_loc + r), end = __ldg(p.row_start_loc + r + 1);
  if (row < start || row >= end || (long long)row - start >= p.max_rows) return Place{-2, 0};
  const long long pos = (long long)__ldg(p.first + r) + ((long long)row - start);
  if (pos < 0 || pos / p.block_size >= p.num_pages) return Place{-1, 0};
  const int page = (int)(pos / p.block_size), block = __ldg(p.block_table + (int64_t)r * p.block_table_row_stride + page);
  return Place{(uint32_t)block < (uint32_t)p.num_blocks ? block : -1, (int)(pos - (long long)page * p.block_size)};
}

// 16 cells times their scale.  wide: rows lie on 32-byte boundaries.
template <int kDtype>
__device__ __forceinline__ void store16(uint8_t* to, uint4 cells, float scale, bool wide) {
  constexpr int kWords = kDtype == PTH_ATTN_F32 ? 16 : 8;
  const uint32_t w[4] = {cells.x, cells.y, cells.z, cells.w};
  uint32_t o[kWords];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = float2_of_e4m3x2(w[i] & 0xffffu), b = float2_of_e4m3x2(w[i] >> 16);
    if constexpr (kDtype == PTH_ATTN_F32) {
      o[4 * i] = __float_as_uint(a.x * scale), o[4 * i + 1] = __float_as_uint(a.y * scale);
      o[4 * i + 2] = __float_as_uint(b.x * scale), o[4 * i + 3] = __float_as_uint(b.y * scale);
    } else {
      o[2 * i] = pack16<kDtype == PTH_ATTN_F16>(a.x * scale, a.y * scale);
      o[2 * i + 1] = pack16<kDtype == PTH_ATTN_F16>(b.x * scale, b.y * scale);
    }
  }
#pragma unroll
  for (int i = 0; i < kWords; i += 8) {
    if (wide) {
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to + i * 4), "r"(o[i]), "r"(o[i + 1]), "r"(o[i + 2]), "r"(o[i + 3]),
                   "r"(o[i + 4]), "r"(o[i + 5]), "r"(o[i + 6]), "r"(o[i + 7])
                   : "memory");
    } else {
      *reinterpret_cast<uint4*>(to + i * 4) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
      *reinterpret_cast<uint4*>(to + i * 4 + 16) = make_uint4(o[i + 4], o[i + 5], o[i + 6], o[i + 7]);
    }
  }
}

template <int HD, int kDtype, int kRows>
__global__ void __launch_bounds__(kThreads) kv8_reader_kernel(const __grid_constant__ Read8Params p) {
  constexpr int kCols = HD / 16, kSize = kDtype == PTH_ATTN_F32 ? 4 : 2;
  __shared__ Place places[kRows];
  const int row0 = (int)blockIdx.x * kRows, rows = min(kRows, p.num_rows - row0);
  pdl_wait();
  if (threadIdx.x < 32) {
    const Place place = place_of(p, row0, rows);
    if (threadIdx.x < rows) places[threadIdx.x] = place;
  }
  __syncthreads();
  // pieces: (row, K or V, head, column), the last fastest
  const int pieces = rows * 2 * p.num_kv_heads * kCols;
#pragma unroll 1
  for (int i0 = threadIdx.x; i0 < pieces; i0 += kThreads * kBatch) {
    uint4 w[kBatch];
    float scale[kBatch];
    uint8_t* to[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int i = i0 + b * kThreads;
      to[b] = nullptr;
      w[b] = make_uint4(0u, 0u, 0u, 0u);
      scale[b] = 0.f;
      if (i >= pieces) continue;
      const int col = i % kCols, x = i / kCols;
      const uint32_t pair = (uint32_t)x / (uint32_t)p.num_kv_heads, head = (uint32_t)x - pair * (uint32_t)p.num_kv_heads, row = pair >> 1, v = pair & 1;
      const Place at = places[row];
      if (at.block == -2) continue;
      to[b] = p.dst[v] + (int64_t)(row0 + (int)row) * p.dst_stride_token[v] + (int64_t)head * p.dst_stride_head[v] + col * 16 * kSize;
      if (at.block < 0) continue;
      w[b] = __ldg(reinterpret_cast<const uint4*>(p.cache[v] + (int64_t)at.block * p.stride_block[v] + (int64_t)at.slot * p.stride_slot[v] + (int64_t)head * p.stride_head[v]) + col);
      scale[b] = __ldg(p.scale[v] + (int64_t)at.block * p.scale_stride_block[v] + (int64_t)((uint32_t)at.slot / (uint32_t)p.scale_tokens) * p.scale_stride_group[v] + (int64_t)head * p.scale_stride_head[v]);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (to[b] != nullptr) store16<kDtype>(to[b], w[b], scale[b], p.wide);
  }
}

template <int HD, int kDtype>
cudaError_t launch_for(const Read8Params& p, cudaStream_t stream) {
  // rows of a CTA: four where there are too few to give every SM several CTAs of sixteen
  const int rows = p.num_rows >= 16 * sm_count() * 4 ? 16 : 4;
  const dim3 grid((unsigned)((p.num_rows + rows - 1) / rows));
  return pdl_launch(rows == 16 ? kv8_reader_kernel<HD, kDtype, 16> : kv8_reader_kernel<HD, kDtype, 4>, grid, kThreads, 0, stream, p);
}
template <int HD>
cudaError_t launch_type(const Read8Params& p, int dtype, cudaStream_t stream) {
  if (dtype == PTH_ATTN_F32) return launch_for<HD, PTH_ATTN_F32>(p, stream);
  if (dtype == PTH_ATTN_F16) return launch_for<HD, PTH_ATTN_F16>(p, stream);
  return launch_for<HD, PTH_ATTN_BF16>(p, stream);
}

}  // namespace

cudaError_t launch_kv8_reader(const PthB200Kv8ReadArgs& a, cudaStream_t stream) {
  Read8Params p{};
  const PthAttnStream* cache[2] = {&a.k_cache, &a.v_cache};
  const PthAttnStream* scale[2] = {&a.k_scale, &a.v_scale};
  p.dst[0] = static_cast<uint8_t*>(a.key);
  p.dst[1] = static_cast<uint8_t*>(a.value);
  p.dst_stride_token[0] = a.key_stride_token;
  p.dst_stride_token[1] = a.value_stride_token;
  p.dst_stride_head[0] = a.key_stride_head;
  p.dst_stride_head[1] = a.value_stride_head;
  p.wide = true;
  for (int i = 0; i < 2; ++i) {
    p.wide = p.wide && reinterpret_cast<uintptr_t>(p.dst[i]) % 32 == 0 && p.dst_stride_token[i] % 32 == 0 && p.dst_stride_head[i] % 32 == 0;
    p.cache[i] = static_cast<const uint8_t*>(cache[i]->data);
    p.stride_block[i] = cache[i]->stride_block;
    p.stride_slot[i] = cache[i]->stride_slot;
    p.stride_head[i] = cache[i]->stride_head;
    p.scale[i] = static_cast<const float*>(scale[i]->data);
    p.scale_stride_block[i] = scale[i]->stride_block / 4;
    p.scale_stride_group[i] = scale[i]->stride_slot / 4;
    p.scale_stride_head[i] = scale[i]->stride_head / 4;
  }
  p.block_table = a.block_table;
  p.block_table_row_stride = a.block_table_row_stride;
  p.first = a.first;
  p.row_start_loc = a.row_start_loc;
  p.num_blocks = a.num_blocks;
  p.block_size = a.block_size;
  p.scale_tokens = a.scale_tokens;
  p.num_kv_heads = a.num_kv_heads;
  p.num_reqs = a.num_reqs;
  p.num_rows = a.num_rows;
  p.num_pages = a.num_pages;
  p.max_rows = a.max_rows;
  switch (a.head_size) {
    case 64:
      return launch_type<64>(p, a.dst_dtype, stream);
    case 128:
      return launch_type<128>(p, a.dst_dtype, stream);
    default:
      return launch_type<256>(p, a.dst_dtype, stream);
  }
}

}  // namespace pthb200
