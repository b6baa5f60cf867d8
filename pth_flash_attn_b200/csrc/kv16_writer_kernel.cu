// Writer of the 16-bit paged cache: the K and V rows of new tokens, rounded to the cache's type, at the slots that
// slot_mapping names.  No arithmetic but the rounding (to nearest even, from 32 bits), so bytes bound it:
// T Hkv D (source + 2) x 2.
//
// A thread moves 16 bytes of the cache, eight elements of a row, at a time and has the loads of kWriteBatch such
// pieces in flight before it stores the first.  (With 1, 2 and 4, bf16 to bf16 behind a flush of L2, us: 4 x 2,048 tokens of 8 heads,
// 128 dims 21.5, 19.3, 19.4, 4 times as many 64.5, 53.2, 53.2, 64 tokens 7.0, 7.1, 9.0: with 4 registers spill.)
//
// Measured behind a flush of L2, the same heads, 4 x 2,048 tokens and 4 times as many: bf16 sources 18.4 and 53.2 us (the latter 5.0
// TB/s of what is read and written; copies move 6.56), fp32 24.5 and 69.6 (5.8 TB/s), fp16 to bf16, element by element, 22.5 and
// 63.5.  One call behind another 4 x 2,048 tokens take 10.8, 15.4 and 13.3: L2 holds what the last one wrote.  64 tokens take
// 2.0 to 2.5 us on the device and 5.7 for the host's call.
#include "kv16.cuh"
#include "pdl.cuh"

namespace pthb200 {
namespace {

constexpr int kWriteThreads = 256;
constexpr int kWriteBatch = 2;

struct WriteParams {
  const uint8_t* src[2];
  int64_t src_stride_token[2], src_stride_head[2];
  uint8_t* dst[2];
  int64_t dst_stride_block[2], dst_stride_slot[2], dst_stride_head[2];
  const int64_t* slot_mapping;
  int64_t slots;  // of the cache
  int32_t block_size, num_kv_heads, num_tokens;
  int32_t src_dtype, cache_dtype;
};

__device__ __forceinline__ float element(const uint8_t* p, int dtype) {
  if (dtype == PTH_ATTN_F32) return *reinterpret_cast<const float*>(p);
  if (dtype == PTH_ATTN_F16) return __half2float(*reinterpret_cast<const __half*>(p));
  return __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(p));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, int dtype) {
  if (dtype == PTH_ATTN_F16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Eight elements of a source row.  kSame: the cache's own type on 16-byte boundaries, moved as they are; kFloat: fp32
// on 16-byte boundaries; kAny: any type and alignment, element by element.
enum Source { kSame, kFloat, kAny };
template <Source kSource>
struct Eight {
  uint4 w[kSource == kFloat ? 2 : 1];
  __device__ __forceinline__ void load(const uint8_t* row, int e0, const WriteParams& p) {
    if constexpr (kSource == kSame) {
      w[0] = __ldg(reinterpret_cast<const uint4*>(row + e0 * 2));
    } else if constexpr (kSource == kFloat) {
      w[0] = __ldg(reinterpret_cast<const uint4*>(row + e0 * 4));
      w[1] = __ldg(reinterpret_cast<const uint4*>(row + e0 * 4) + 1);
    } else {
      const int es = p.src_dtype == PTH_ATTN_F32 ? 4 : 2;
      uint32_t r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        r[i] = pack2(element(row + (e0 + 2 * i) * es, p.src_dtype), element(row + (e0 + 2 * i + 1) * es, p.src_dtype), p.cache_dtype);
      w[0] = make_uint4(r[0], r[1], r[2], r[3]);
    }
  }
  __device__ __forceinline__ uint4 rounded(const WriteParams& p) const {
    if constexpr (kSource == kFloat) {
      const uint4 a = w[0], b = w[1];
      return make_uint4(pack2(__uint_as_float(a.x), __uint_as_float(a.y), p.cache_dtype),
                        pack2(__uint_as_float(a.z), __uint_as_float(a.w), p.cache_dtype),
                        pack2(__uint_as_float(b.x), __uint_as_float(b.y), p.cache_dtype),
                        pack2(__uint_as_float(b.z), __uint_as_float(b.w), p.cache_dtype));
    } else {
      return w[0];
    }
  }
};

// Pieces are numbered token-major: piece = ((token * 2 + (0 for K, 1 for V)) * Hkv + head) * (D / 8) + column.
template <int HD, Source kSource>
__global__ void __launch_bounds__(kWriteThreads) kv16_writer_kernel(const __grid_constant__ WriteParams p) {
  constexpr int kCols = HD / 8;
  const int64_t pieces = (int64_t)p.num_tokens * 2 * p.num_kv_heads * kCols;
  const int64_t base = (int64_t)blockIdx.x * (kWriteThreads * kWriteBatch) + threadIdx.x;
  pdl_wait();
  Eight<kSource> e[kWriteBatch];
  uint8_t* dst[kWriteBatch];
#pragma unroll
  for (int b = 0; b < kWriteBatch; ++b) {
    const int64_t i = base + b * kWriteThreads;
    dst[b] = nullptr;
    if (i >= pieces) continue;
    const int col = (int)(i % kCols);
    const int64_t row = i / kCols;
    int token, head, v;
    if (row <= 0xffffffffll) {
      const uint32_t half = (uint32_t)row / (uint32_t)p.num_kv_heads;
      head = (int)((uint32_t)row - half * (uint32_t)p.num_kv_heads);
      token = (int)(half >> 1);
      v = (int)(half & 1);
    } else {
      const int64_t half = row / p.num_kv_heads;
      head = (int)(row - half * p.num_kv_heads);
      token = (int)(half >> 1);
      v = (int)(half & 1);
    }
    const int64_t slot = __ldg(p.slot_mapping + token);
    if (slot < 0 || slot >= p.slots) continue;
    int64_t block;
    int at;
    if (slot <= 0xffffffffll) {
      block = (uint32_t)slot / (uint32_t)p.block_size;
      at = (int)((uint32_t)slot - (uint32_t)block * (uint32_t)p.block_size);
    } else {
      block = slot / p.block_size;
      at = (int)(slot - block * p.block_size);
    }
    e[b].load(p.src[v] + (int64_t)token * p.src_stride_token[v] + (int64_t)head * p.src_stride_head[v], col * 8, p);
    dst[b] = p.dst[v] + block * p.dst_stride_block[v] + (int64_t)at * p.dst_stride_slot[v] + (int64_t)head * p.dst_stride_head[v] + col * 16;
  }
#pragma unroll
  for (int b = 0; b < kWriteBatch; ++b)
    if (dst[b] != nullptr) *reinterpret_cast<uint4*>(dst[b]) = e[b].rounded(p);
}

template <int HD>
cudaError_t launch_for(const WriteParams& p, Source source, cudaStream_t stream) {
  const int64_t pieces = (int64_t)p.num_tokens * 2 * p.num_kv_heads * (HD / 8);
  const int64_t ctas = (pieces + kWriteThreads * kWriteBatch - 1) / (kWriteThreads * kWriteBatch);
  if (ctas > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const dim3 grid((unsigned)ctas);
  if (source == kSame) return pdl_launch(kv16_writer_kernel<HD, kSame>, grid, kWriteThreads, 0, stream, p);
  if (source == kFloat) return pdl_launch(kv16_writer_kernel<HD, kFloat>, grid, kWriteThreads, 0, stream, p);
  return pdl_launch(kv16_writer_kernel<HD, kAny>, grid, kWriteThreads, 0, stream, p);
}

}  // namespace

cudaError_t launch_kv16_writer(const PthB200Kv16WriteArgs& a, cudaStream_t stream) {
  WriteParams p;
  const PthAttnStream* cache[2] = {&a.k_cache, &a.v_cache};
  p.src[0] = static_cast<const uint8_t*>(a.key);
  p.src[1] = static_cast<const uint8_t*>(a.value);
  p.src_stride_token[0] = a.key_stride_token;
  p.src_stride_token[1] = a.value_stride_token;
  p.src_stride_head[0] = a.key_stride_head;
  p.src_stride_head[1] = a.value_stride_head;
  bool wide = true;  // every source row on a 16-byte boundary
  for (int i = 0; i < 2; ++i) {
    p.dst[i] = static_cast<uint8_t*>(const_cast<void*>(cache[i]->data));
    p.dst_stride_block[i] = cache[i]->stride_block;
    p.dst_stride_slot[i] = cache[i]->stride_slot;
    p.dst_stride_head[i] = cache[i]->stride_head;
    wide = wide && reinterpret_cast<uintptr_t>(p.src[i]) % 16 == 0 && p.src_stride_token[i] % 16 == 0 && p.src_stride_head[i] % 16 == 0;
  }
  p.slot_mapping = a.slot_mapping;
  p.slots = (int64_t)a.num_blocks * a.block_size;
  p.block_size = a.block_size;
  p.num_kv_heads = a.num_kv_heads;
  p.num_tokens = a.num_tokens;
  p.src_dtype = a.src_dtype;
  p.cache_dtype = a.cache_dtype;
  const Source source = !wide ? kAny : a.src_dtype == a.cache_dtype ? kSame : a.src_dtype == PTH_ATTN_F32 ? kFloat : kAny;
  switch (a.head_size) {
    case 64:
      return launch_for<64>(p, source, stream);
    case 128:
      return launch_for<128>(p, source, stream);
    default:
      return launch_for<256>(p, source, stream);
  }
}

}  // namespace pthb200
