// How cells and scales of the 8-bit paged cache get to shared memory: TMA boxes of a page's slots, 4-byte copies.
#pragma once

#include "kv8.cuh"
#include "page_copy.cuh"

namespace pthb200 {
namespace {

// Tiled TMA load of one box of a rank-4 tensor map into shared memory.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(tc::smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
// Tensor map over one of the caches, [dims][heads][slots][blocks], a box being up to 128 dims of `slots` slots of one head, swizzled by its
// rows.  False: the driver refuses the view, or it is broadcast along a dimension (a stride of 0), which boxes are not asked for.  A dimension of one entry may
// have any stride: it gets a valid one.  (Encoded for every call: a microsecond of the host.)
bool cell_box_map(const Kv8Params& p, const uint8_t* base, int slots, CUtensorMap* map) {
  const EncodeTiledFn fn = encode_tiled_fn();
  const cuuint64_t dims[4] = {(cuuint64_t)p.head_size, (cuuint64_t)p.num_kv_heads, (cuuint64_t)p.block_size, (cuuint64_t)p.num_blocks};
  cuuint64_t strides[3] = {(cuuint64_t)p.stride_head, (cuuint64_t)p.stride_slot, (cuuint64_t)p.stride_block};
  for (int i = 0; i < 3; ++i) {
    if (dims[i + 1] == 1) strides[i] = (cuuint64_t)p.head_size;
    if (strides[i] == 0) return false;
  }
  const cuuint32_t box[4] = {(cuuint32_t)(p.head_size < 128 ? 64 : 128), 1, (cuuint32_t)slots, 1}, elem[4] = {1, 1, 1, 1};
  return fn != nullptr && fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<uint8_t*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                             p.head_size < 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
}  // namespace pthb200
