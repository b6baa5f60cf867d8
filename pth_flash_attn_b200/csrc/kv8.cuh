// Parameters shared by the kernels of the 8-bit paged cache (include/pthb200_attn.h: pthb200_kv8_*), its number format, and the
// kernels' host-side launchers.
//
// A cell holds e4m3 numbers c; every `group` slots of a page share a scale per KV head and per K / V, so that an element is c x scale.
// group is a multiple of 16 and divides the page, so 16 keys whose first one's position is a multiple of 16 have one scale.
#pragma once

#include <cuda_fp8.h>

#include "kv16_sched.cuh"

namespace pthb200 {

struct Kv8Params : Kv16Params {
  const float* k_scale;
  const float* v_scale;
  int64_t scale_stride_block, scale_stride_group, scale_stride_head;   // of both, in elements
  int32_t scale_tokens;    // slots of a scale
  int32_t causal;
};

constexpr float kLargestE4m3 = 448.f;

namespace {

// Two numbers as e4m3, to nearest even, beyond the largest to the largest (infinities too); the first in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_of_f16x2(__half2 h) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<const uint32_t*>(&h)));
  return r;
}
// Two e4m3 numbers (of the low half of w) as fp16, which holds them all.
__device__ __forceinline__ uint32_t f16x2_of_e4m3x2(uint32_t w) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)w));
  return r;
}
__device__ __forceinline__ float2 float2_of_e4m3x2(uint32_t w) {
  const uint32_t h = f16x2_of_e4m3x2(w);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// Exponent of the smallest power of two with x <= 448 times it (448 = 1.75 x 2^8; x normal or zero).
__device__ __forceinline__ int e4m3_exponent(float x) {
  const uint32_t bits = __float_as_uint(x);
  return (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
}
// 2^e, e in [-126, 127].
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Instruction descriptor of tcgen05.mma.kind::f8f6f4 with e4m3 operands and an fp32 accumulator.
__host__ __device__ constexpr uint32_t instr_desc_e4m3(uint32_t m, uint32_t n, uint32_t a_mn, uint32_t b_mn) { return tc::instr_desc(m, n, 0, 0, a_mn, b_mn); }
__device__ __forceinline__ void mma_e4m3(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}

// NaN cells of a word: the top bit of their bytes.
__device__ __forceinline__ uint32_t nan_cells(uint32_t w) { return (w & 0x7f7f7f7fu) + 0x01010101u & 0x80808080u; }
// The same; they become zero.
__device__ __forceinline__ uint32_t take_nan(uint32_t& w) {
  const uint32_t nan = nan_cells(w);
  w &= ~((nan >> 7) * 0xffu);
  return nan;
}
// The block and slot of a key of a request; -1: there is none.
__device__ __forceinline__ int block_of(const Kv16Params& p, int r, int pos, int* slot) {
  const int page = pos / p.block_size;
  *slot = pos - page * p.block_size;
  const int blk = __ldg(p.block_table + (int64_t)r * p.block_table_row_stride + page);
  return (uint32_t)blk < (uint32_t)p.num_blocks ? blk : -1;
}

}  // namespace

// (Not in the unnamed namespace: the schedule's templates find these by their argument's namespace.)
// A request's query tokens and the keys that they see together.  Token i (of `all`) has position pos0 + i; tokens past the caller's
// bound are not computed.
struct ReqShape8 : ReqShape {
  int pos0;
};
__device__ __forceinline__ void kv8_tokens(const Kv8Params& p, int r, int* first, int* tokens, int* all) {
  if (p.query_start_loc == nullptr) {
    *first = r;
    *tokens = *all = 1;
    return;
  }
  *first = max(0, __ldg(p.query_start_loc + r));
  const int end = min(max(0, __ldg(p.query_start_loc + r + 1)), p.num_tokens);   // (so that the difference stays in 32 bits)
  *all = max(0, end - *first);
  *tokens = min(*all, p.max_query_len);
}
// Keys [lo, hi) that the token at position pos sees; seq: the request's length.
__device__ __forceinline__ int kv8_low(const Kv8Params& p, int pos) { return p.window > 0 ? max(0, max(pos, -1) - p.window + 1) : 0; }
__device__ __forceinline__ int kv8_high(const Kv8Params& p, int pos, int seq) { return max(0, min(p.causal ? pos + 1 : seq, p.most_keys)); }
template <int RP>
__device__ __forceinline__ ReqShape8 req_shape(const Kv8Params& p, int r) {
  ReqShape8 s;
  int all;
  const int seq = max(0, __ldg(p.seq_lens + r));
  kv8_tokens(p, r, &s.first, &s.tokens, &all);
  s.pos0 = seq - all;
  s.lo = kv8_low(p, s.pos0);
  s.hi = kv8_high(p, s.pos0 + s.tokens - 1, seq);
  const int rows = s.tokens * p.group;
  s.row_tiles = (rows + RP - 1) / RP;
  s.tiles = s.hi > s.lo && rows > 0 ? (s.hi + kTile - 1) / kTile - s.lo / kTile : 0;
  return s;
}
// What only the 8-bit kernels ask of a piece.
__device__ __forceinline__ void place_piece(Piece* out, const ReqShape8& s) { out->pos0 = s.pos0; }

// kv8_short_kernel.cu
int64_t kv8_short_workspace_bytes(int head_size, int num_sms);
cudaError_t launch_kv8_short(const Kv8Params& p, cudaStream_t stream);
cudaError_t launch_kv8_short_held(const Kv8Params& p, cudaStream_t stream);   // 128 dims, bf16, at most 8 rows
// kv8_tall_kernel.cu.  *taken: whether the cache's view can be read by TMA boxes; if not, nothing has been launched.
int64_t kv8_tall_workspace_bytes(int head_size, int num_sms);
cudaError_t launch_kv8_tall(const Kv8Params& p, cudaStream_t stream, bool* taken);
cudaError_t launch_kv8_tall_held(const Kv8Params& p, cudaStream_t stream);    // 128 dims, bf16
// kv8_writer_kernel.cu, kv8_reader_kernel.cu, rotary_kernel.cu
cudaError_t launch_kv8_writer(const PthB200Kv8WriteArgs& a, cudaStream_t stream);
cudaError_t launch_kv8_reader(const PthB200Kv8ReadArgs& a, cudaStream_t stream);
cudaError_t launch_rotary(const PthB200RotaryArgs& a, cudaStream_t stream);

}  // namespace pthb200
