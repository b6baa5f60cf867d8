// Parameters shared by the kernels of the 16-bit paged cache (include/pthb200_attn.h: pthb200_page_tables,
// pthb200_kv16_*), and their host-side launchers.
#pragma once

#include <string>

#include "params.cuh"
#include "tcgen05.cuh"

namespace pthb200 {

struct Kv16Params {
  const uint8_t* q;
  int64_t q_stride_token, q_stride_head;
  uint8_t* out;
  int64_t out_stride_token, out_stride_head;
  float* lse;  // [num_tokens, num_q_heads] or nullptr
  const uint8_t* k;
  const uint8_t* v;
  int64_t stride_block, stride_slot, stride_head;  // of both
  const int32_t* block_table;
  int64_t block_table_row_stride;
  const int32_t* seq_lens;
  const int32_t* query_start_loc;  // nullptr: token r is request r's only one
  uint8_t* workspace;
  int32_t dtype;
  int32_t block_size, block_shift;  // block_shift: log2(block_size), -1 if it is not a power of two
  int32_t num_kv_heads, num_q_heads, group, head_size;
  int32_t num_reqs, num_tokens, max_query_len, window;
  int32_t num_blocks;
  int32_t most_keys;  // that a row of the block table has room for
  int32_t box_slots;  // slots of a TMA box (tall kernel; 0: none)
  int32_t out_wide;   // rows of out lie on 32-byte boundaries (tall kernel)
  float scale_log2;  // softmax_scale * log2(e)
  int32_t held_role, held_after;  // read by the test's instances alone
};
// The test's instances of the attention kernels leave out what one warp of CTA 0 does from some point on, so that the CTA's waits
// run out.
enum Kv16Held { kHeldNone = 0, kHeldSchedule = 1, kHeldCopies = 2, kHeldMma = 3 };
template <bool kHeld>
__device__ __forceinline__ bool kv16_held(const Kv16Params& p, Kv16Held role, uint32_t done) {
  return kHeld && blockIdx.x == 0 && p.held_role == role && done >= (uint32_t)p.held_after;
}

// The query tokens of a request (none past the caller's bound or the end of the token arrays), and its visible keys.
__device__ __forceinline__ int kv16_tokens(const Kv16Params& p, int r, int* first) {
  if (p.query_start_loc == nullptr) {
    *first = r;
    return 1;
  }
  *first = max(0, __ldg(p.query_start_loc + r));
  const int end = min(max(0, __ldg(p.query_start_loc + r + 1)), p.num_tokens);   // (so that the difference stays in 32 bits)
  return max(0, min(end - *first, p.max_query_len));
}
__device__ __forceinline__ void kv16_visible(const Kv16Params& p, int r, int* lo, int* hi) {
  *hi = max(0, min(__ldg(p.seq_lens + r), p.most_keys));
  *lo = p.window > 0 ? max(0, *hi - p.window) : 0;
}

// ---- shared memory images and waits of the tensor-core kernels ----

// Shared-memory operand descriptor, rows of 128 bytes in the 128-byte swizzle (chunk c of 16 bytes of row r lies at
// chunk c ^ (r & 7)): groups of 8 rows are 1,024 bytes.  K-major: sbo = next 8 rows.  MN-major (the row is a K index and
// holds 64 elements of M / N): sbo = next 8 rows, lbo = next 64 elements.
__device__ __forceinline__ uint64_t swizzled_desc(uint32_t saddr, uint32_t lbo_bytes, uint32_t sbo_bytes) {
  return tc::smem_desc(saddr, lbo_bytes, sbo_bytes) | (uint64_t)2 << 61;
}
// Bounded wait for a phase of an mbarrier; once any wait of the CTA has given up, all do.  A try sleeps for one microsecond, or for
// four where all warps of a CTA wait, so the bound is 0.3 to 1.1 s, or as many times that as the caller says, who may wait for other
// warps' whole pieces (20 million keys in one piece take 0.3 s).  (A test goes first: a try that may sleep takes 200 cycles where
// the phase is complete already, a test 100, and a softmax step has little else to wait for.)
constexpr uint32_t kWaitTries = 1u << 18;
template <uint32_t kTimes = 1>
__device__ __forceinline__ bool kv16_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (tc::mbar_test_wait(bar, parity)) return true;
#pragma unroll 1
  for (uint32_t i = 0; i < kTimes * kWaitTries; ++i) {
    if (tc::mbar_try_wait_hint(bar, parity, 1000u)) return true;
    if (*abort_flag) return false;
  }
  *abort_flag = 1;
  return false;
}
// Wait for what is in flight when a CTA leaves behind a wait that gave up: for 20 to 70 ms at most, whatever the flag says.
__device__ __forceinline__ void kv16_drain(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
  for (uint32_t i = 0; i < (1u << 14) && !tc::mbar_try_wait_hint(bar, parity, 1000u); ++i) {
  }
}
// Asynchronous copy of 16 bytes, or of none: then the destination is zeroed.
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
// One arrival on the barrier when this thread's copies so far have landed (it counts like any other arrival).
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void copies_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ float kv16_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A sum under a weight.  Weights are above zero: one that has run out of exponents leaves an infinite sum as it is.
__device__ __forceinline__ float weighed(float sum, float w) { return w == 0.f && isinf(sum) ? sum : sum * w; }

// launcher.cu: the calling thread's error text.
int32_t clear_error();
int32_t set_error(int32_t code, const std::string& msg);

// kv16_short_kernel.cu, kv16_tall_kernel.cu
int64_t kv16_short_workspace_bytes(int head_size, int num_sms);
int64_t kv16_tall_workspace_bytes(int head_size, int num_sms);
cudaError_t launch_kv16_short(const Kv16Params& p, cudaStream_t stream);
cudaError_t launch_kv16_tall(const Kv16Params& p, cudaStream_t stream);
cudaError_t launch_kv16_short_held(const Kv16Params& p, cudaStream_t stream);   // 128 dims, bf16, at most 8 rows
cudaError_t launch_kv16_tall_held(const Kv16Params& p, cudaStream_t stream);    // 128 dims, bf16
cudaError_t launch_kv16_writer(const PthB200Kv16WriteArgs& a, cudaStream_t stream);
cudaError_t launch_page_tables(const PthB200TablesArgs& a, cudaStream_t stream);

}  // namespace pthb200
