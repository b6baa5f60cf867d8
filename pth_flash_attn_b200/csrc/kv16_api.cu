// C entries of the 16-bit paged cache (include/pthb200_attn.h): argument checks, each naming its field, and the
// launches.  Nothing here allocates, reads device memory or synchronises.
#include <algorithm>
#include <climits>
#include <cmath>

#include "kv16.cuh"

namespace pthb200 {
namespace {

#define KV16_REQUIRE(cond, msg)                               \
  do {                                                        \
    if (!(cond)) return set_error(PTH_ATTN_EINVAL, (msg));    \
  } while (0)

bool aligned(const void* ptr, int64_t a) { return reinterpret_cast<uintptr_t>(ptr) % (uintptr_t)a == 0; }
bool is_head_size(int32_t d) { return d == 64 || d == 128 || d == 256; }
bool is_16bit(int32_t t) { return t == PTH_ATTN_F16 || t == PTH_ATTN_BF16; }

template <class Args>
int32_t check_header(const Args* a, const char* type) {
  KV16_REQUIRE(a != nullptr, "args is NULL");
  KV16_REQUIRE(a->abi_version == PTH_ATTN_ABI_VERSION, "args.abi_version does not match the library");
  KV16_REQUIRE(a->struct_bytes == (int32_t)sizeof(Args), std::string("args.struct_bytes != sizeof(") + type + ")");
  return PTH_ATTN_OK;
}
int32_t check_rows(const void* data, int64_t stride_token, int64_t stride_head, int64_t align, const char* name) {
  const std::string n(name), a = std::to_string(align);
  KV16_REQUIRE(data != nullptr, n + " is NULL");
  KV16_REQUIRE(aligned(data, align), n + " must be " + a + "-byte aligned");
  KV16_REQUIRE(stride_token >= 0 && stride_head >= 0 && stride_token % align == 0 && stride_head % align == 0,
               n + " byte strides must be non-negative multiples of " + a);
  return PTH_ATTN_OK;
}
int32_t check_cache(const PthAttnStream& s, const char* name) {
  const std::string n(name);
  KV16_REQUIRE(s.data != nullptr, n + ".data is NULL");
  KV16_REQUIRE(aligned(s.data, 16), n + ".data must be 16-byte aligned");
  KV16_REQUIRE(s.stride_block >= 0 && s.stride_slot >= 0 && s.stride_head >= 0, n + " strides must be >= 0");
  KV16_REQUIRE(s.stride_block % 16 == 0 && s.stride_slot % 16 == 0 && s.stride_head % 16 == 0,
               n + " byte strides must be multiples of 16");
  return PTH_ATTN_OK;
}
int32_t launched(cudaError_t err, const char* what) {
  if (err != cudaSuccess) return set_error(PTH_ATTN_ECUDA, std::string(what) + " launch failed: " + cudaGetErrorString(err));
  return PTH_ATTN_OK;
}

int32_t build(const PthB200Kv16Args* a, bool cross, Kv16Params* p) {
  if (int32_t rc = check_header(a, "PthB200Kv16Args")) return rc;
  KV16_REQUIRE(is_16bit(a->dtype), "dtype must be F16 or BF16");
  KV16_REQUIRE(is_head_size(a->head_size), "head_size must be 64, 128 or 256");
  KV16_REQUIRE(a->num_kv_heads >= 1 && a->num_q_heads >= 1 && a->num_q_heads % a->num_kv_heads == 0,
               "num_q_heads must be a positive multiple of num_kv_heads");
  KV16_REQUIRE(a->num_q_heads / a->num_kv_heads <= 64, "num_q_heads / num_kv_heads must be <= 64");
  KV16_REQUIRE(a->num_reqs >= 0 && a->num_tokens >= 0, "num_reqs and num_tokens must be >= 0");
  KV16_REQUIRE(a->block_size >= 1 && a->num_blocks >= 1, "block_size and num_blocks must be >= 1");
  KV16_REQUIRE(std::isfinite(a->softmax_scale) && a->softmax_scale > 0.f, "softmax_scale must be finite and > 0");
  KV16_REQUIRE(a->window >= 0, "window must be >= 0");
  if (cross) {
    KV16_REQUIRE(a->query_start_loc != nullptr, "query_start_loc is NULL");
    KV16_REQUIRE(a->max_query_len >= 0 && a->max_query_len <= a->num_tokens, "max_query_len must be in [0, num_tokens]");
    KV16_REQUIRE(a->window == 0, "window must be 0 for cross attention");
  } else {
    KV16_REQUIRE(a->query_start_loc == nullptr, "query_start_loc must be NULL for decode");
    KV16_REQUIRE(a->num_tokens == a->num_reqs, "num_tokens must equal num_reqs for decode");
  }
  if (a->num_tokens == 0 || a->num_reqs == 0) return PTH_ATTN_OK;
  if (int32_t rc = check_rows(a->q, a->q_stride_token, a->q_stride_head, 16, "q")) return rc;
  if (int32_t rc = check_rows(a->out, a->out_stride_token, a->out_stride_head, 16, "out")) return rc;
  KV16_REQUIRE(aligned(a->lse, 4), "lse must be 4-byte aligned");
  if (int32_t rc = check_cache(a->k_cache, "k_cache")) return rc;
  if (int32_t rc = check_cache(a->v_cache, "v_cache")) return rc;
  KV16_REQUIRE(a->k_cache.stride_block == a->v_cache.stride_block && a->k_cache.stride_slot == a->v_cache.stride_slot &&
                   a->k_cache.stride_head == a->v_cache.stride_head,
               "k_cache and v_cache must have the same strides");
  KV16_REQUIRE(a->num_pages == 0 || a->block_table != nullptr, "block_table is NULL");
  KV16_REQUIRE(a->seq_lens != nullptr, "seq_lens is NULL");
  KV16_REQUIRE(a->block_table_row_stride >= 0 && a->num_pages >= 0, "block_table_row_stride and num_pages must be >= 0");
  KV16_REQUIRE(a->workspace != nullptr && aligned(a->workspace, 256), "workspace must not be NULL and 256-byte aligned");

  *p = Kv16Params{};
  p->q = static_cast<const uint8_t*>(a->q);
  p->q_stride_token = a->q_stride_token;
  p->q_stride_head = a->q_stride_head;
  p->out = static_cast<uint8_t*>(a->out);
  p->out_stride_token = a->out_stride_token;
  p->out_stride_head = a->out_stride_head;
  p->lse = a->lse;
  p->k = static_cast<const uint8_t*>(a->k_cache.data);
  p->v = static_cast<const uint8_t*>(a->v_cache.data);
  p->stride_block = a->k_cache.stride_block;
  p->stride_slot = a->k_cache.stride_slot;
  p->stride_head = a->k_cache.stride_head;
  p->block_table = a->block_table;
  p->block_table_row_stride = a->block_table_row_stride;
  p->seq_lens = a->seq_lens;
  p->query_start_loc = cross ? a->query_start_loc : nullptr;
  p->workspace = static_cast<uint8_t*>(a->workspace);
  p->dtype = a->dtype;
  p->block_size = a->block_size;
  p->block_shift = -1;
  for (int s = 0; s < 31; ++s)
    if ((1 << s) == a->block_size) p->block_shift = s;
  p->num_kv_heads = a->num_kv_heads;
  p->num_q_heads = a->num_q_heads;
  p->group = a->num_q_heads / a->num_kv_heads;
  p->head_size = a->head_size;
  p->num_blocks = a->num_blocks;
  p->most_keys = (int32_t)std::min<int64_t>((int64_t)a->num_pages * a->block_size, INT32_MAX - 1024);
  p->num_reqs = a->num_reqs;
  p->num_tokens = a->num_tokens;
  p->max_query_len = cross ? a->max_query_len : 1;
  p->window = a->window;
  p->scale_log2 = a->softmax_scale * 1.4426950408889634f;
  return PTH_ATTN_OK;
}

// Rows (query tokens x G) from which a launch of more than one token goes to the kernel with the rows on the MMA's M
// dimension.  Keys on M against rows on M, us:
//   rows  D 128, G 4: 8 x 500  8 x 4,000  64 x 500  64 x 4,000 keys   D 64, G 1: 64 x 500  64 x 4,000   D 256, G 4: 64 x 4,000
//     16         27 / 33      48 / 57      67 / 58     203 / 244             69 / 58     209 / 245             352 / 491
//     32         37 / 33      57 / 56     131 / 59     317 / 244            198 / 59     408 / 246             545 / 493
//     64         56 / 33      89 / 58     219 / 59     588 / 244            346 / 64     800 / 253           1,111 / 494
// Single tokens of wide groups stay with the keys on M, which divides few requests better: 8 x 4,000 keys, 32 heads of 1 KV head
// 55 / 68, 1 x 131,072, 64 of 2 183 / 243; 64 x 4,000, 64 of 2 88 / 83, and 64 x 8,000, 48 of 2 131 / 127.
constexpr int64_t kTallRows = 17;

int64_t workspace_bytes(int head_size, int num_sms) {
  return std::max(kv16_short_workspace_bytes(head_size, num_sms), kv16_tall_workspace_bytes(head_size, num_sms));
}

int32_t attention(const PthB200Kv16Args* a, bool cross, void* stream, Kv16Held held = kHeldNone, int32_t held_after = 0) {
  clear_error();
  Kv16Params p;
  if (int32_t rc = build(a, cross, &p)) return rc;
  if (a->num_tokens == 0 || a->num_reqs == 0 || (cross && a->max_query_len == 0)) return PTH_ATTN_OK;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return set_error(PTH_ATTN_ECUDA, "cannot query the current device");
  const int64_t need = workspace_bytes(a->head_size, sms);
  KV16_REQUIRE(a->workspace_bytes >= need, "workspace has " + std::to_string(a->workspace_bytes) + " bytes, " + std::to_string(need) + " are needed");
  const bool tall = (int64_t)p.max_query_len * p.group >= kTallRows && p.max_query_len > 1;
  if (held != kHeldNone) {
    KV16_REQUIRE(a->head_size == 128 && a->dtype == PTH_ATTN_BF16 && (tall || (int64_t)p.max_query_len * p.group <= 8),
                 "the test's instances take 128 dims, bf16, and at most 8 rows or more than 16");
    p.held_role = held;
    p.held_after = held_after;
    return launched((tall ? launch_kv16_tall_held : launch_kv16_short_held)(p, static_cast<cudaStream_t>(stream)), "attention");
  }
  return launched((tall ? launch_kv16_tall : launch_kv16_short)(p, static_cast<cudaStream_t>(stream)), "attention");
}

}  // namespace
}  // namespace pthb200

extern "C" {

int32_t pthb200_tables_args_bytes(void) { return (int32_t)sizeof(PthB200TablesArgs); }
int32_t pthb200_kv16_write_args_bytes(void) { return (int32_t)sizeof(PthB200Kv16WriteArgs); }
int32_t pthb200_kv16_args_bytes(void) { return (int32_t)sizeof(PthB200Kv16Args); }
int64_t pthb200_kv16_workspace_bytes(int32_t head_size, int32_t num_sms) {
  return pthb200::is_head_size(head_size) && num_sms >= 1 ? pthb200::workspace_bytes(head_size, num_sms) : -1;
}

int32_t pthb200_page_tables(const PthB200TablesArgs* a, void* stream) {
  using namespace pthb200;
  clear_error();
  if (int32_t rc = check_header(a, "PthB200TablesArgs")) return rc;
  KV16_REQUIRE(a->num_reqs >= 0 && a->num_reqs <= 16384, "num_reqs must be in [0, 16384]");
  KV16_REQUIRE(a->num_tokens >= 0 && a->num_free >= 0 && a->num_pages >= 0, "num_tokens, num_free and num_pages must be >= 0");
  KV16_REQUIRE(a->block_size >= 1, "block_size must be >= 1");
  KV16_REQUIRE(a->block_table_row_stride >= 0, "block_table_row_stride must be >= 0");
  KV16_REQUIRE(a->query_start_loc != nullptr && a->pages_taken != nullptr, "query_start_loc and pages_taken must not be NULL");
  KV16_REQUIRE(a->num_reqs == 0 || (a->context_lens != nullptr && a->query_lens != nullptr && a->seq_lens != nullptr),
               "context_lens, query_lens and seq_lens must not be NULL");
  KV16_REQUIRE(a->num_reqs == 0 || a->num_pages == 0 || a->block_table != nullptr, "block_table is NULL");
  KV16_REQUIRE(a->num_free == 0 || a->free_blocks != nullptr, "free_blocks is NULL");
  KV16_REQUIRE(a->num_tokens == 0 || a->slot_mapping != nullptr, "slot_mapping is NULL");
  KV16_REQUIRE(aligned(a->slot_mapping, 8) && aligned(a->positions, 8), "slot_mapping and positions must be 8-byte aligned");
  return launched(launch_page_tables(*a, static_cast<cudaStream_t>(stream)), "tables");
}

int32_t pthb200_kv16_write(const PthB200Kv16WriteArgs* a, void* stream) {
  using namespace pthb200;
  clear_error();
  if (int32_t rc = check_header(a, "PthB200Kv16WriteArgs")) return rc;
  KV16_REQUIRE(is_head_size(a->head_size), "head_size must be 64, 128 or 256");
  KV16_REQUIRE(a->num_kv_heads >= 1 && a->block_size >= 1 && a->num_blocks >= 1, "num_kv_heads, block_size and num_blocks must be >= 1");
  KV16_REQUIRE(a->num_tokens >= 0, "num_tokens must be >= 0");
  KV16_REQUIRE(a->src_dtype == PTH_ATTN_F32 || is_16bit(a->src_dtype), "src_dtype must be F32, F16 or BF16");
  KV16_REQUIRE(is_16bit(a->cache_dtype), "cache_dtype must be F16 or BF16");
  if (a->num_tokens == 0) return PTH_ATTN_OK;
  const int64_t elem = a->src_dtype == PTH_ATTN_F32 ? 4 : 2;
  if (int32_t rc = check_rows(a->key, a->key_stride_token, a->key_stride_head, elem, "key")) return rc;
  if (int32_t rc = check_rows(a->value, a->value_stride_token, a->value_stride_head, elem, "value")) return rc;
  if (int32_t rc = check_cache(a->k_cache, "k_cache")) return rc;
  if (int32_t rc = check_cache(a->v_cache, "v_cache")) return rc;
  KV16_REQUIRE(a->slot_mapping != nullptr && aligned(a->slot_mapping, 8), "slot_mapping must not be NULL and 8-byte aligned");
  return launched(launch_kv16_writer(*a, static_cast<cudaStream_t>(stream)), "writer");
}

int32_t pthb200_kv16_check(const PthB200Kv16Args* a) {
  pthb200::clear_error();
  pthb200::Kv16Params p;
  return pthb200::build(a, a != nullptr && a->query_start_loc != nullptr, &p);
}
int32_t pthb200_kv16_decode(const PthB200Kv16Args* a, void* stream) { return pthb200::attention(a, false, stream); }
int32_t pthb200_kv16_cross(const PthB200Kv16Args* a, void* stream) { return pthb200::attention(a, true, stream); }
int32_t pthb200_test_kv16_held(const PthB200Kv16Args* a, int32_t role, int32_t after, void* stream) {
  using namespace pthb200;
  clear_error();
  KV16_REQUIRE(a != nullptr, "args is NULL");
  KV16_REQUIRE(role >= kHeldSchedule && role <= kHeldMma && after >= 0, "role must be in [1, 3], after >= 0");
  return attention(a, a->query_start_loc != nullptr, stream, static_cast<Kv16Held>(role), after);
}

}  // extern "C"
