// C entries of the 8-bit paged cache and of rotary positions (include/pthb200_attn.h): argument checks, each naming its
// field, and the launches.  Nothing here allocates, reads device memory or synchronises.
#include <algorithm>
#include <climits>
#include <cmath>

#include "kv8.cuh"

namespace pthb200 {
namespace {

#define KV8_REQUIRE(cond, msg)                                \
  do {                                                        \
    if (!(cond)) return set_error(PTH_ATTN_EINVAL, (msg));    \
  } while (0)

bool aligned(const void* ptr, int64_t a) { return reinterpret_cast<uintptr_t>(ptr) % (uintptr_t)a == 0; }
bool is_head_size(int32_t d) { return d == 64 || d == 128 || d == 256; }
bool is_16bit(int32_t t) { return t == PTH_ATTN_F16 || t == PTH_ATTN_BF16; }
bool is_float(int32_t t) { return t == PTH_ATTN_F32 || is_16bit(t); }
int64_t size_of(int32_t t) { return t == PTH_ATTN_F32 ? 4 : 2; }

template <class Args>
int32_t check_header(const Args* a, const char* type) {
  KV8_REQUIRE(a != nullptr, "args is NULL");
  KV8_REQUIRE(a->abi_version == PTH_ATTN_ABI_VERSION, "args.abi_version does not match the library");
  KV8_REQUIRE(a->struct_bytes == (int32_t)sizeof(Args), std::string("args.struct_bytes != sizeof(") + type + ")");
  return PTH_ATTN_OK;
}
int32_t check_rows(const void* data, int64_t stride_token, int64_t stride_head, int64_t align, const char* name) {
  const std::string n(name), a = std::to_string(align);
  KV8_REQUIRE(data != nullptr, n + " is NULL");
  KV8_REQUIRE(aligned(data, align), n + " must be " + a + "-byte aligned");
  KV8_REQUIRE(stride_token >= 0 && stride_head >= 0 && stride_token % align == 0 && stride_head % align == 0,
              n + " byte strides must be non-negative multiples of " + a);
  return PTH_ATTN_OK;
}
int32_t check_stream(const PthAttnStream& s, int64_t align, const char* name) {
  const std::string n(name), a = std::to_string(align);
  KV8_REQUIRE(s.data != nullptr, n + ".data is NULL");
  KV8_REQUIRE(aligned(s.data, align), n + ".data must be " + a + "-byte aligned");
  KV8_REQUIRE(s.stride_block >= 0 && s.stride_slot >= 0 && s.stride_head >= 0, n + " strides must be >= 0");
  KV8_REQUIRE(s.stride_block % align == 0 && s.stride_slot % align == 0 && s.stride_head % align == 0,
              n + " byte strides must be multiples of " + a);
  return PTH_ATTN_OK;
}
// What every call asks of its cache's shape, and of its cells and scales.
template <class Args>
int32_t check_shape(const Args* a) {
  KV8_REQUIRE(is_head_size(a->head_size), "head_size must be 64, 128 or 256");
  KV8_REQUIRE(a->num_kv_heads >= 1 && a->block_size >= 1 && a->num_blocks >= 1, "num_kv_heads, block_size and num_blocks must be >= 1");
  KV8_REQUIRE(a->num_kv_heads <= 65536, "num_kv_heads must be <= 65536");
  KV8_REQUIRE(a->scale_tokens >= 16 && a->scale_tokens % 16 == 0 && a->block_size % a->scale_tokens == 0,
              "scale_tokens must be a multiple of 16 that divides block_size");
  KV8_REQUIRE(a->num_reqs >= 0 && a->num_pages >= 0 && a->block_table_row_stride >= 0, "num_reqs, num_pages and block_table_row_stride must be >= 0");
  return PTH_ATTN_OK;
}
template <class Args>
int32_t check_cache(const Args* a, int64_t align) {
  if (int32_t rc = check_stream(a->k_cache, align, "k_cache")) return rc;
  if (int32_t rc = check_stream(a->v_cache, align, "v_cache")) return rc;
  if (int32_t rc = check_stream(a->k_scale, 4, "k_scale")) return rc;
  if (int32_t rc = check_stream(a->v_scale, 4, "v_scale")) return rc;
  KV8_REQUIRE(a->num_pages == 0 || a->block_table != nullptr, "block_table is NULL");
  return PTH_ATTN_OK;
}
int32_t launched(cudaError_t err, const char* what) {
  if (err != cudaSuccess) return set_error(PTH_ATTN_ECUDA, std::string(what) + " launch failed: " + cudaGetErrorString(err));
  return PTH_ATTN_OK;
}
bool same_strides(const PthAttnStream& a, const PthAttnStream& b) {
  return a.stride_block == b.stride_block && a.stride_slot == b.stride_slot && a.stride_head == b.stride_head;
}

int32_t build(const PthB200Kv8Args* a, bool decode, Kv8Params* p) {
  if (int32_t rc = check_header(a, "PthB200Kv8Args")) return rc;
  KV8_REQUIRE(is_16bit(a->dtype), "dtype must be F16 or BF16");
  if (int32_t rc = check_shape(a)) return rc;
  KV8_REQUIRE(a->num_q_heads >= 1 && a->num_q_heads % a->num_kv_heads == 0, "num_q_heads must be a positive multiple of num_kv_heads");
  KV8_REQUIRE(a->num_q_heads / a->num_kv_heads <= 64, "num_q_heads / num_kv_heads must be <= 64");
  KV8_REQUIRE(a->num_tokens >= 0, "num_tokens must be >= 0");
  KV8_REQUIRE(std::isfinite(a->softmax_scale) && a->softmax_scale > 0.f, "softmax_scale must be finite and > 0");
  KV8_REQUIRE(a->window >= 0, "window must be >= 0");
  if (decode) {
    KV8_REQUIRE(a->query_start_loc == nullptr, "query_start_loc must be NULL for decode");
    KV8_REQUIRE(a->num_tokens == a->num_reqs, "num_tokens must equal num_reqs for decode");
    KV8_REQUIRE(a->causal != 0, "causal must be 1 for decode");
  } else {
    KV8_REQUIRE(a->query_start_loc != nullptr, "query_start_loc is NULL");
    KV8_REQUIRE(a->max_query_len >= 0 && a->max_query_len <= a->num_tokens, "max_query_len must be in [0, num_tokens]");
  }
  if (a->num_tokens == 0 || a->num_reqs == 0) return PTH_ATTN_OK;
  if (int32_t rc = check_rows(a->q, a->q_stride_token, a->q_stride_head, 16, "q")) return rc;
  if (int32_t rc = check_rows(a->out, a->out_stride_token, a->out_stride_head, 16, "out")) return rc;
  KV8_REQUIRE(aligned(a->lse, 4), "lse must be 4-byte aligned");
  if (int32_t rc = check_cache(a, 16)) return rc;
  KV8_REQUIRE(same_strides(a->k_cache, a->v_cache), "k_cache and v_cache must have the same strides");
  KV8_REQUIRE(same_strides(a->k_scale, a->v_scale), "k_scale and v_scale must have the same strides");
  KV8_REQUIRE(a->seq_lens != nullptr, "seq_lens is NULL");
  KV8_REQUIRE(a->workspace != nullptr && aligned(a->workspace, 256), "workspace must not be NULL and 256-byte aligned");

  *p = Kv8Params{};
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
  p->k_scale = static_cast<const float*>(a->k_scale.data);
  p->v_scale = static_cast<const float*>(a->v_scale.data);
  p->scale_stride_block = a->k_scale.stride_block / 4;
  p->scale_stride_group = a->k_scale.stride_slot / 4;
  p->scale_stride_head = a->k_scale.stride_head / 4;
  p->scale_tokens = a->scale_tokens;
  p->causal = a->causal != 0;
  p->block_table = a->block_table;
  p->block_table_row_stride = a->block_table_row_stride;
  p->seq_lens = a->seq_lens;
  p->query_start_loc = a->query_start_loc;
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
  p->max_query_len = decode ? 1 : a->max_query_len;
  p->window = a->window;
  p->scale_log2 = a->softmax_scale * 1.4426950408889634f;
  return PTH_ATTN_OK;
}

// Rows (query tokens x G) from which a launch of more than one token goes to the kernel with the rows on the MMA's M
// dimension.  Keys on M against rows on M, us, four heads of a KV head:
//   rows   D 128: 8 x 500  8 x 4,000  64 x 500  64 x 4,000 keys   D 64: 64 x 500  64 x 4,000   D 256: 64 x 500  64 x 4,000
//     16         20 / 23      32 / 48      43 / 64     109 / 237           42 / 36     106 / 126        67 / 101    188 / 353
//     24         33 / 23      42 / 48      80 / 64     181 / 237                                       114 / 102    271 / 354
//     32         37 / 23      45 / 48      85 / 62     190 / 237           78 / 36     184 / 126       122 / 103    289 / 358
//     48         31 / 22      56 / 48     142 / 65     327 / 237
// Single tokens of wide groups stay with the keys on M, which divides few requests better.
int64_t tall_rows(int head_size) { return head_size == 64 ? 17 : 33; }

int64_t workspace_bytes(int head_size, int num_sms) {
  return std::max(kv8_short_workspace_bytes(head_size, num_sms), kv8_tall_workspace_bytes(head_size, num_sms));
}

int32_t attention(const PthB200Kv8Args* a, bool decode, void* stream, Kv16Held held = kHeldNone, int32_t held_after = 0) {
  clear_error();
  Kv8Params p;
  if (int32_t rc = build(a, decode, &p)) return rc;
  if (a->num_tokens == 0 || a->num_reqs == 0 || (!decode && a->max_query_len == 0)) return PTH_ATTN_OK;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return set_error(PTH_ATTN_ECUDA, "cannot query the current device");
  const int64_t need = workspace_bytes(a->head_size, sms);
  KV8_REQUIRE(a->workspace_bytes >= need, "workspace has " + std::to_string(a->workspace_bytes) + " bytes, " + std::to_string(need) + " are needed");
  const bool tall = (int64_t)p.max_query_len * p.group >= tall_rows(a->head_size) && p.max_query_len > 1;
  if (held != kHeldNone) {
    KV8_REQUIRE(a->head_size == 128 && a->dtype == PTH_ATTN_BF16 && (tall || (int64_t)p.max_query_len * p.group <= 8),
                "the test's instances take 128 dims, bf16, and at most 8 rows or more than 32");
    p.held_role = held;
    p.held_after = held_after;
    return launched((tall ? launch_kv8_tall_held : launch_kv8_short_held)(p, static_cast<cudaStream_t>(stream)), "attention");
  }
  if (tall) {
    bool taken = false;
    const int32_t rc = launched(launch_kv8_tall(p, static_cast<cudaStream_t>(stream), &taken), "attention");
    if (rc != PTH_ATTN_OK || taken) return rc;
  }
  return launched(launch_kv8_short(p, static_cast<cudaStream_t>(stream)), "attention");
}

}  // namespace
}  // namespace pthb200

extern "C" {

int32_t pthb200_kv8_write_args_bytes(void) { return (int32_t)sizeof(PthB200Kv8WriteArgs); }
int32_t pthb200_kv8_read_args_bytes(void) { return (int32_t)sizeof(PthB200Kv8ReadArgs); }
int32_t pthb200_kv8_args_bytes(void) { return (int32_t)sizeof(PthB200Kv8Args); }
int32_t pthb200_rotary_args_bytes(void) { return (int32_t)sizeof(PthB200RotaryArgs); }
int64_t pthb200_kv8_workspace_bytes(int32_t head_size, int32_t num_sms) {
  return pthb200::is_head_size(head_size) && num_sms >= 1 ? pthb200::workspace_bytes(head_size, num_sms) : -1;
}

int32_t pthb200_kv8_write(const PthB200Kv8WriteArgs* a, void* stream) {
  using namespace pthb200;
  clear_error();
  if (int32_t rc = check_header(a, "PthB200Kv8WriteArgs")) return rc;
  KV8_REQUIRE(is_float(a->src_dtype), "src_dtype must be F32, F16 or BF16");
  if (int32_t rc = check_shape(a)) return rc;
  KV8_REQUIRE(a->num_tokens >= 0 && a->max_query_len >= 0 && a->max_query_len <= a->num_tokens, "max_query_len must be in [0, num_tokens]");
  if (a->num_tokens == 0 || a->num_reqs == 0 || a->max_query_len == 0) return PTH_ATTN_OK;
  const int64_t elem = size_of(a->src_dtype);
  if (int32_t rc = check_rows(a->key, a->key_stride_token, a->key_stride_head, elem, "key")) return rc;
  if (int32_t rc = check_rows(a->value, a->value_stride_token, a->value_stride_head, elem, "value")) return rc;
  if (int32_t rc = check_cache(a, 8)) return rc;
  KV8_REQUIRE(a->seq_lens != nullptr && a->query_start_loc != nullptr, "seq_lens and query_start_loc must not be NULL");
  return launched(launch_kv8_writer(*a, static_cast<cudaStream_t>(stream)), "writer");
}

int32_t pthb200_kv8_read(const PthB200Kv8ReadArgs* a, void* stream) {
  using namespace pthb200;
  clear_error();
  if (int32_t rc = check_header(a, "PthB200Kv8ReadArgs")) return rc;
  KV8_REQUIRE(is_float(a->dst_dtype), "dst_dtype must be F32, F16 or BF16");
  if (int32_t rc = check_shape(a)) return rc;
  KV8_REQUIRE(a->num_rows >= 0 && a->max_rows >= 0 && a->max_rows <= a->num_rows, "max_rows must be in [0, num_rows]");
  if (a->num_rows == 0 || a->num_reqs == 0 || a->max_rows == 0) return PTH_ATTN_OK;
  if (int32_t rc = check_rows(a->key, a->key_stride_token, a->key_stride_head, 16, "key")) return rc;
  if (int32_t rc = check_rows(a->value, a->value_stride_token, a->value_stride_head, 16, "value")) return rc;
  if (int32_t rc = check_cache(a, 16)) return rc;
  KV8_REQUIRE(a->first != nullptr && a->row_start_loc != nullptr, "first and row_start_loc must not be NULL");
  return launched(launch_kv8_reader(*a, static_cast<cudaStream_t>(stream)), "reader");
}

int32_t pthb200_kv8_check(const PthB200Kv8Args* a) {
  pthb200::clear_error();
  pthb200::Kv8Params p;
  return pthb200::build(a, a != nullptr && a->query_start_loc == nullptr, &p);
}
int32_t pthb200_kv8_decode(const PthB200Kv8Args* a, void* stream) { return pthb200::attention(a, true, stream); }
int32_t pthb200_kv8_attend(const PthB200Kv8Args* a, void* stream) { return pthb200::attention(a, false, stream); }
int32_t pthb200_test_kv8_held(const PthB200Kv8Args* a, int32_t role, int32_t after, void* stream) {
  using namespace pthb200;
  clear_error();
  KV8_REQUIRE(a != nullptr, "args is NULL");
  KV8_REQUIRE(role >= kHeldSchedule && role <= kHeldMma && after >= 0, "role must be in [1, 3], after >= 0");
  return attention(a, a->query_start_loc == nullptr, stream, static_cast<Kv16Held>(role), after);
}

int32_t pthb200_rotary(const PthB200RotaryArgs* a, void* stream) {
  using namespace pthb200;
  clear_error();
  if (int32_t rc = check_header(a, "PthB200RotaryArgs")) return rc;
  KV8_REQUIRE(is_float(a->dtype), "dtype must be F32, F16 or BF16");
  KV8_REQUIRE(a->head_size >= 1 && a->head_size <= 1024, "head_size must be in [1, 1024]");
  KV8_REQUIRE(a->num_frequencies >= 1 && a->num_frequencies <= a->head_size / 2, "num_frequencies must be in [1, head_size / 2]");
  KV8_REQUIRE(a->num_tokens >= 0 && a->num_q_heads >= 0 && a->num_k_heads >= 0, "num_tokens, num_q_heads and num_k_heads must be >= 0");
  KV8_REQUIRE(((int64_t)a->num_q_heads + a->num_k_heads) * a->head_size < (1 << 28), "a token's heads must have fewer than 2^28 dimensions");
  KV8_REQUIRE(std::isfinite(a->scale), "scale must be finite");
  if (a->num_tokens == 0 || (a->num_q_heads == 0 && a->num_k_heads == 0)) return PTH_ATTN_OK;
  const int64_t elem = size_of(a->dtype);
  if (a->num_q_heads > 0) {
    if (int32_t rc = check_rows(a->q, a->q_stride_token, a->q_stride_head, elem, "q")) return rc;
    if (int32_t rc = check_rows(a->q_out, a->q_out_stride_token, a->q_out_stride_head, elem, "q_out")) return rc;
  }
  if (a->num_k_heads > 0) {
    if (int32_t rc = check_rows(a->k, a->k_stride_token, a->k_stride_head, elem, "k")) return rc;
    if (int32_t rc = check_rows(a->k_out, a->k_out_stride_token, a->k_out_stride_head, elem, "k_out")) return rc;
  }
  KV8_REQUIRE(a->positions != nullptr && aligned(a->positions, 8), "positions must not be NULL and 8-byte aligned");
  KV8_REQUIRE(a->frequencies != nullptr && aligned(a->frequencies, a->frequencies_64 ? 8 : 4), "frequencies must not be NULL and aligned");
  return launched(launch_rotary(*a, static_cast<cudaStream_t>(stream)), "rotary");
}

}  // extern "C"
