// The torch ops of the 16-bit paged cache (pth_flash_attn::page_tables, kv16_write, kv16_decode_attention,
// kv16_cross_attention): argument checks, then the C ABI of libpthb200_attn.so.  Registered for the CUDA and CPU keys
// through the libtorch stable ABI, like the op of torch_op.cpp; on the CPU key a call raises behind its checks.
// Nothing here allocates, reads device data on the host or synchronises.
#include "torch_check.h"

namespace {

// k_cache / v_cache [NB, BS, Hkv, D] of one 16-bit type.
void check_caches(const Check& c, const Tensor& k_cache, const Tensor& v_cache) {
  c.rank(k_cache, 4, "k_cache");
  c.rank(v_cache, 4, "v_cache");
  STD_TORCH_CHECK(k_cache.scalar_type() == ScalarType::BFloat16 || k_cache.scalar_type() == ScalarType::Half, c.op,
                  "k_cache must be bfloat16 or float16, got ", type_name(k_cache.scalar_type()));
  c.dtype(v_cache, k_cache.scalar_type(), "v_cache (same dtype as k_cache)");
  const int64_t D = k_cache.size(3);
  STD_TORCH_CHECK(D == 64 || D == 128 || D == 256, c.op, "head size D = k_cache.size(3) must be 64, 128 or 256, got ", D);
  STD_TORCH_CHECK(k_cache.size(0) >= 1 && k_cache.size(1) >= 1 && k_cache.size(2) >= 1, c.op, "k_cache must not be empty");
  c.size(v_cache, 0, k_cache.size(0), "v_cache", "NB");
  c.size(v_cache, 1, k_cache.size(1), "v_cache", "BS");
  c.size(v_cache, 2, k_cache.size(2), "v_cache", "Hkv");
  c.size(v_cache, 3, D, "v_cache", "D");
  c.inner(k_cache, "k_cache");
  c.inner(v_cache, "v_cache");
  c.count(k_cache.size(0), "NB");
  c.count(k_cache.size(1), "BS");
  c.count(k_cache.size(2), "Hkv");
}

void page_tables(const Tensor& context_lens, const Tensor& query_lens, const Tensor& free_blocks, Tensor& block_table,
                 Tensor& seq_lens, Tensor& query_start_loc, Tensor& slot_mapping, Tensor& positions, Tensor& pages_taken,
                 int64_t block_size) {
  const Check c{"page_tables: "};
  c.vector(context_lens, ScalarType::Int, "context_lens");
  c.vector(query_lens, ScalarType::Int, "query_lens");
  c.vector(free_blocks, ScalarType::Int, "free_blocks");
  c.rank(block_table, 2, "block_table");
  c.dtype(block_table, ScalarType::Int, "block_table");
  c.inner(block_table, "block_table");
  c.vector(seq_lens, ScalarType::Int, "seq_lens");
  c.vector(query_start_loc, ScalarType::Int, "query_start_loc");
  c.vector(slot_mapping, ScalarType::Long, "slot_mapping");
  c.vector(positions, ScalarType::Long, "positions");
  c.vector(pages_taken, ScalarType::Int, "pages_taken");
  const int64_t R = context_lens.size(0);
  c.size(query_lens, 0, R, "query_lens", "num_reqs");
  c.size(seq_lens, 0, R, "seq_lens", "num_reqs");
  c.size(query_start_loc, 0, R + 1, "query_start_loc", "num_reqs + 1");
  c.size(pages_taken, 0, 1, "pages_taken", "1");
  STD_TORCH_CHECK(block_table.size(0) >= R, c.op, "block_table has ", block_table.size(0), " rows, fewer than num_reqs = ", R);
  if (positions.size(0) != 0) c.size(positions, 0, slot_mapping.size(0), "positions", "slot_mapping.size(0)");
  STD_TORCH_CHECK(block_size >= 1 && block_size <= INT32_MAX, c.op, "block_size must be >= 1, got ", block_size);
  c.count(R, "num_reqs");
  c.count(slot_mapping.size(0), "slot_mapping.size(0)");
  c.count(free_blocks.size(0), "free_blocks.size(0)");
  c.count(block_table.size(1), "block_table.size(1)");
  const Tensor* others[] = {&query_lens, &free_blocks, &block_table, &seq_lens, &query_start_loc, &slot_mapping, &positions, &pages_taken};
  const char* names[] = {"query_lens", "free_blocks", "block_table", "seq_lens", "query_start_loc", "slot_mapping", "positions", "pages_taken"};
  for (int i = 0; i < 8; ++i) c.device(*others[i], context_lens, names[i], "context_lens");
  int32_t device = 0;
  void* stream = c.stream(context_lens, &device);
  PthB200TablesArgs a = new_args<PthB200TablesArgs>();
  a.context_lens = static_cast<const int32_t*>(context_lens.data_ptr());
  a.query_lens = static_cast<const int32_t*>(query_lens.data_ptr());
  a.free_blocks = static_cast<const int32_t*>(free_blocks.data_ptr());
  a.block_table = static_cast<int32_t*>(block_table.data_ptr());
  a.block_table_row_stride = block_table.stride(0);
  a.seq_lens = static_cast<int32_t*>(seq_lens.data_ptr());
  a.query_start_loc = static_cast<int32_t*>(query_start_loc.data_ptr());
  a.slot_mapping = static_cast<int64_t*>(slot_mapping.data_ptr());
  a.positions = positions.size(0) != 0 ? static_cast<int64_t*>(positions.data_ptr()) : nullptr;
  a.pages_taken = static_cast<int32_t*>(pages_taken.data_ptr());
  a.num_reqs = static_cast<int32_t>(R);
  a.num_tokens = static_cast<int32_t>(slot_mapping.size(0));
  a.num_free = static_cast<int32_t>(free_blocks.size(0));
  a.num_pages = static_cast<int32_t>(block_table.size(1));
  a.block_size = static_cast<int32_t>(block_size);
  const torch::stable::accelerator::DeviceGuard guard(device);
  c.done(pthb200_page_tables(&a, stream));
}

void kv16_write(const Tensor& key, const Tensor& value, Tensor& k_cache, Tensor& v_cache, const Tensor& slot_mapping) {
  const Check c{"kv16_write: "};
  check_caches(c, k_cache, v_cache);
  c.rank(key, 3, "key");
  c.rank(value, 3, "value");
  STD_TORCH_CHECK(key.scalar_type() == ScalarType::Float || key.scalar_type() == ScalarType::BFloat16 || key.scalar_type() == ScalarType::Half,
                  c.op, "key must be float32, bfloat16 or float16, got ", type_name(key.scalar_type()));
  c.dtype(value, key.scalar_type(), "value (same dtype as key)");
  const int64_t T = key.size(0), Hkv = k_cache.size(2), D = k_cache.size(3);
  c.size(key, 1, Hkv, "key", "Hkv");
  c.size(key, 2, D, "key", "D");
  c.size(value, 0, T, "value", "T");
  c.size(value, 1, Hkv, "value", "Hkv");
  c.size(value, 2, D, "value", "D");
  c.inner(key, "key");
  c.inner(value, "value");
  c.vector(slot_mapping, ScalarType::Long, "slot_mapping");
  c.size(slot_mapping, 0, T, "slot_mapping", "T");
  c.count(T, "T");
  c.device(value, key, "value", "key");
  c.device(k_cache, key, "k_cache", "key");
  c.device(v_cache, key, "v_cache", "key");
  c.device(slot_mapping, key, "slot_mapping", "key");
  int32_t device = 0;
  void* stream = c.stream(key, &device);
  PthB200Kv16WriteArgs a = new_args<PthB200Kv16WriteArgs>();
  a.key = key.data_ptr();
  a.value = value.data_ptr();
  a.src_dtype = type_code(key.scalar_type());
  a.cache_dtype = type_code(k_cache.scalar_type());
  a.key_stride_token = bytes(key, 0);
  a.key_stride_head = bytes(key, 1);
  a.value_stride_token = bytes(value, 0);
  a.value_stride_head = bytes(value, 1);
  a.k_cache = as_stream(k_cache);
  a.v_cache = as_stream(v_cache);
  a.slot_mapping = static_cast<const int64_t*>(slot_mapping.data_ptr());
  a.num_blocks = static_cast<int32_t>(k_cache.size(0));
  a.block_size = static_cast<int32_t>(k_cache.size(1));
  a.num_kv_heads = static_cast<int32_t>(Hkv);
  a.head_size = static_cast<int32_t>(D);
  a.num_tokens = static_cast<int32_t>(T);
  const torch::stable::accelerator::DeviceGuard guard(device);
  c.done(pthb200_kv16_write(&a, stream));
}

// What both attention calls ask of their tensors, and the arguments that they share.
PthB200Kv16Args attention_args(const Check& c, Tensor& out, Tensor& lse, const Tensor& q, const Tensor& k_cache, const Tensor& v_cache,
                               const Tensor& block_table, const Tensor& seq_lens, double softmax_scale, Tensor& workspace) {
  c.rank(q, 3, "q");
  check_caches(c, k_cache, v_cache);
  c.dtype(q, k_cache.scalar_type(), "q (same dtype as k_cache)");
  const int64_t T = q.size(0), Hq = q.size(1), Hkv = k_cache.size(2), D = k_cache.size(3);
  c.size(q, 2, D, "q", "D");
  c.inner(q, "q");
  c.rank(out, 3, "out");
  c.dtype(out, q.scalar_type(), "out (same dtype as q)");
  c.size(out, 0, T, "out", "T");
  c.size(out, 1, Hq, "out", "Hq");
  c.size(out, 2, D, "out", "D");
  c.inner(out, "out");
  STD_TORCH_CHECK(Hq >= 1 && Hq % Hkv == 0, c.op, "Hq = ", Hq, " must be a positive multiple of Hkv = ", Hkv);
  STD_TORCH_CHECK(Hq / Hkv <= 64, c.op, "G = Hq/Hkv = ", Hq / Hkv, " exceeds the supported maximum 64");
  c.dtype(lse, ScalarType::Float, "lse");
  if (lse.numel() != 0) {
    c.rank(lse, 2, "lse");
    c.size(lse, 0, T, "lse", "T");
    c.size(lse, 1, Hq, "lse", "Hq");
    STD_TORCH_CHECK(lse.stride(1) == 1 && lse.stride(0) == Hq, c.op, "lse must be contiguous");
  }
  c.rank(block_table, 2, "block_table");
  c.dtype(block_table, ScalarType::Int, "block_table");
  c.inner(block_table, "block_table");
  c.vector(seq_lens, ScalarType::Int, "seq_lens");
  const int64_t R = seq_lens.size(0);
  STD_TORCH_CHECK(block_table.size(0) >= R, c.op, "block_table has ", block_table.size(0), " rows, fewer than num_reqs = ", R);
  STD_TORCH_CHECK(std::isfinite(softmax_scale) && softmax_scale > 0.0, c.op, "softmax_scale must be finite and > 0, got ", softmax_scale);
  c.vector(workspace, ScalarType::Byte, "workspace");
  c.count(T, "T");
  c.count(Hq, "Hq");
  c.count(R, "num_reqs");
  c.count(block_table.size(1), "block_table.size(1)");
  c.device(out, q, "out", "q");
  c.device(lse, q, "lse", "q");
  c.device(k_cache, q, "k_cache", "q");
  c.device(v_cache, q, "v_cache", "q");
  c.device(block_table, q, "block_table", "q");
  c.device(seq_lens, q, "seq_lens", "q");
  c.device(workspace, q, "workspace", "q");
  PthB200Kv16Args a = new_args<PthB200Kv16Args>();
  a.q = q.data_ptr();
  a.q_stride_token = bytes(q, 0);
  a.q_stride_head = bytes(q, 1);
  a.out = out.data_ptr();
  a.out_stride_token = bytes(out, 0);
  a.out_stride_head = bytes(out, 1);
  a.lse = lse.numel() != 0 ? static_cast<float*>(lse.data_ptr()) : nullptr;
  a.k_cache = as_stream(k_cache);
  a.v_cache = as_stream(v_cache);
  a.block_table = static_cast<const int32_t*>(block_table.data_ptr());
  a.block_table_row_stride = block_table.stride(0);
  a.seq_lens = static_cast<const int32_t*>(seq_lens.data_ptr());
  a.workspace = workspace.data_ptr();
  a.workspace_bytes = workspace.numel();
  a.dtype = type_code(q.scalar_type());
  a.num_blocks = static_cast<int32_t>(k_cache.size(0));
  a.block_size = static_cast<int32_t>(k_cache.size(1));
  a.num_kv_heads = static_cast<int32_t>(Hkv);
  a.num_q_heads = static_cast<int32_t>(Hq);
  a.head_size = static_cast<int32_t>(D);
  a.num_reqs = static_cast<int32_t>(R);
  a.num_tokens = static_cast<int32_t>(T);
  a.num_pages = static_cast<int32_t>(block_table.size(1));
  a.softmax_scale = static_cast<float>(softmax_scale);
  return a;
}

void kv16_decode_attention(Tensor& out, Tensor& lse, const Tensor& q, const Tensor& k_cache, const Tensor& v_cache,
                           const Tensor& block_table, const Tensor& seq_lens, double softmax_scale, Tensor& workspace, int64_t window) {
  const Check c{"kv16_decode_attention: "};
  PthB200Kv16Args a = attention_args(c, out, lse, q, k_cache, v_cache, block_table, seq_lens, softmax_scale, workspace);
  c.size(q, 0, seq_lens.size(0), "q", "num_reqs");
  STD_TORCH_CHECK(window >= 0, c.op, "window must be >= 0, got ", window);
  a.window = window > INT32_MAX ? INT32_MAX : static_cast<int32_t>(window);
  a.max_query_len = 1;
  int32_t device = 0;
  void* stream = c.stream(q, &device);
  const torch::stable::accelerator::DeviceGuard guard(device);
  c.done(pthb200_kv16_decode(&a, stream));
}

void kv16_cross_attention(Tensor& out, Tensor& lse, const Tensor& q, const Tensor& k_cache, const Tensor& v_cache,
                          const Tensor& block_table, const Tensor& context_lens, const Tensor& query_start_loc, int64_t max_query_len,
                          double softmax_scale, Tensor& workspace) {
  const Check c{"kv16_cross_attention: "};
  PthB200Kv16Args a = attention_args(c, out, lse, q, k_cache, v_cache, block_table, context_lens, softmax_scale, workspace);
  c.vector(query_start_loc, ScalarType::Int, "query_start_loc");
  c.size(query_start_loc, 0, context_lens.size(0) + 1, "query_start_loc", "num_reqs + 1");
  STD_TORCH_CHECK(max_query_len >= 0 && max_query_len <= q.size(0), c.op, "max_query_len must be in [0, T = ", q.size(0), "], got ",
                  max_query_len);
  c.device(query_start_loc, q, "query_start_loc", "q");
  a.query_start_loc = static_cast<const int32_t*>(query_start_loc.data_ptr());
  a.max_query_len = static_cast<int32_t>(max_query_len);
  int32_t device = 0;
  void* stream = c.stream(q, &device);
  const torch::stable::accelerator::DeviceGuard guard(device);
  c.done(pthb200_kv16_cross(&a, stream));
}

}  // namespace

STABLE_TORCH_LIBRARY_FRAGMENT(pth_flash_attn, m) {
  m.def(
      "page_tables(Tensor context_lens, Tensor query_lens, Tensor free_blocks, Tensor! block_table, Tensor! seq_lens, "
      "Tensor! query_start_loc, Tensor! slot_mapping, Tensor! positions, Tensor! pages_taken, int block_size) -> ()");
  m.def("kv16_write(Tensor key, Tensor value, Tensor! k_cache, Tensor! v_cache, Tensor slot_mapping) -> ()");
  m.def(
      "kv16_decode_attention(Tensor! out, Tensor! lse, Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, "
      "Tensor seq_lens, float softmax_scale, Tensor! workspace, int window=0) -> ()");
  m.def(
      "kv16_cross_attention(Tensor! out, Tensor! lse, Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, "
      "Tensor context_lens, Tensor query_start_loc, int max_query_len, float softmax_scale, Tensor! workspace) -> ()");
}

STABLE_TORCH_LIBRARY_IMPL(pth_flash_attn, CUDA, m) {
  m.impl("page_tables", TORCH_BOX(&page_tables));
  m.impl("kv16_write", TORCH_BOX(&kv16_write));
  m.impl("kv16_decode_attention", TORCH_BOX(&kv16_decode_attention));
  m.impl("kv16_cross_attention", TORCH_BOX(&kv16_cross_attention));
}
STABLE_TORCH_LIBRARY_IMPL(pth_flash_attn, CPU, m) {
  m.impl("page_tables", TORCH_BOX(&page_tables));
  m.impl("kv16_write", TORCH_BOX(&kv16_write));
  m.impl("kv16_decode_attention", TORCH_BOX(&kv16_decode_attention));
  m.impl("kv16_cross_attention", TORCH_BOX(&kv16_cross_attention));
}
