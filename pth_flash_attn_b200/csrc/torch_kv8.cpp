// The torch ops of the 8-bit paged cache and of rotary positions (pth_flash_attn::rotary, kv8_write, kv8_read,
// kv8_decode_attention, kv8_attention): argument checks, then the C ABI of libpthb200_attn.so.  Registered for the CUDA and
// CPU keys through the libtorch stable ABI; on the CPU key a call raises behind its checks.
// Nothing here allocates, reads device data on the host or synchronises.
#include "torch_check.h"

namespace {

bool is_float(ScalarType t) { return t == ScalarType::Float || t == ScalarType::BFloat16 || t == ScalarType::Half; }
bool is_16bit(ScalarType t) { return t == ScalarType::BFloat16 || t == ScalarType::Half; }
int32_t clamp32(int64_t n) { return n > INT32_MAX ? INT32_MAX : static_cast<int32_t>(n); }

// k_cache / v_cache [NB, BS, Hkv, D] of e4m3 numbers, k_scale / v_scale [NB, BS / tokens of a scale, Hkv].  Returns the latter.
int32_t check_caches(const Check& c, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale) {
  c.rank(k_cache, 4, "k_cache");
  c.rank(v_cache, 4, "v_cache");
  c.rank(k_scale, 3, "k_scale");
  c.rank(v_scale, 3, "v_scale");
  c.dtype(k_cache, ScalarType::Float8_e4m3fn, "k_cache");
  c.dtype(v_cache, ScalarType::Float8_e4m3fn, "v_cache");
  c.dtype(k_scale, ScalarType::Float, "k_scale");
  c.dtype(v_scale, ScalarType::Float, "v_scale");
  const int64_t NB = k_cache.size(0), BS = k_cache.size(1), Hkv = k_cache.size(2), D = k_cache.size(3), groups = k_scale.size(1);
  STD_TORCH_CHECK(D == 64 || D == 128 || D == 256, c.op, "head size D = k_cache.size(3) must be 64, 128 or 256, got ", D);
  STD_TORCH_CHECK(NB >= 1 && BS >= 1 && Hkv >= 1, c.op, "k_cache must not be empty");
  c.size(v_cache, 0, NB, "v_cache", "NB");
  c.size(v_cache, 1, BS, "v_cache", "BS");
  c.size(v_cache, 2, Hkv, "v_cache", "Hkv");
  c.size(v_cache, 3, D, "v_cache", "D");
  c.size(k_scale, 0, NB, "k_scale", "NB");
  STD_TORCH_CHECK(groups >= 1 && BS % groups == 0 && BS / groups % 16 == 0, c.op,
                  "BS / k_scale.size(1), the tokens of a scale, must be a multiple of 16, got ", BS, " / ", groups);
  c.size(k_scale, 2, Hkv, "k_scale", "Hkv");
  c.size(v_scale, 0, NB, "v_scale", "NB");
  c.size(v_scale, 1, groups, "v_scale", "k_scale.size(1)");
  c.size(v_scale, 2, Hkv, "v_scale", "Hkv");
  c.inner(k_cache, "k_cache");
  c.inner(v_cache, "v_cache");
  c.count(NB, "NB");
  c.count(BS, "BS");
  c.count(Hkv, "Hkv");
  return static_cast<int32_t>(BS / groups);
}
void check_table(const Check& c, const Tensor& block_table, const Tensor& lens, const char* name) {
  c.rank(block_table, 2, "block_table");
  c.dtype(block_table, ScalarType::Int, "block_table");
  c.inner(block_table, "block_table");
  c.vector(lens, ScalarType::Int, name);
  STD_TORCH_CHECK(block_table.size(0) >= lens.size(0), c.op, "block_table has ", block_table.size(0), " rows, fewer than num_reqs = ", lens.size(0));
  c.count(lens.size(0), "num_reqs");
  c.count(block_table.size(1), "block_table.size(1)");
}
// key / value [T, Hkv, D] of one floating type.
void check_rows(const Check& c, const Tensor& key, const Tensor& value, const Tensor& k_cache) {
  c.rank(key, 3, "key");
  c.rank(value, 3, "value");
  STD_TORCH_CHECK(is_float(key.scalar_type()), c.op, "key must be float32, bfloat16 or float16, got ", type_name(key.scalar_type()));
  c.dtype(value, key.scalar_type(), "value (same dtype as key)");
  c.size(key, 1, k_cache.size(2), "key", "Hkv");
  c.size(key, 2, k_cache.size(3), "key", "D");
  c.size(value, 0, key.size(0), "value", "T");
  c.size(value, 1, k_cache.size(2), "value", "Hkv");
  c.size(value, 2, k_cache.size(3), "value", "D");
  c.inner(key, "key");
  c.inner(value, "value");
  c.count(key.size(0), "T");
}
void check_starts(const Check& c, const Tensor& starts, int64_t R, int64_t longest, int64_t T, const char* name, const char* bound) {
  c.vector(starts, ScalarType::Int, name);
  c.size(starts, 0, R + 1, name, "num_reqs + 1");
  STD_TORCH_CHECK(longest >= 0 && longest <= T, c.op, bound, " must be in [0, T = ", T, "], got ", longest);
}
void check_devices(const Check& c, std::initializer_list<std::pair<const Tensor*, const char*>> others, const Tensor& as, const char* of) {
  for (const auto& [t, name] : others) c.device(*t, as, name, of);
}
template <class Args>
void fill_cache(Args& a, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale, int32_t scale_tokens,
                const Tensor& block_table) {
  a.k_cache = as_stream(k_cache);
  a.v_cache = as_stream(v_cache);
  a.k_scale = as_stream(k_scale);
  a.v_scale = as_stream(v_scale);
  a.block_table = static_cast<const int32_t*>(block_table.data_ptr());
  a.block_table_row_stride = block_table.stride(0);
  a.num_blocks = static_cast<int32_t>(k_cache.size(0));
  a.block_size = static_cast<int32_t>(k_cache.size(1));
  a.scale_tokens = scale_tokens;
  a.num_kv_heads = static_cast<int32_t>(k_cache.size(2));
  a.head_size = static_cast<int32_t>(k_cache.size(3));
  a.num_pages = static_cast<int32_t>(block_table.size(1));
}
template <class Args>
void fill_rows(Args& a, const Tensor& key, const Tensor& value) {
  a.key = key.data_ptr();
  a.value = value.data_ptr();
  a.key_stride_token = bytes(key, 0);
  a.key_stride_head = bytes(key, 1);
  a.value_stride_token = bytes(value, 0);
  a.value_stride_head = bytes(value, 1);
}

void kv8_write(const Tensor& key, const Tensor& value, Tensor& k_cache, Tensor& v_cache, Tensor& k_scale, Tensor& v_scale, const Tensor& block_table,
               const Tensor& seq_lens, const Tensor& query_start_loc, int64_t max_query_len) {
  const Check c{"kv8_write: "};
  const int32_t scale_tokens = check_caches(c, k_cache, v_cache, k_scale, v_scale);
  check_rows(c, key, value, k_cache);
  check_table(c, block_table, seq_lens, "seq_lens");
  check_starts(c, query_start_loc, seq_lens.size(0), max_query_len, key.size(0), "query_start_loc", "max_query_len");
  c.written(k_cache, "k_cache");
  c.written(v_cache, "v_cache");
  c.written(k_scale, "k_scale");
  c.written(v_scale, "v_scale");
  check_devices(c, {{&value, "value"}, {&k_cache, "k_cache"}, {&v_cache, "v_cache"}, {&k_scale, "k_scale"}, {&v_scale, "v_scale"},
                    {&block_table, "block_table"}, {&seq_lens, "seq_lens"}, {&query_start_loc, "query_start_loc"}}, key, "key");
  int32_t device = 0;
  void* stream = c.stream(key, &device);
  PthB200Kv8WriteArgs a = new_args<PthB200Kv8WriteArgs>();
  fill_rows(a, key, value);
  fill_cache(a, k_cache, v_cache, k_scale, v_scale, scale_tokens, block_table);
  a.seq_lens = static_cast<const int32_t*>(seq_lens.data_ptr());
  a.query_start_loc = static_cast<const int32_t*>(query_start_loc.data_ptr());
  a.src_dtype = type_code(key.scalar_type());
  a.num_reqs = static_cast<int32_t>(seq_lens.size(0));
  a.num_tokens = static_cast<int32_t>(key.size(0));
  a.max_query_len = static_cast<int32_t>(max_query_len);
  const torch::stable::accelerator::DeviceGuard guard(device);
  c.done(pthb200_kv8_write(&a, stream));
}

void kv8_read(Tensor& key, Tensor& value, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
              const Tensor& block_table, const Tensor& first, const Tensor& row_start_loc, int64_t max_rows) {
  const Check c{"kv8_read: "};
  const int32_t scale_tokens = check_caches(c, k_cache, v_cache, k_scale, v_scale);
  check_rows(c, key, value, k_cache);
  check_table(c, block_table, first, "first");
  check_starts(c, row_start_loc, first.size(0), max_rows, key.size(0), "row_start_loc", "max_rows");
  c.written(key, "key");
  c.written(value, "value");
  check_devices(c, {{&value, "value"}, {&k_cache, "k_cache"}, {&v_cache, "v_cache"}, {&k_scale, "k_scale"}, {&v_scale, "v_scale"},
                    {&block_table, "block_table"}, {&first, "first"}, {&row_start_loc, "row_start_loc"}}, key, "key");
  int32_t device = 0;
  void* stream = c.stream(key, &device);
  PthB200Kv8ReadArgs a = new_args<PthB200Kv8ReadArgs>();
  fill_rows(a, key, value);
  fill_cache(a, k_cache, v_cache, k_scale, v_scale, scale_tokens, block_table);
  a.first = static_cast<const int32_t*>(first.data_ptr());
  a.row_start_loc = static_cast<const int32_t*>(row_start_loc.data_ptr());
  a.dst_dtype = type_code(key.scalar_type());
  a.num_reqs = static_cast<int32_t>(first.size(0));
  a.num_rows = static_cast<int32_t>(key.size(0));
  a.max_rows = static_cast<int32_t>(max_rows);
  const torch::stable::accelerator::DeviceGuard guard(device);
  c.done(pthb200_kv8_read(&a, stream));
}

// What both attention calls ask of their tensors, and the arguments that they share.
PthB200Kv8Args attention_args(const Check& c, Tensor& out, Tensor& lse, const Tensor& q, const Tensor& k_cache, const Tensor& v_cache,
                              const Tensor& k_scale, const Tensor& v_scale, const Tensor& block_table, const Tensor& seq_lens,
                              double softmax_scale, Tensor& workspace, int64_t window) {
  c.rank(q, 3, "q");
  const int32_t scale_tokens = check_caches(c, k_cache, v_cache, k_scale, v_scale);
  STD_TORCH_CHECK(is_16bit(q.scalar_type()), c.op, "q must be bfloat16 or float16, got ", type_name(q.scalar_type()));
  const int64_t T = q.size(0), Hq = q.size(1), Hkv = k_cache.size(2), D = k_cache.size(3);
  c.size(q, 2, D, "q", "D");
  c.inner(q, "q");
  c.rank(out, 3, "out");
  c.dtype(out, q.scalar_type(), "out (same dtype as q)");
  c.size(out, 0, T, "out", "T");
  c.size(out, 1, Hq, "out", "Hq");
  c.size(out, 2, D, "out", "D");
  c.inner(out, "out");
  c.written(out, "out");
  STD_TORCH_CHECK(Hq >= 1 && Hq % Hkv == 0, c.op, "Hq = ", Hq, " must be a positive multiple of Hkv = ", Hkv);
  STD_TORCH_CHECK(Hq / Hkv <= 64, c.op, "G = Hq/Hkv = ", Hq / Hkv, " exceeds the supported maximum 64");
  c.dtype(lse, ScalarType::Float, "lse");
  if (lse.numel() != 0) {
    c.rank(lse, 2, "lse");
    c.size(lse, 0, T, "lse", "T");
    c.size(lse, 1, Hq, "lse", "Hq");
    STD_TORCH_CHECK(lse.stride(1) == 1 && lse.stride(0) == Hq, c.op, "lse must be contiguous");
  }
  check_table(c, block_table, seq_lens, "seq_lens");
  STD_TORCH_CHECK(std::isfinite(softmax_scale) && softmax_scale > 0.0, c.op, "softmax_scale must be finite and > 0, got ", softmax_scale);
  STD_TORCH_CHECK(window >= 0, c.op, "window must be >= 0, got ", window);
  c.vector(workspace, ScalarType::Byte, "workspace");
  c.count(T, "T");
  c.count(Hq, "Hq");
  check_devices(c, {{&out, "out"}, {&lse, "lse"}, {&k_cache, "k_cache"}, {&v_cache, "v_cache"}, {&k_scale, "k_scale"}, {&v_scale, "v_scale"},
                    {&block_table, "block_table"}, {&seq_lens, "seq_lens"}, {&workspace, "workspace"}}, q, "q");
  PthB200Kv8Args a = new_args<PthB200Kv8Args>();
  a.q = q.data_ptr();
  a.q_stride_token = bytes(q, 0);
  a.q_stride_head = bytes(q, 1);
  a.out = out.data_ptr();
  a.out_stride_token = bytes(out, 0);
  a.out_stride_head = bytes(out, 1);
  a.lse = lse.numel() != 0 ? static_cast<float*>(lse.data_ptr()) : nullptr;
  fill_cache(a, k_cache, v_cache, k_scale, v_scale, scale_tokens, block_table);
  a.seq_lens = static_cast<const int32_t*>(seq_lens.data_ptr());
  a.workspace = workspace.data_ptr();
  a.workspace_bytes = workspace.numel();
  a.dtype = type_code(q.scalar_type());
  a.num_q_heads = static_cast<int32_t>(Hq);
  a.num_reqs = static_cast<int32_t>(seq_lens.size(0));
  a.num_tokens = static_cast<int32_t>(T);
  a.window = clamp32(window);
  a.causal = 1;
  a.softmax_scale = static_cast<float>(softmax_scale);
  return a;
}

void kv8_decode_attention(Tensor& out, Tensor& lse, const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale,
                          const Tensor& v_scale, const Tensor& block_table, const Tensor& seq_lens, double softmax_scale, Tensor& workspace,
                          int64_t window) {
  const Check c{"kv8_decode_attention: "};
  PthB200Kv8Args a = attention_args(c, out, lse, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, softmax_scale, workspace, window);
  c.size(q, 0, seq_lens.size(0), "q", "num_reqs");
  a.max_query_len = 1;
  int32_t device = 0;
  void* stream = c.stream(q, &device);
  const torch::stable::accelerator::DeviceGuard guard(device);
  c.done(pthb200_kv8_decode(&a, stream));
}

void kv8_attention(Tensor& out, Tensor& lse, const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale,
                   const Tensor& v_scale, const Tensor& block_table, const Tensor& seq_lens, const Tensor& query_start_loc, int64_t max_query_len,
                   double softmax_scale, Tensor& workspace, int64_t window, bool causal) {
  const Check c{"kv8_attention: "};
  PthB200Kv8Args a = attention_args(c, out, lse, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, softmax_scale, workspace, window);
  check_starts(c, query_start_loc, seq_lens.size(0), max_query_len, q.size(0), "query_start_loc", "max_query_len");
  c.device(query_start_loc, q, "query_start_loc", "q");
  a.query_start_loc = static_cast<const int32_t*>(query_start_loc.data_ptr());
  a.max_query_len = static_cast<int32_t>(max_query_len);
  a.causal = causal ? 1 : 0;
  int32_t device = 0;
  void* stream = c.stream(q, &device);
  const torch::stable::accelerator::DeviceGuard guard(device);
  c.done(pthb200_kv8_attend(&a, stream));
}

void rotary(Tensor& q_out, Tensor& k_out, const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& frequencies, double scale,
            bool interleaved, bool inverse) {
  const Check c{"rotary: "};
  c.rank(q, 3, "q");
  c.rank(k, 3, "k");
  STD_TORCH_CHECK(is_float(q.scalar_type()), c.op, "q must be float32, bfloat16 or float16, got ", type_name(q.scalar_type()));
  c.dtype(k, q.scalar_type(), "k (same dtype as q)");
  const int64_t T = q.size(0), D = q.size(2), half = frequencies.numel();
  STD_TORCH_CHECK(D >= 1 && D <= 1024, c.op, "head size D = q.size(2) must be in [1, 1024], got ", D);
  c.size(k, 0, T, "k", "T");
  c.size(k, 2, D, "k", "D");
  const Tensor* in[] = {&q, &k};
  const Tensor* out[] = {&q_out, &k_out};
  const char* in_names[] = {"q", "k"};
  const char* names[] = {"q_out", "k_out"};
  for (int i = 0; i < 2; ++i) {
    c.inner(*in[i], in_names[i]);
    c.rank(*out[i], 3, names[i]);
    c.dtype(*out[i], q.scalar_type(), i == 0 ? "q_out (same dtype as q)" : "k_out (same dtype as q)");
    c.size(*out[i], 0, T, names[i], "T");
    c.size(*out[i], 1, in[i]->size(1), names[i], i == 0 ? "q.size(1)" : "k.size(1)");
    c.size(*out[i], 2, D, names[i], "D");
    c.inner(*out[i], names[i]);
    c.written(*out[i], names[i]);
    if (in[i]->numel() != 0 && in[i]->data_ptr() == out[i]->data_ptr())
      STD_TORCH_CHECK(in[i]->stride(0) == out[i]->stride(0) && in[i]->stride(1) == out[i]->stride(1), c.op, names[i], " in the place of ", in_names[i],
                      " must have its strides");
  }
  c.vector(positions, ScalarType::Long, "positions");
  c.size(positions, 0, T, "positions", "T");
  c.rank(frequencies, 1, "frequencies");
  STD_TORCH_CHECK(frequencies.scalar_type() == ScalarType::Double || frequencies.scalar_type() == ScalarType::Float, c.op,
                  "frequencies must be float64 or float32, got ", type_name(frequencies.scalar_type()));
  c.inner(frequencies, "frequencies");
  STD_TORCH_CHECK(half >= 1 && 2 * half <= D, c.op, "frequencies.size(0) must be in [1, D / 2 = ", D / 2, "], got ", half);
  STD_TORCH_CHECK(std::isfinite(scale) && std::isfinite(static_cast<float>(scale)), c.op, "scale must be finite, got ", scale);
  c.count(T, "T");
  c.count(q.size(1), "q.size(1)");
  c.count(k.size(1), "k.size(1)");
  check_devices(c, {{&k, "k"}, {&q_out, "q_out"}, {&k_out, "k_out"}, {&positions, "positions"}, {&frequencies, "frequencies"}}, q, "q");
  int32_t device = 0;
  void* stream = c.stream(q, &device);
  PthB200RotaryArgs a = new_args<PthB200RotaryArgs>();
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.q_out = q_out.data_ptr();
  a.k_out = k_out.data_ptr();
  a.q_stride_token = bytes(q, 0);
  a.q_stride_head = bytes(q, 1);
  a.k_stride_token = bytes(k, 0);
  a.k_stride_head = bytes(k, 1);
  a.q_out_stride_token = bytes(q_out, 0);
  a.q_out_stride_head = bytes(q_out, 1);
  a.k_out_stride_token = bytes(k_out, 0);
  a.k_out_stride_head = bytes(k_out, 1);
  a.positions = static_cast<const int64_t*>(positions.data_ptr());
  a.frequencies = frequencies.data_ptr();
  a.frequencies_64 = frequencies.scalar_type() == ScalarType::Double;
  a.dtype = type_code(q.scalar_type());
  a.num_tokens = static_cast<int32_t>(T);
  a.num_q_heads = static_cast<int32_t>(q.size(1));
  a.num_k_heads = static_cast<int32_t>(k.size(1));
  a.head_size = static_cast<int32_t>(D);
  a.num_frequencies = static_cast<int32_t>(half);
  a.interleaved = interleaved;
  a.inverse = inverse;
  a.scale = static_cast<float>(scale);
  const torch::stable::accelerator::DeviceGuard guard(device);
  c.done(pthb200_rotary(&a, stream));
}

}  // namespace

STABLE_TORCH_LIBRARY_FRAGMENT(pth_flash_attn, m) {
  m.def(
      "rotary(Tensor! q_out, Tensor! k_out, Tensor q, Tensor k, Tensor positions, Tensor frequencies, float scale=1.0, "
      "bool interleaved=False, bool inverse=False) -> ()");
  m.def(
      "kv8_write(Tensor key, Tensor value, Tensor! k_cache, Tensor! v_cache, Tensor! k_scale, Tensor! v_scale, Tensor block_table, "
      "Tensor seq_lens, Tensor query_start_loc, int max_query_len) -> ()");
  m.def(
      "kv8_read(Tensor! key, Tensor! value, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor block_table, "
      "Tensor first, Tensor row_start_loc, int max_rows) -> ()");
  m.def(
      "kv8_decode_attention(Tensor! out, Tensor! lse, Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, "
      "Tensor block_table, Tensor seq_lens, float softmax_scale, Tensor! workspace, int window=0) -> ()");
  m.def(
      "kv8_attention(Tensor! out, Tensor! lse, Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, "
      "Tensor block_table, Tensor seq_lens, Tensor query_start_loc, int max_query_len, float softmax_scale, Tensor! workspace, "
      "int window=0, bool causal=True) -> ()");
}

STABLE_TORCH_LIBRARY_IMPL(pth_flash_attn, CUDA, m) {
  m.impl("rotary", TORCH_BOX(&rotary));
  m.impl("kv8_write", TORCH_BOX(&kv8_write));
  m.impl("kv8_read", TORCH_BOX(&kv8_read));
  m.impl("kv8_decode_attention", TORCH_BOX(&kv8_decode_attention));
  m.impl("kv8_attention", TORCH_BOX(&kv8_attention));
}
STABLE_TORCH_LIBRARY_IMPL(pth_flash_attn, CPU, m) {
  m.impl("rotary", TORCH_BOX(&rotary));
  m.impl("kv8_write", TORCH_BOX(&kv8_write));
  m.impl("kv8_read", TORCH_BOX(&kv8_read));
  m.impl("kv8_decode_attention", TORCH_BOX(&kv8_decode_attention));
  m.impl("kv8_attention", TORCH_BOX(&kv8_attention));
}
