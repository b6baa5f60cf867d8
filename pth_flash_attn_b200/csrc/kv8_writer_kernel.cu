// Writer of the 8-bit paged cache: new tokens' K and V rows as e4m3 numbers, with a power of two as the scale of a block of tokens.
//
// A unit of work is a block of tokens of a request that the call writes to, a KV head, K or V.  Its new rows' largest finite value
// gives the scale that they need; a block that goes on keeps its own unless it is too small, and then the cells in front of the
// new ones are rounded again.  A power of two costs e4m3 nothing (its relative error is the same at any size) and makes both the
// quotients and the re-rounding exact up to the one rounding.
//
// Blocks up to 32 tokens are a warp's work: its rows of 16 bytes a lane stay in registers between the maximum and the rounding.
// Larger ones are a CTA's, which reads the rows again (from L2) for the rounding; but where a request has one token at most, a warp's too, whose CTA rounds
// more than 32 older rows again for it (with a CTA for each, 64 requests that have nothing to round again took 10.8 us instead of 3.7; with the
// warp alone, 815 older rows of 128 dims 94 us instead of 20, of 256 dims 166 instead of 35).  Bytes bound it: T Hkv D (source + 1) x 2.
// 4 x 2,048 bf16 tokens of 8 heads, 128 dims: 11.3 to 13.1 us one call behind another, 7.7 of them bytes at the copy bandwidth; the others are the
// launch and a unit's dependent look-ups (offsets, block table, scale).  64 tokens: 3.2 us on the device, less than the host takes.
//
// Units find their block without a list: request r's blocks are numbered from start_r / g + 2 r on, which leaves room for the two
// more blocks than q / g that its tokens may touch (r itself where a request has one token at most).  Numbers that no block has
// end at once.
#include "kv8.cuh"

#include "pdl.cuh"

namespace pthb200 {
namespace {

constexpr int kWarps = 8;
constexpr int kMostOlder = 32;   // older rows that a warp rounds again by itself

struct Write8Params {
  const uint8_t* src[2];
  int64_t src_stride_token[2], src_stride_head[2];
  uint8_t* cache[2];
  int64_t stride_block[2], stride_slot[2], stride_head[2];
  float* scale[2];
  int64_t scale_stride_block[2], scale_stride_group[2], scale_stride_head[2];   // in elements
  const int32_t* block_table;
  int64_t block_table_row_stride;
  const int32_t* seq_lens;
  const int32_t* query_start_loc;
  int32_t num_blocks, block_size, scale_tokens, num_kv_heads, num_reqs, num_tokens, num_pages, max_query_len, src_dtype;
};

// Eight elements of a source row, as they are.  kWide: rows lie on 16-byte boundaries.
template <int kDtype>
struct Eight {
  uint32_t w[kDtype == PTH_ATTN_F32 ? 8 : 4];
  template <bool kWide>
  __device__ __forceinline__ void load(const uint8_t* row, int e0) {
    constexpr int kWords = kDtype == PTH_ATTN_F32 ? 8 : 4;
    if constexpr (kWide) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(row) + (e0 * kWords / 8 + i) / 4);
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
    } else if constexpr (kDtype == PTH_ATTN_F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __ldg(reinterpret_cast<const uint32_t*>(row) + e0 + i);
    } else {
      const uint16_t* const h = reinterpret_cast<const uint16_t*>(row) + e0;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (uint32_t)__ldg(h + 2 * i) | (uint32_t)__ldg(h + 2 * i + 1) << 16;
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(w) / 4); ++i) w[i] = 0u;
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (kDtype == PTH_ATTN_F32) return __uint_as_float(w[i]);
    else if constexpr (kDtype == PTH_ATTN_F16) return __half2float(__ushort_as_half((unsigned short)(w[i / 2] >> 16 * (i & 1))));
    else return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
};
// The largest finite magnitude of some rows' pieces.
template <int kDtype, int kCount>
__device__ __forceinline__ float finite_max(const Eight<kDtype> (&x)[kCount]) {
  float m = 0.f;
  if constexpr (kDtype != PTH_ATTN_F32) {   // magnitudes are ordered as 16-bit integers, of which infinities and NaN are the largest
    constexpr uint32_t kInf = kDtype == PTH_ATTN_F16 ? 0x7c00u : 0x7f80u;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      top = __vimax3_u16x2(top, x[i].w[0] & 0x7fff7fffu, x[i].w[1] & 0x7fff7fffu);
      top = __vimax3_u16x2(top, x[i].w[2] & 0x7fff7fffu, x[i].w[3] & 0x7fff7fffu);
    }
    const uint32_t one = max(top & 0xffffu, top >> 16);
    if (one < kInf) return kDtype == PTH_ATTN_F16 ? __half2float(__ushort_as_half((unsigned short)one)) : __uint_as_float(one << 16);
  }
#pragma unroll
  for (int i = 0; i < kCount; ++i) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float a = fabsf(x[i].get(k));
      m = a < INFINITY ? fmaxf(m, a) : m;
    }
  }
  return m;
}
// The smallest power of two, 2^-126 to 2^120, with most <= 448 times it.
__device__ __forceinline__ float needed_scale(float most) { return power_of_two(min(120, max(-126, e4m3_exponent(most)))); }
// Eight numbers as cells, x / scale: exactly scaled where the scale is a power of two (up: its reciprocal; 0: it is none).
template <int kDtype>
__device__ __forceinline__ uint2 cells8(const Eight<kDtype>& x, float scale, float up) {
  float y[8];
  if (up != 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x.get(i) * up;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __fdiv_rn(x.get(i), scale);
  }
  return make_uint2(e4m3x2(y[0], y[1]) | e4m3x2(y[2], y[3]) << 16, e4m3x2(y[4], y[5]) | e4m3x2(y[6], y[7]) << 16);
}
__device__ __forceinline__ uint32_t rescaled(uint32_t w, float ratio) {
  const float2 a = float2_of_e4m3x2(w & 0xffffu), b = float2_of_e4m3x2(w >> 16);
  return e4m3x2(a.x * ratio, a.y * ratio) | e4m3x2(b.x * ratio, b.y * ratio) << 16;
}

// A block of tokens that the call writes to.
struct Block {
  int row0, rows;      // first new row of the source, their number
  int begin;           // first new position in the block of tokens
  int block, group;    // of the cache; the block may be none of it
};

// Block number x of the launch, found by a warp (the same in all lanes); false: there is none.
__device__ __forceinline__ bool find_block(const Write8Params& p, int x, Block* out) {
  const int g = p.scale_tokens, lane = threadIdx.x & 31;
  const bool single = p.max_query_len == 1;
  auto start_of = [&](int r) -> int { return min(max(0, __ldg(p.query_start_loc + r)), p.num_tokens); };
  auto number_of = [&](int r, int start) -> long long { return single ? r : (long long)(start / g) + 2ll * r; };
  // the last request whose numbers begin at or in front of x: among 32, whose offsets and lengths a lane each loads
  int lo = single ? x : 0, hi = single ? x + 1 : p.num_reqs;
  if (lo >= p.num_reqs) return false;
#pragma unroll 1
  while (hi - lo > 32) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    const uint32_t before = __ballot_sync(0xffffffffu, at < hi && number_of(at, start_of(at)) <= x);
    if (before == 0) return false;   // (start offsets that go backwards)
    const int last = 31 - __clz(before);
    hi = min(hi, lo + (last + 1) * step);
    lo += last * step;
  }
  const int mine = min(lo + lane, hi - 1), begin = start_of(mine), stop = start_of(mine + 1), length = max(0, __ldg(p.seq_lens + mine));
  const uint32_t before = __ballot_sync(0xffffffffu, lo + lane < hi && number_of(mine, begin) <= x);
  if (before == 0) return false;
  const int from_lane = 31 - __clz(before), r = lo + from_lane;
  const int first = __shfl_sync(0xffffffffu, begin, from_lane), end = __shfl_sync(0xffffffffu, stop, from_lane), seq = __shfl_sync(0xffffffffu, length, from_lane);
  const int all = max(0, end - first), tokens = min(all, p.max_query_len), pos0 = seq - all;
  const int skip = max(0, -pos0);   // tokens at negative positions
  if (tokens <= skip) return false;
  const long long nth = x - number_of(r, first);
  const long long start = ((long long)(pos0 + skip) / g + nth) * g;
  const long long from = max(start, (long long)pos0 + skip), to = min(start + g, (long long)pos0 + tokens);
  if (nth < 0 || to <= from) return false;
  const long long page = from / p.block_size;
  if (page >= p.num_pages) return false;
  out->block = __ldg(p.block_table + (int64_t)r * p.block_table_row_stride + page);   // (not looked at here: the rows' loads go out beside it)
  out->group = (int)(start - page * p.block_size) / g;
  out->begin = (int)(from - start);
  out->rows = (int)(to - from);
  out->row0 = first + (int)(from - pos0);
  return true;
}

// Rounds `rows` older rows again, of which these threads take every step-th from `first` on, kOlder of them in flight.
template <int kOlder>
__device__ __forceinline__ void round_again(uint8_t* cells, int64_t stride, int rows, int first, int step, float ratio) {
#pragma unroll 1
  for (int n0 = first; n0 < rows; n0 += kOlder * step) {
    uint2 w[kOlder];
#pragma unroll
    for (int i = 0; i < kOlder; ++i)
      if (n0 + i * step < rows) w[i] = *reinterpret_cast<const uint2*>(cells + (int64_t)(n0 + i * step) * stride);
#pragma unroll
    for (int i = 0; i < kOlder; ++i)
      if (n0 + i * step < rows) *reinterpret_cast<uint2*>(cells + (int64_t)(n0 + i * step) * stride) = make_uint2(rescaled(w[i].x, ratio), rescaled(w[i].y, ratio));
  }
}
// Older rows that are left to the whole CTA.
struct Older {
  uint8_t* cells;
  int64_t stride;
  int rows;
  float ratio;
};

// A unit of work, by a warp or a CTA.  A warp leaves more than kMostOlder older rows to its CTA.
// kKept: pieces of eight elements that a lane keeps, as many as 16 rows of a warp.
template <int HD, int kDtype, bool kWide, bool kCta>
__device__ __forceinline__ void write_unit(const Write8Params& p, float* most_of, Older* older) {
  constexpr int kLanes = HD / 8, kAtOnce = 32 / kLanes;      // lanes of a row, rows of a warp at a time
  constexpr int kKept = kDtype == PTH_ATTN_F32 || HD == 256 ? 8 : 16 / kAtOnce;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunk = lane % kLanes, sub = lane / kLanes;
  // units: (block number, head, K or V), the last fastest
  const int per = 2 * p.num_kv_heads;
  const int64_t unit = kCta ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * kWarps + warp;
  const int x = (int)(unit / per), rest = (int)(unit - (int64_t)x * per), head = rest >> 1, v = rest & 1;
  Block b;
  if (!find_block(p, x, &b)) return;
  const uint8_t* const src = p.src[v] + (int64_t)b.row0 * p.src_stride_token[v] + (int64_t)head * p.src_stride_head[v];
  const int64_t stride = p.src_stride_token[v];
  constexpr int kStep = (kCta ? kWarps : 1) * kAtOnce;       // rows of a round
  const int mine = (kCta ? warp * kAtOnce : 0) + sub;
  float most = 0.f;
  Eight<kDtype> kept[kKept];
#pragma unroll 1
  for (int n0 = 0; n0 < b.rows; n0 += kKept * kStep) {
    const uint8_t* at = src + (n0 + mine) * stride;
#pragma unroll
    for (int i = 0; i < kKept; ++i, at += kStep * stride) {
      kept[i].clear();
      if (n0 + i * kStep + mine < b.rows) kept[i].template load<kWide>(at, chunk * 8);
    }
    most = fmaxf(most, finite_max(kept));
  }
  if ((uint32_t)b.block >= (uint32_t)p.num_blocks) return;   // (the same in all threads that share the block)
  uint8_t* const cells = p.cache[v] + (int64_t)b.block * p.stride_block[v] + (int64_t)(b.group * p.scale_tokens) * p.stride_slot[v] + (int64_t)head * p.stride_head[v] + chunk * 8;
  float* const scale_at = p.scale[v] + (int64_t)b.block * p.scale_stride_block[v] + (int64_t)b.group * p.scale_stride_group[v] + (int64_t)head * p.scale_stride_head[v];
  float was = b.begin > 0 ? *scale_at : 0.f;
  if (!(was > 0.f && was < INFINITY)) was = 0.f;
  most = redux_max(most);
  if constexpr (kCta) {
    if (lane == 0) most_of[warp] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) most = fmaxf(most, most_of[w]);
  }
  const float scale = fmaxf(was, needed_scale(most));
  // the cells in front of the new ones
  if (b.begin > 0 && scale > was) {
    const float ratio = was / scale;
    if (kCta || b.begin <= kMostOlder) round_again<4>(cells, p.stride_slot[v], b.begin, mine, kStep, ratio);
    else if (lane == 0) *older = Older{cells, p.stride_slot[v], b.begin, ratio};
  }
  const float up = (__float_as_uint(scale) & 0x7fffffu) == 0 ? power_of_two(127 - (int)(__float_as_uint(scale) >> 23)) : 0.f;
  const bool once = b.rows <= kKept * kStep;   // (the rows are in registers still)
#pragma unroll 1
  for (int n0 = 0; n0 < b.rows; n0 += kKept * kStep) {
    if (!once) {
#pragma unroll
      for (int i = 0; i < kKept; ++i)
        if (n0 + i * kStep + mine < b.rows) kept[i].template load<kWide>(src + (n0 + i * kStep + mine) * stride, chunk * 8);
    }
    uint8_t* to = cells + (int64_t)(b.begin + n0 + mine) * p.stride_slot[v];
#pragma unroll
    for (int i = 0; i < kKept; ++i, to += kStep * p.stride_slot[v])
      if (n0 + i * kStep + mine < b.rows) *reinterpret_cast<uint2*>(to) = cells8(kept[i], scale, up);
  }
  if constexpr (kCta) __syncthreads();   // (all have read the old scale)
  if (lane == 0 && (!kCta || warp == 0) && scale != was) *scale_at = scale;
}

template <int HD, int kDtype, bool kWide, bool kCta>
__global__ void __launch_bounds__(kWarps * 32, kDtype != PTH_ATTN_F32 && HD < 256 && !kCta ? 4 : 1) kv8_writer_kernel(const __grid_constant__ Write8Params p) {
  __shared__ float most_of[kWarps];
  __shared__ Older older[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) older[warp].rows = 0;
  __syncwarp();
  pdl_wait();
  write_unit<HD, kDtype, kWide, kCta>(p, most_of, &older[warp]);
  if constexpr (!kCta) {
    if (p.scale_tokens <= kMostOlder) return;
    __syncthreads();
    constexpr int kLanes = HD / 8, kAtOnce = 32 / kLanes;
#pragma unroll 1
    for (int w = 0; w < kWarps; ++w)   // (cells: from the first lane's on)
      if (older[w].rows > 0) round_again<8>(older[w].cells + lane % kLanes * 8, older[w].stride, older[w].rows, warp * kAtOnce + lane / kLanes, kWarps * kAtOnce, older[w].ratio);
  }
}

template <int HD, int kDtype>
cudaError_t launch_for(const Write8Params& p, bool wide, cudaStream_t stream) {
  const int64_t numbers = p.max_query_len == 1 ? p.num_reqs : (int64_t)(p.num_tokens / p.scale_tokens) + 2ll * p.num_reqs;
  const int64_t units = numbers * 2 * p.num_kv_heads;
  const bool cta = p.scale_tokens > kMostOlder && p.max_query_len > 1;
  const int64_t ctas = cta ? units : (units + kWarps - 1) / kWarps;
  if (numbers > 0x7fffffff || ctas > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const dim3 grid((unsigned)ctas), block(kWarps * 32);
  if (cta) return pdl_launch(wide ? kv8_writer_kernel<HD, kDtype, true, true> : kv8_writer_kernel<HD, kDtype, false, true>, grid, block, 0, stream, p);
  return pdl_launch(wide ? kv8_writer_kernel<HD, kDtype, true, false> : kv8_writer_kernel<HD, kDtype, false, false>, grid, block, 0, stream, p);
}
template <int HD>
cudaError_t launch_type(const Write8Params& p, bool wide, cudaStream_t stream) {
  if (p.src_dtype == PTH_ATTN_F32) return launch_for<HD, PTH_ATTN_F32>(p, wide, stream);
  if (p.src_dtype == PTH_ATTN_F16) return launch_for<HD, PTH_ATTN_F16>(p, wide, stream);
  return launch_for<HD, PTH_ATTN_BF16>(p, wide, stream);
}

}  // namespace

cudaError_t launch_kv8_writer(const PthB200Kv8WriteArgs& a, cudaStream_t stream) {
  Write8Params p{};
  const PthAttnStream* cache[2] = {&a.k_cache, &a.v_cache};
  const PthAttnStream* scale[2] = {&a.k_scale, &a.v_scale};
  p.src[0] = static_cast<const uint8_t*>(a.key);
  p.src[1] = static_cast<const uint8_t*>(a.value);
  p.src_stride_token[0] = a.key_stride_token;
  p.src_stride_token[1] = a.value_stride_token;
  p.src_stride_head[0] = a.key_stride_head;
  p.src_stride_head[1] = a.value_stride_head;
  bool wide = true;
  for (int i = 0; i < 2; ++i) {
    p.cache[i] = static_cast<uint8_t*>(const_cast<void*>(cache[i]->data));
    p.stride_block[i] = cache[i]->stride_block;
    p.stride_slot[i] = cache[i]->stride_slot;
    p.stride_head[i] = cache[i]->stride_head;
    p.scale[i] = static_cast<float*>(const_cast<void*>(scale[i]->data));
    p.scale_stride_block[i] = scale[i]->stride_block / 4;
    p.scale_stride_group[i] = scale[i]->stride_slot / 4;
    p.scale_stride_head[i] = scale[i]->stride_head / 4;
    wide = wide && reinterpret_cast<uintptr_t>(p.src[i]) % 16 == 0 && p.src_stride_token[i] % 16 == 0 && p.src_stride_head[i] % 16 == 0;
  }
  p.block_table = a.block_table;
  p.block_table_row_stride = a.block_table_row_stride;
  p.seq_lens = a.seq_lens;
  p.query_start_loc = a.query_start_loc;
  p.num_blocks = a.num_blocks;
  p.block_size = a.block_size;
  p.scale_tokens = a.scale_tokens;
  p.num_kv_heads = a.num_kv_heads;
  p.num_reqs = a.num_reqs;
  p.num_tokens = a.num_tokens;
  p.num_pages = a.num_pages;
  p.max_query_len = a.max_query_len;
  p.src_dtype = a.src_dtype;
  switch (a.head_size) {
    case 64:
      return launch_type<64>(p, wide, stream);
    case 128:
      return launch_type<128>(p, wide, stream);
    default:
      return launch_type<256>(p, wide, stream);
  }
}

}  // namespace pthb200
