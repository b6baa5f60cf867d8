// Attention over the 8-bit paged cache for requests of few query rows (a row is a query token and head): one-token decode,
// verification of a few tokens.
//
// Orientation: the 128 keys of a tile sit on the MMA's M dimension, the rows of a KV head on N:
//   S^T[key, row] = sum_d c_K[key, d] Q[row, d]         A = c_K as it lies in the cache (K-major), B = digits of Q
//   O^T[d, row]  += sum_key c_V[key, d] Y[key, row]     A = c_V as it lies in the cache (MN-major), B = digits of Y
// with Y = P scale_V / U.  Both operands A are the cache's own bytes (kind::f8f6f4): no cell passes through a register.
//
// Digits.  An MMA of this kind takes 8-bit numbers on both sides, so a factor of B goes in as a sum of e4m3 numbers, side by
// side on N, each with an accumulator of its own: x = u (d0 + d1 / 16 + d2 / 256), every digit the rounding of what is left.  Digits have
// four bits, and subnormal ones a step of 2^-9, so n digits keep 4 n bits of numbers down to 2^-14 of the largest, and are off by
// 2^-(14 + 4 n) of it below.  bf16 queries take two (they are exact), fp16 queries three.  Y is rounded to fp16, which three digits
// hold: 2^-11 of a weight is an eighth of the rounding of a bf16 output, and a key of 2^-24 of its row's largest weight still
// counts, over 131,072 keys.  At eight rows and 16 or 32 columns they cost the tensor core nothing that shows.
//   u is a power of two per row for Q (its largest into [128, 256)).  U is the power of two above the largest scale_V of a piece's first tile.
// scale_K multiplies a key's scores.
//
// Softmax in one pass: P = 2^(s - ref), l = sum P, and ref (log2 units) is a running bound of a row's s + log2(scale_V / U), over the keys that the row sees: it is
// their maximum less kGainY when it is set, and moves (with l and O rescaled) only when one outgrows it by kSlackY.  So Y is at most 2^8,
// whatever the scales, and a row's weights have their bits whatever the scales of keys that it does not see.
//
// What bounds it: the cache's bytes, 2 D per key and KV head.  The tile's parts (128 keys x 128 dims of K, of V) are units of one
// ring of shared memory, K of the next tile ahead of V of this one (the other way round, the four tokens below took 136 us
// instead of 126 then).  One warp fills it with TMA boxes of 16 or 32 slots; runs of 16 keys that are not wholly visible, and all of them at 64 dims,
// come by 16-byte copies, zero where a key is not visible, so what lies there in memory, NaN included, is never read.
// Scales come with them, one per 16 keys.  The warp that works out the pieces makes the digits of their queries.
//
// Measured (32 heads of 8, 128 dims, bf16, calls behind one another): one token of 64 requests x 8,192 keys, 1.08 GB, 169 to 175 us, 0.94 to 0.97 of the
// copy bandwidth; four tokens of 32 requests of 2,000 to 16,384 keys, 0.65 GB, 127 us with part of the cells in L2, 136 among other work, 0.73: 16 rows'
// softmax, two groups of warps with a barrier for each tile's vote, takes longer than their bytes.  12 heads of 2, 256 dims, 0.53 GB: 90 us, 0.90.  Eight requests of up to 4,095 keys
// 19 us, of which 10 are one tile's way through launch, look-ups, queries, products and rows, and 2 to 5 the merge.
//
// Schedule and merge: kv16_short.cuh.
#include "kv8.cuh"

#include "kv16_short.cuh"
#include "kv8_boxes.cuh"
#include "pdl.cuh"

namespace pthb200 {

__device__ unsigned int g_kv8_short_status = 0;

namespace {

constexpr float kGainY = 6.f, kSlackY = 2.f;
constexpr float kUnset = -1e30f;       // ref of a row that has seen no key: below every score, finite so that a hidden one gives P = 0
constexpr int kRun = 16;               // keys that surely share a scale
constexpr int kScaleTiles = 16;        // tiles whose scales are kept: more than the ring holds units of either kind, and two
constexpr int kDigitsY = 3;

// A unit is 128 rows, of a key each, of up to 128 bytes, in the swizzle of its rows' length (128 or 64 bytes): a row's 16-byte pieces stay
// together.  (In column blocks of 16 dims, a row's pieces 2,064 bytes apart and on banks of their own, 64
// requests x 8,192 keys of 8 heads took 307 us instead of 175: copies of 16 bytes to eight lines of shared memory move half as fast.)
template <int kDims>
__device__ __forceinline__ uint32_t swizzled_chunk(int row, int chunk) {   // where piece `chunk` of a row lies
  return kDims == 128 ? (uint32_t)(chunk ^ (row & 7)) : (uint32_t)(chunk ^ ((row >> 1) & 3));
}
template <int kDims>
__device__ __forceinline__ uint64_t unit_desc(uint32_t saddr, uint32_t lbo) {   // either major: the next 8 rows follow
  return tc::smem_desc(saddr, lbo, 8 * kDims) | (uint64_t)(kDims == 128 ? 2 : 4) << 61;
}

template <int HD, int RP, bool kHalf>
struct Geo8 {
  static constexpr int dims = HD < 128 ? HD : 128;   // of a unit
  static constexpr int parts = HD / dims;            // units of a tile's K, and of its V
  static constexpr int unit = kTile * dims;
  static constexpr int q_digits = kHalf ? 3 : 2;
  // Softmax warpgroups, which share the rows out among themselves; thread t of each is key t of a tile, then dim t of the output.
  static constexpr int groups = RP == 8 ? 1 : 2;
  static constexpr int rows = RP / groups;           // of a group
  // One warp asks for boxes; rows of 64 bytes come faster by 16-byte copies of four (64 x 8,192 keys, 32 heads of 8, us: 123 / 142 by
  // boxes; at 128 dims 176 / 174 with 8 rows, 142 / 126 with 16, at 256 dims 92 / 93 and 104 / 105).
  static constexpr int load_warps = HD == 64 ? 4 : 1;
  static constexpr int load_warp = 4 * groups, mma_warp = load_warp + load_warps, schedule_warp = mma_warp + 1;
  static constexpr int others = (load_warps + 2 + 3) / 4 * 4;    // whole warpgroups beside the softmax, whose last warps have nothing to do
  static constexpr int threads = (load_warp + others) * 32;
  static constexpr int cols = (q_digits * RP + 15) / 16 * 16;     // N of QK
  static constexpr int pcols = (kDigitsY * RP + 15) / 16 * 16;    // N of PV
  static constexpr int qimage = cols * HD;           // column block c of 16 dims at c (cols 16), column n at n 16
  static constexpr int pimage = pcols * kTile;       // block of 16 columns at 2,048 each, key t at t 16
  // Images of Y: two where a tile's PV takes long, so that the next softmax need not wait for it (8 rows, 256 dims, 61 requests of 4,096 to
  // 12,288 keys: 90.3 us instead of 93.5; 128 dims, one token of 64 requests, the same; 16 rows, four of 32 requests, 125.3 us, with one 124.5).
  static constexpr int p_images = HD == 256 && RP == 8 ? 2 : 1;
  static constexpr int fixed = 2 * qimage + p_images * pimage + 9 * RP * 4 + 2 * RP * 4 + kScaleTiles * 64 + 1024;
  static constexpr int units2 = (115712 - fixed - 1024) / unit;
  static constexpr int ctas = units2 >= 3 && RP <= 16 ? 2 : 1;
  static constexpr int most = 2 * (kScaleTiles - 3);   // (see kScaleTiles)
  static constexpr int fit = ctas == 2 ? units2 : (232448 - fixed - 1024) / unit;
  // (Four with 16 rows, whose registers spill: what spills goes round in the first level cache, which shared memory leaves small.  Four and as many
  // as fit, us: four tokens of 32 requests 124.5 / 126.3, 16 heads each of 64 requests 60.8 / 63.0, at 256 dims 103.3 / 109.2, at 64 dims 106.7 / 109.)
  static constexpr int units = RP == 16 && fit > 4 ? 4 : fit < most ? fit : most;
  static_assert(units >= 3, "K and V of a tile, and the next K");
  // Registers that the other warps hand to the softmax from what a thread starts with (launch_one asks).
  static constexpr int start_regs = HD == 64 ? (RP == 8 ? 80 : ctas == 2 ? 64 : 128) : RP == 8 ? 128 : ctas == 2 ? 80 : 168;
  static constexpr int other_regs = HD == 64 ? (RP == 8 ? 64 : ctas == 2 ? 48 : 80) : RP == 8 ? 128 : ctas == 2 ? 64 : 104;
  static constexpr int softmax_regs = HD == 64 ? (RP == 8 ? 112 : ctas == 2 ? 80 : 176) : RP == 8 ? 128 : ctas == 2 ? 88 : 200;
  static constexpr bool moves = softmax_regs != start_regs;
  static_assert(4 * groups * softmax_regs + others * other_regs <= (4 * groups + others) * start_regs, "a split that the launch holds");
  static constexpr int s_col = 0, o_col = 2 * cols;  // TMEM columns: S twice, O of every part
  static constexpr int tmem_need = 2 * cols + parts * pcols;
  static constexpr int tmem = tmem_need <= 64 ? 64 : tmem_need <= 128 ? 128 : tmem_need <= 256 ? 256 : 512;
  static_assert(tmem_need <= 512 && tmem * ctas <= 512, "the SM's columns");
  // shared memory, behind the first 1,024-byte boundary
  static constexpr int q = units * unit;
  static constexpr int p = q + 2 * qimage;
  static constexpr int wmax = p + p_images * pimage;    // float [groups][4 warps][rows]
  static constexpr int wsum = wmax + 4 * RP * 4;     // float [groups][4 warps][rows]
  static constexpr int at = wsum + 4 * RP * 4;       // int [RP]: positions of the piece's rows
  static constexpr int qfactor = at + RP * 4;    // float [2][RP]: a row's u x softmax scale x log2(e)
  static constexpr int scales = qfactor + 2 * RP * 4;   // [kScaleTiles][2][8]: of the keys, of the values
  static constexpr int pieces = scales + kScaleTiles * 64;   // PieceQueue's entries
  static constexpr int bars = pieces + kQueue * 64;
  static constexpr int n_bars = 2 * units + 2 + 2 + 2 + 2 * 2 + 2 * kQueue + 1;
  static constexpr int misc = bars + n_bars * 8;     // ints: abort flag, TMEM address, arrival, stop; scratch of find_run, then NanNotes
  static constexpr int total = misc + 176 + 1024;
  static_assert(kQueue * 64 + n_bars * 8 + 160 <= 1024, "fixed part");
};

struct Bars8 {  // offsets behind [units] full, [units] empty
  static constexpr int q_full = 0, q_empty = 2, s_ready = 4, p_ready = 6, pv_done = 8, queue = 10, drained = queue + 2 * kQueue;
};

// Barrier of a softmax warpgroup that tells whether any of its threads has seen `x`.
__device__ __forceinline__ bool group_any(int wg, bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t"
      "}\n"
      : "=r"(r)
      : "r"((uint32_t)x), "r"(1 + wg)
      : "memory");
  return r != 0;
}

// Two numbers' digits, the first in the low byte: d0 = round(x), d1 = round(16 (x - d0)), d2 = round(256 (x - d0 - d1 / 16)).
template <int kDigits>
__device__ __forceinline__ void digits2(float a, float b, uint32_t (&d)[kDigits]) {
#pragma unroll
  for (int i = 0; i < kDigits; ++i) {
    d[i] = e4m3x2(a, b);
    if (i + 1 < kDigits) {
      const float2 f = float2_of_e4m3x2(d[i]);
      a = (a - f.x) * 16.f;
      b = (b - f.y) * 16.f;
    }
  }
}

// Two weights' digits, the first in the low byte: of their rounding to fp16, whose 11 bits three digits hold.
__device__ __forceinline__ void weight_digits2(float a, float b, uint32_t (&d)[kDigitsY]) {
  __half2 h = __floats2half2_rn(a, b);
#pragma unroll
  for (int i = 0; i < kDigitsY; ++i) {
    d[i] = e4m3x2_of_f16x2(h);
    if (i + 1 < kDigitsY) {
      const uint32_t f = f16x2_of_e4m3x2(d[i]);
      const __half2 sixteen = __float2half2_rn(16.f);
      h = __hfma2(*reinterpret_cast<const __half2*>(&f), __float2half2_rn(-16.f), __hmul2(h, sixteen));   // (exact)
    }
  }
}

// ---- copies by four warps, 16 bytes at a time ----
// The 32 keys of a warp, from `base_key` of a tile on: rows of `kDims` bytes from off (the lane's key's) into a unit.
template <int kDims>
__device__ __forceinline__ void copy_keys8(uint32_t unit, int base_key, const uint8_t* src, long long off) {
  constexpr int kChunks = kDims / 16, kRows = 32 / kChunks;
  const int lane = threadIdx.x & 31, chunk = lane % kChunks, sub = lane / kChunks;
  const uint32_t dst = unit + base_key * kDims;
#pragma unroll
  for (int i = 0; i < 32 / kRows; ++i) {
    const int row = i * kRows + sub;
    const long long o = __shfl_sync(0xffffffffu, off, row);
    copy16(dst + row * kDims + (swizzled_chunk<kDims>(row, chunk) << 4), o >= 0 ? src + o + chunk * 16 : src, o >= 0);
  }
}
// The scales of a warp's two runs of 16 keys: of the first key of each that is visible (they share them).
__device__ __forceinline__ void copy_scales(const Kv8Params& p, uint32_t to, int base_key, int kvh, int blk, int slot) {
  const int lane = threadIdx.x & 31;
  const uint32_t live = __ballot_sync(0xffffffffu, blk >= 0) >> (lane & 16) & 0xffffu;
  const int from = (lane & 16) + (live != 0 ? __ffs(live) - 1 : 0);
  const int b = __shfl_sync(0xffffffffu, blk, from), s = __shfl_sync(0xffffffffu, slot, from);
  if ((lane & 15) < 2) {   // lane 0 the keys', lane 1 the values'
    const int64_t at = (int64_t)b * p.scale_stride_block + (int64_t)((uint32_t)s / (uint32_t)p.scale_tokens) * p.scale_stride_group + (int64_t)kvh * p.scale_stride_head;
    const float* const base = (lane & 15) == 0 ? p.k_scale : p.v_scale;
    copy4(to + (lane & 15) * 32 + (base_key / kRun + (lane >> 4)) * 4, live != 0 ? base + at : base, live != 0);
  }
}

// ---- copies by one warp, in boxes ----
// Where the runs of 16 keys of a tile lie, one per lane of the first eight.
struct TileRuns {
  int key0, lo, hi, kvh;
  int blk, slot;       // the lane's run: block (-1: none that is seen) and first slot
};
__device__ __forceinline__ void tile_runs(const Kv8Params& p, const Piece& it, int t, TileRuns* r) {
  const int lane = threadIdx.x & 31;
  r->key0 = it.key0 + t * kTile;
  r->lo = it.lo;
  r->hi = it.hi;
  r->kvh = it.kvh;
  r->blk = -1;
  const int pos = r->key0 + lane * kRun;
  if (lane < kTile / kRun && pos < r->hi && pos + kRun > r->lo) {
    const int page = p.block_shift >= 0 ? pos >> p.block_shift : (int)((uint32_t)pos / (uint32_t)p.block_size);
    r->slot = pos - page * p.block_size;
    r->blk = __ldg(p.block_table + (int64_t)it.r * p.block_table_row_stride + page);
  }
}
// One unit of the tile's keys or values: boxes that the lanes of `boxes` ask for, and 16-byte copies of the runs `copied`, which zero
// what is not seen.  All lanes; the unit's barrier counts their 32 copies' ends and one arrival with the boxes' bytes.
template <int kDims>
__device__ __forceinline__ void load_unit(const Kv8Params& p, const TileRuns& r, const CUtensorMap& map, const uint8_t* src, int part, uint32_t unit, uint64_t* full,
                                          uint32_t boxes, uint32_t copied) {
  constexpr int kChunks = kDims / 16, kRows = 32 / kChunks;   // 16-byte chunks of a row, rows at a time
  const int lane = threadIdx.x & 31, chunk = lane % kChunks, sub = lane / kChunks;
  if (lane == 0) mbar_arrive_expect_tx(full, __popc(boxes) * p.box_slots * kDims);
  __syncwarp();
  if (boxes >> lane & 1) tma_load_4d(unit + lane * kRun * kDims, &map, part * 128, r.kvh, r.slot, r.blk, full);
#pragma unroll 1
  for (; copied != 0; copied &= copied - 1) {
    const int run = __ffs(copied) - 1, blk = __shfl_sync(0xffffffffu, r.blk, run), slot = __shfl_sync(0xffffffffu, r.slot, run);
    const uint8_t* from = src + (int64_t)blk * p.stride_block + (int64_t)(slot + sub) * p.stride_slot + (int64_t)r.kvh * p.stride_head + part * 128 + chunk * 16;
    const int row0 = run * kRun + sub;
#pragma unroll
    for (int i = 0; i < kRun / kRows; ++i) {
      const int row = row0 + i * kRows, pos = r.key0 + row;
      const bool live = blk >= 0 && pos >= r.lo && pos < r.hi;
      copy16(unit + row * kDims + (swizzled_chunk<kDims>(row, chunk) << 4), live ? from : src, live);
      from += kRows * p.stride_slot;
    }
  }
  copies_arrive(full);
}
// The scales of a tile's runs: lanes 0 to 7 the keys', 8 to 15 the values'.
__device__ __forceinline__ void load_scales(const Kv8Params& p, const TileRuns& r, uint32_t to) {
  const int lane = threadIdx.x & 31, blk = __shfl_sync(0xffffffffu, r.blk, lane & 7), slot = __shfl_sync(0xffffffffu, r.slot, lane & 7);
  if (lane < 16) {
    const int64_t at = (int64_t)blk * p.scale_stride_block + (int64_t)((uint32_t)slot / (uint32_t)p.scale_tokens) * p.scale_stride_group + (int64_t)r.kvh * p.scale_stride_head;
    const float* const base = lane < 8 ? p.k_scale : p.v_scale;
    copy4(to + lane * 4, blk >= 0 ? base + at : base, blk >= 0);
  }
}

// The digits of a piece's queries: one warp, a row by as many lanes as it has pieces of 8 dims, kBatch pieces of a lane in flight.
template <int HD, int RP, bool kHalf>
__device__ __forceinline__ void stage_queries(const Kv8Params& p, const Piece& it, uint8_t* image, float* factor) {
  using G = Geo8<HD, RP, kHalf>;
  constexpr int kLanes = HD / 8, kAtOnce = 32 / kLanes, kSteps = RP / kAtOnce, kBatch = kSteps < 4 ? kSteps : 4;
  const int lane = threadIdx.x & 31, chunk = lane % kLanes, sub = lane / kLanes;
#pragma unroll 1
  for (int s0 = 0; s0 < kSteps; s0 += kBatch) {
    uint4 w[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int n = (s0 + b) * kAtOnce + sub;
      w[b] = make_uint4(0u, 0u, 0u, 0u);
      if (n < it.rows) {
        int token, head;
        row_of(p, it.first_token, it.kvh, it.row0 + n, &token, &head);
        w[b] = __ldg(reinterpret_cast<const uint4*>(p.q + (int64_t)token * p.q_stride_token + (int64_t)head * p.q_stride_head) + chunk);
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int n = (s0 + b) * kAtOnce + sub;
      const uint32_t words[4] = {w[b].x, w[b].y, w[b].z, w[b].w};
      float x[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (kHalf) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&words[i]));
          x[2 * i] = f.x;
          x[2 * i + 1] = f.y;
        } else {
          x[2 * i] = __uint_as_float(words[i] << 16);
          x[2 * i + 1] = __uint_as_float(words[i] & 0xffff0000u);
        }
      }
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // u = 2^e: the row's largest into [128, 256); an empty row takes any.  A row with an infinity is NaN as a whole (not its factor: keys that it does
      // not see have scores of -inf, and those stay)
      const int e = min(120, max(-119, (int)(__float_as_uint(top) >> 23) - 127 - 7));
      const float up = isinf(top) ? NAN : power_of_two(-e);
      uint32_t d[4][G::q_digits];
#pragma unroll
      for (int i = 0; i < 4; ++i) digits2<G::q_digits>(x[2 * i] * up, x[2 * i + 1] * up, d[i]);
      uint8_t* const to = image + (chunk >> 1) * (G::cols * 16) + n * 16 + (chunk & 1) * 8;
#pragma unroll
      for (int g = 0; g < G::q_digits; ++g)
        *reinterpret_cast<uint2*>(to + g * (RP * 16)) = make_uint2(d[0][g] | d[1][g] << 16, d[2][g] | d[3][g] << 16);
      if (chunk == 0) factor[n] = fmaxf(power_of_two(e) * p.scale_log2, 1e-37f);   // (never zero: hidden scores are -inf)
    }
  }
}

// The exponent of the power of two at or above the largest of a tile's eight scales.  Scales of 2^-126, which are those of values that are all zero, do
// not count; where there is no other, the exponent is one that scales of ordinary values are near.
__device__ __forceinline__ int unit_exponent(const float* scales) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = fmaxf(most, scales[i]);
  return most > 0x1p-126f ? min(126, (int)((__float_as_uint(most) + 0x7fffffu) >> 23) - 127) : -7;
}
__device__ __forceinline__ float log2_approx(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Rows of several tokens: keys that some of them see and others do not, [.., lo) and [hi, ..); keys that any of them sees, [first, last).
struct Masks {
  int lo, hi, first, last;
  __device__ __forceinline__ Masks(const Kv8Params& p, const Piece& it) : lo(0), hi(INT_MAX), first(0), last(INT_MAX) {
    if (p.query_start_loc == nullptr) return;
    const int top = it.pos0 + it.row0 / p.group, bottom = it.pos0 + (it.row0 + it.rows - 1) / p.group;   // positions of the first and last row
    if (p.causal) {
      hi = top + 1;
      last = bottom + 1;
    }
    lo = kv8_low(p, bottom);
    first = kv8_low(p, top);
  }
  __device__ __forceinline__ bool divide(int key0) const { return key0 < lo || key0 + kTile > hi; }
  __device__ __forceinline__ bool see(int key0) const { return key0 < last && key0 + kTile > first; }
};
// A value that is NaN under a hidden key: its weight is zero, but zero times NaN is NaN.  So where the rows of a piece do not all see a
// tile's keys, NaN among its values becomes zero in front of the MMA, and where some of them do, its keys are noted: what the rows see of them is put in at the
// piece's end.  The rows are of 32 tokens at most, so such tiles are four at most: key0 is in 158 places about the windows' edges, and in as many about
// the rows' own keys.
constexpr int kNanTiles = 4;
struct NanNotes {
  uint32_t item;           // 1 + the item that they are of
  uint32_t any;
  int tiles, key0[kNanTiles];
  uint32_t keys[kNanTiles][4];
};
static_assert(sizeof(NanNotes) <= 144, "find_run's scratch");
__device__ __forceinline__ void note_tile(NanNotes* notes, uint32_t item, int key0) {   // one thread
  if (notes->item != item) {
    notes->item = item;
    notes->any = 0;
    notes->tiles = 0;
  }
  const int i = min(notes->tiles, kNanTiles - 1);
  notes->key0[i] = key0;
  for (int w = 0; w < 4; ++w) notes->keys[i][w] = 0;
  notes->tiles = i + 1;
}
template <int kDims>
__device__ __forceinline__ void clear_nan(uint8_t* unit, NanNotes* notes) {   // one warp; notes: of the tile noted last, nullptr: none are taken
  uint4* const cells = reinterpret_cast<uint4*>(unit);
#pragma unroll 1
  for (int i0 = threadIdx.x & 31; i0 < kTile * kDims / 16; i0 += 128) {
    uint32_t nan = 0;
#pragma unroll
    for (int i = i0; i < i0 + 128; i += 32) nan |= nan_cells(cells[i].x) | nan_cells(cells[i].y) | nan_cells(cells[i].z) | nan_cells(cells[i].w);
    if (nan == 0) continue;
#pragma unroll 1
    for (int i = i0; i < i0 + 128; i += 32) {
      uint4 v = cells[i];
      if ((take_nan(v.x) | take_nan(v.y) | take_nan(v.z) | take_nan(v.w)) == 0) continue;
      cells[i] = v;
      if (notes == nullptr) continue;
      const int key = i / (kDims / 16);
      atomicOr(&notes->keys[notes->tiles - 1][key >> 5], 1u << (key & 31));
      notes->any = 1;
    }
  }
}
// The rows, of `rows` from row0 of the piece on, that see a key whose value is NaN at dimension d.
__device__ __forceinline__ uint32_t nan_rows(const Kv8Params& p, const Piece& it, const NanNotes* notes, int row0, int rows, int d) {
  uint32_t seen = 0;
#pragma unroll 1
  for (int i = 0; i < 4 * notes->tiles; ++i) {
#pragma unroll 1
    for (uint32_t keys = notes->keys[i >> 2][i & 3]; keys != 0; keys &= keys - 1) {
      const int pos = notes->key0[i >> 2] + (i & 3) * 32 + __ffs(keys) - 1;
      if (pos < it.lo || pos >= it.hi) continue;
      int slot;
      const int blk = block_of(p, it.r, pos, &slot);
      if (blk < 0) continue;
      const uint8_t c = p.v[(int64_t)blk * p.stride_block + (int64_t)slot * p.stride_slot + (int64_t)it.kvh * p.stride_head + d];
      if ((c & 0x7f) != 0x7f) continue;
      for (int n = 0; n < rows; ++n) {
        const int own = it.pos0 + (it.row0 + row0 + n) / p.group;
        if ((!p.causal || pos <= own) && pos >= kv8_low(p, own)) seen |= 1u << n;
      }
    }
  }
  return seen;
}

template <int HD, int RP, bool kHalf, bool kHeld>
__global__ void __launch_bounds__((Geo8<HD, RP, kHalf>::threads), (Geo8<HD, RP, kHalf>::ctas)) kv8_short_kernel(const __grid_constant__ Kv8Params p, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  using G = Geo8<HD, RP, kHalf>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024u - (tc::smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* const full = reinterpret_cast<uint64_t*>(smem + G::bars);
  uint64_t* const empty = full + G::units;
  uint64_t* const bars = empty + G::units;
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + G::misc);
  uint32_t* const tslot = reinterpret_cast<uint32_t*>(smem + G::misc + 4);
  int* const arrival = reinterpret_cast<int*>(smem + G::misc + 8);
  int* const stop = arrival + 1;
  NanNotes* const notes = reinterpret_cast<NanNotes*>(smem + G::misc + 16);   // (where find_run's scratch was)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (warp == G::load_warp && lane < 2 && p.box_slots > 0)
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(lane == 0 ? &k_map : &v_map)) : "memory");
  if (warp == G::mma_warp) {
    if (lane == 0) {
      for (int i = 0; i < G::units; ++i) {
        tc::mbar_init(&full[i], G::load_warps == 4 ? 128 : 33);   // (copies_arrive, load_unit)
        tc::mbar_init(&empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        tc::mbar_init(&bars[Bars8::q_full + i], 1);
        tc::mbar_init(&bars[Bars8::q_empty + i], 1 + G::groups);   // the last QK has read the digits, the softmax the factors
        tc::mbar_init(&bars[Bars8::s_ready + i], 2);   // the MMAs are complete; this warp has seen the tile's scales land
      }
      for (int i = 0; i < 2; ++i) {
        tc::mbar_init(&bars[Bars8::p_ready + i], kSoftmaxThreads * G::groups);
        tc::mbar_init(&bars[Bars8::pv_done + i], 1);
      }
      tc::mbar_init(&bars[Bars8::drained], 1);
      PieceQueue(nullptr, &bars[Bars8::queue], stop).init(4 * G::groups + G::load_warps + 1);
      *abort_flag = 0;
      tc::mbar_init_fence();
    }
    __syncwarp();
    tc::tmem_alloc(tslot, G::tmem);
    tc::tmem_relinquish();
  }
  pdl_wait();
  ShortWalk<RP, Kv8Params> walk = find_run<RP, G::threads>(p, reinterpret_cast<long long*>(smem + G::misc + 16));
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem_base = *tslot;
  if (warp == G::mma_warp && lane == 0) notes->item = 0;   // (read behind PV's barriers)
  PieceQueue queue(reinterpret_cast<Piece*>(smem + G::pieces), &bars[Bars8::queue], stop);
  float* const qfactor = reinterpret_cast<float*>(smem + G::qfactor);
  bool ok = true;
  uint32_t asked = 0;   // units that the loading warp has asked for

  if (warp == G::schedule_warp) {
    // =========================== schedule and queries ============================
    if constexpr (G::moves) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::other_regs));
    Piece it;
    uint32_t item = 0;
    bool going = true;
    while (going && walk.next(p, &it)) {
      if (kv16_held<kHeld>(p, kHeldSchedule, queue.i)) kv16_wait(&bars[Bars8::drained], 0, abort_flag);   // (that nothing arrives on here)
      going = queue.put(it, abort_flag);
      if (!going) break;
      // (behind a wait that gave up the digits may still be read: nothing is written, and the next put ends the queue)
      if (__all_sync(0xffffffffu, item < 2 || kv16_wait<kPieceTimes>(&bars[Bars8::q_empty + (item & 1)], ((item >> 1) - 1) & 1, abort_flag))) {
        stage_queries<HD, RP, kHalf>(p, it, smem + G::q + (item & 1) * G::qimage, qfactor + (item & 1) * RP);
        tc::fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[Bars8::q_full + (item & 1)]);
      }
      ++item;
    }
    if (going) {
      it.tiles = 0;
      queue.put(it, abort_flag);
    }
  } else if (warp >= G::load_warp && warp < G::mma_warp) {
    // =========================== copies ==========================================
    if constexpr (G::moves) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::other_regs));
    if constexpr (G::load_warps == 4) {
      // A warp owns 32 keys of every tile: lane l knows where key l of them lies.
      const int base_key = (warp - G::load_warp) * 32;
      const uint32_t ring = tc::smem_u32(smem), scales = tc::smem_u32(smem + G::scales);
      uint32_t unit = 0, tile = 0;
      auto next_unit = [&]() -> uint32_t {
        const uint32_t s = unit % G::units;
        if (unit >= G::units) ok &= kv16_wait(&empty[s], ((unit / G::units) - 1) & 1, abort_flag);
        ++unit;
        return s;
      };
      {
        KeyLookup keys(p, queue, abort_flag, base_key + lane);
        bool have = keys.fetch(), have_v = false;
        long long off_v = 0;
        int64_t head_v = 0;
        while (have || have_v) {
          const bool now = have;
          long long off = 0;
          int64_t head_k = 0;
          if (now) {
            off = keys.offset();
            const int kvh = keys.it.kvh, blk = keys.blk, slot = keys.slot;
            head_k = (int64_t)kvh * p.stride_head;
            have = keys.fetch();
#pragma unroll
            for (int part = 0; part < G::parts; ++part) {
              const uint32_t s = next_unit();
              if (part == 0) copy_scales(p, scales + (tile++ % kScaleTiles) * 64, base_key, kvh, blk, slot);
              copy_keys8<G::dims>(ring + s * G::unit, base_key, p.k + head_k + part * 128, off);
              copies_arrive(&full[s]);
            }
          }
          if (have_v) {
#pragma unroll
            for (int part = 0; part < G::parts; ++part) {
              const uint32_t s = next_unit();
              copy_keys8<G::dims>(ring + s * G::unit, base_key, p.v + head_v + part * 128, off_v);
              copies_arrive(&full[s]);
            }
          }
          off_v = off;
          head_v = head_k;
          have_v = now;
        }
      }
    } else {
      // (Behind a wait that gave up nothing more is asked for: a unit that is not free may be waiting for its boxes.)
      const uint32_t ring = tc::smem_u32(smem), scales = tc::smem_u32(smem + G::scales);
      uint32_t tile = 0;
      Piece it;
      int left = 0, t = 0;
      TileRuns next;
      next.slot = 0;
      auto fetch = [&]() -> bool {
        if (left == 0) {
          if (!queue.get(&it, abort_flag)) return false;
          left = it.tiles;
          t = 0;
        }
        tile_runs(p, it, t++, &next);
        --left;
        return true;
      };
      // K of a tile is asked for ahead of V of the one before.
      auto units = [&](const TileRuns& r, const CUtensorMap& map, const uint8_t* src, uint32_t boxes, uint32_t copied, bool with_scales) {
#pragma unroll
        for (int part = 0; part < G::parts; ++part, ++asked) {
          const uint32_t s = asked % G::units;
          if (asked >= G::units) ok &= kv16_wait(&empty[s], ((asked / G::units) - 1) & 1, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) return;
          // (the scales go where the unit that is free now says that they have been read)
          if (part == 0 && with_scales) load_scales(p, r, scales + (tile % kScaleTiles) * 64);
          load_unit<G::dims>(p, r, map, src, part, ring + s * G::unit, &full[s], boxes, copied);
        }
      };
      bool have = fetch(), have_v = false;
      TileRuns last;
      uint32_t last_boxes = 0, last_copied = 0;
      while ((have || have_v) && ok) {
        if (kv16_held<kHeld>(p, kHeldCopies, asked)) break;
        const bool now = have;
        TileRuns here = next;
        uint32_t boxes = 0, copied = 0;
        if (now) {
          have = fetch();   // (the look-up of the next tile is on its way while this one's cells are asked for)
          const int pos = here.key0 + lane * kRun;
          if ((uint32_t)here.blk >= (uint32_t)p.num_blocks) here.blk = -1;
          const uint32_t seen = __ballot_sync(0xffffffffu, lane < kTile / kRun && pos < here.hi && pos + kRun > here.lo);
          const uint32_t whole = __ballot_sync(0xffffffffu, here.blk >= 0 && pos >= here.lo && pos + kRun <= here.hi);
          boxes = p.box_slots == 32 ? whole & whole >> 1 & 0x55u : p.box_slots == 16 ? whole : 0u;
          copied = 0xffu & ~(p.box_slots == 32 ? boxes | boxes << 1 : boxes);
          // (scores of keys that nobody sees are replaced, whatever they are: those need no zeros)
          units(here, k_map, p.k, boxes, copied & seen, true);
          ++tile;
        }
        if (have_v && ok) units(last, v_map, p.v, last_boxes, last_copied, false);
        last = here;
        last_boxes = boxes;
        last_copied = copied;
        have_v = now;
      }
    }
    copies_wait_all();
  } else if (warp == G::mma_warp) {
    // =========================== MMAs ============================================
    if constexpr (G::moves) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::other_regs));
    // QK of a tile is issued ahead of PV of the one before, in the order in which the units arrive.
    constexpr uint32_t qk_desc = instr_desc_e4m3(128, G::cols, 0, 0);
    constexpr uint32_t pv_desc = instr_desc_e4m3(128, G::pcols, 1, 1);
    const uint32_t ring = tc::smem_u32(smem), q_s = tc::smem_u32(smem + G::q), p_s = tc::smem_u32(smem + G::p);
    uint32_t unit = 0, tile = 0, item = 0;
    auto arrived = [&]() -> uint32_t {
      const uint32_t s = unit % G::units;
      ok &= kv16_wait(&full[s], (unit / G::units) & 1, abort_flag);
      tc::fence_async_smem();   // (copies wrote through the generic proxy)
      ++unit;
      return s;
    };
    auto qk = [&](bool first_of_item, bool last_of_item) {
      if (first_of_item) ok &= kv16_wait(&bars[Bars8::q_full + (item & 1)], (item >> 1) & 1, abort_flag);
#pragma unroll
      for (int part = 0; part < G::parts; ++part) {
        const uint32_t s = arrived();
        if (elect_one()) {
          tc::fence_after_sync();
#pragma unroll
          for (int kk = 0; kk < G::dims / 32; ++kk) {
            const uint64_t a = unit_desc<G::dims>(ring + s * G::unit + kk * 32, 16);
            const uint64_t b = tc::smem_desc(q_s + (item & 1) * G::qimage + (part * (G::dims / 16) + kk * 2) * (G::cols * 16), G::cols * 16, 128);
            mma_e4m3(tmem_base + G::s_col + (tile & 1) * G::cols, a, b, qk_desc, part > 0 || kk > 0);
          }
          if (ok) tc::mma_commit(&empty[s]);   // (a unit that has not landed is not given back)
          if (part == G::parts - 1) {
            tc::mma_commit(&bars[Bars8::s_ready + (tile & 1)]);
            mbar_arrive(&bars[Bars8::s_ready + (tile & 1)]);
            if (last_of_item) tc::mma_commit(&bars[Bars8::q_empty + (item & 1)]);
          }
        }
        __syncwarp();
      }
      ++tile;
      if (last_of_item) ++item;
    };
    uint32_t pv_tile = 0;
    auto pv = [&](bool first_of_item, bool divided, bool seen, uint32_t its_item, int key0) {
      ok &= kv16_wait(&bars[Bars8::p_ready + pv_tile % G::p_images], (pv_tile / G::p_images) & 1, abort_flag);
#pragma unroll
      for (int part = 0; part < G::parts; ++part) {
        const uint32_t s = arrived();
        if (divided) {
          if (part == 0 && lane == 0 && seen) note_tile(notes, its_item + 1, key0);
          __syncwarp();
          clear_nan<G::dims>(smem + s * G::unit, seen ? notes : nullptr);
          tc::fence_async_smem();
          __syncwarp();
        }
        if (elect_one()) {
          tc::fence_after_sync();
#pragma unroll
          for (int kk = 0; kk < kTile / 32; ++kk) {
            // (64 dims: the instruction's other 64 rows are the same bytes again, which nothing reads)
            const uint64_t a = unit_desc<G::dims>(ring + s * G::unit + kk * 32 * G::dims, 0);
            const uint64_t b = tc::smem_desc(p_s + pv_tile % G::p_images * G::pimage + kk * 512, 128, kTile * 16);
            mma_e4m3(tmem_base + G::o_col + part * G::pcols, a, b, pv_desc, !first_of_item || kk > 0);
          }
          if (ok) tc::mma_commit(&empty[s]);
          if (part == G::parts - 1) tc::mma_commit(&bars[Bars8::pv_done + pv_tile % G::p_images]);
        }
        __syncwarp();
      }
      ++pv_tile;
    };
    Piece it;
    bool pending = false, pending_first = false, pending_divided = false, pending_seen = false;
    uint32_t pending_item = 0;
    int pending_key0 = 0;
    while (queue.get(&it, abort_flag)) {
      const Masks masks(p, it);
      for (int t = 0; t < it.tiles; ++t) {
        if (kv16_held<kHeld>(p, kHeldMma, tile)) break;
        const uint32_t here = item;
        qk(t == 0, t == it.tiles - 1);
        if (pending) pv(pending_first, pending_divided, pending_seen, pending_item, pending_key0);
        pending = true;
        pending_first = t == 0;
        pending_key0 = it.key0 + t * kTile;
        pending_divided = masks.divide(pending_key0);
        pending_seen = masks.see(pending_key0);
        pending_item = here;
      }
    }
    if (pending) pv(pending_first, pending_divided, pending_seen, pending_item, pending_key0);
  } else if (warp < G::load_warp) {
    // =========================== softmax =========================================
    if constexpr (G::moves) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::softmax_regs));
    constexpr int RW = G::rows;
    const int wg = warp >> 2, key = tid & 127, row_base = wg * RW;
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    float* const wmax = reinterpret_cast<float*>(smem + G::wmax) + 4 * row_base;
    float* const wsum = reinterpret_cast<float*>(smem + G::wsum) + 4 * row_base;
    int* const row_at = reinterpret_cast<int*>(smem + G::at) + row_base;
    uint8_t* const p_img = smem + G::p + key * 16;
    auto group_sync = [&] { named_barrier(1 + wg, kSoftmaxThreads); };
    auto all_sync = [&] { named_barrier(1 + G::groups, kSoftmaxThreads * G::groups); };
    uint32_t tile = 0, item = 0;
    zero_requests<HD, RP, kSoftmaxThreads * G::groups>(p);
    {
      const int heads = min(p.num_kv_heads, (int)gridDim.x), hslot = (int)blockIdx.x % heads;
      Piece it;
      while (queue.get(&it, abort_flag)) {
        const int kvh = it.kvh, rows = it.rows - row_base;   // of the group: RW or fewer, or none
        ok &= kv16_wait(&bars[Bars8::q_full + (item & 1)], (item >> 1) & 1, abort_flag);
        const float* const factor = qfactor + (item & 1) * RP + row_base;
        const Masks masks(p, it);
        if (p.query_start_loc != nullptr) {
          if (key < RW) row_at[key] = it.pos0 + (it.row0 + min(row_base + key, it.rows - 1)) / p.group;
          group_sync();
        }
        float ref[RW], l[RW];
        int unit_e = 0;   // U = 2^unit_e
#pragma unroll
        for (int n = 0; n < RW; ++n) {
          ref[n] = kUnset;
          l[n] = 0.f;
        }
        for (int t = 0; t < it.tiles; ++t, ++tile) {
          ok &= kv16_wait(&bars[Bars8::s_ready + (tile & 1)], (tile >> 1) & 1, abort_flag);
          tc::fence_after_sync();
          uint32_t sr[G::q_digits][RW];
#pragma unroll
          for (int g = 0; g < G::q_digits; ++g) tmem_load<RW>(tmem_base + G::s_col + (tile & 1) * G::cols + g * RP + row_base + lane_addr, sr[g]);
          const float* const scale = reinterpret_cast<const float*>(smem + G::scales + (tile % kScaleTiles) * 64);
          const float k_scale = scale[key / kRun], v_scale = scale[8 + key / kRun];
          if (t == 0) unit_e = unit_exponent(scale + 8);
          // (a scale far below U, or zero: its keys' P are 2^90 at most)
          const float value_lg = fmaxf(log2_approx(v_scale) - (float)unit_e, -90.f);
          tc::tmem_ld_wait();
#pragma unroll
          for (int g = 0; g < G::q_digits; ++g) tc::tmem_landed<RW>(sr[g]);
          const int key0 = it.key0 + t * kTile, pos = key0 + key;
          float s[RW], x[RW], top = -INFINITY;   // a key's scores but for the rows' factors; above ref
#pragma unroll
          for (int n = 0; n < RW; ++n) {
            float sum = fmaf(__uint_as_float(sr[1][n]), 0.0625f, __uint_as_float(sr[0][n]));
            if constexpr (G::q_digits == 3) sum = fmaf(__uint_as_float(sr[G::q_digits - 1][n]), 0.00390625f, sum);
            s[n] = sum * k_scale;
          }
          if (pos < it.lo || pos >= it.hi) {
#pragma unroll
            for (int n = 0; n < RW; ++n) s[n] = -INFINITY;
          } else if (masks.divide(key0)) {
#pragma unroll
            for (int n = 0; n < RW; ++n) {
              const int own = row_at[n];
              if ((p.causal && pos > own) || pos < kv8_low(p, own)) s[n] = -INFINITY;
            }
          }
#pragma unroll
          for (int n = 0; n < RW; ++n) {
            x[n] = fmaf(s[n], factor[n], -ref[n]);
            top = fmaxf(top, x[n]);
          }
          const bool outgrown = top + value_lg > kGainY + kSlackY;   // (also where a ref is not set yet)
          if (group_any(wg, outgrown)) {
#pragma unroll
            for (int n = 0; n < RW; ++n) {
              const float m = redux_max(fmaf(s[n], factor[n], value_lg));
              if (lane == 0) wmax[(warp & 3) * RW + n] = m;
            }
            group_sync();
            float alpha[RW];
            bool moved = false;
#pragma unroll
            for (int n = 0; n < RW; ++n) {
              const float m = fmaxf(fmaxf(wmax[n], wmax[RW + n]), fmaxf(wmax[2 * RW + n], wmax[3 * RW + n])) - kGainY;
              const float to = fmaxf(ref[n], m);
              alpha[n] = kv16_exp2(ref[n] - to);
              moved |= alpha[n] != 1.f;
              ref[n] = to;
              l[n] *= alpha[n];
              x[n] = fmaf(s[n], factor[n], -to);
            }
            if (t > 0 && moved) {   // (the same in all of the group's threads)
              ok &= kv16_wait(&bars[Bars8::pv_done + (tile - 1) % G::p_images], ((tile - 1) / G::p_images) & 1, abort_flag);
              tc::fence_after_sync();
#pragma unroll
              for (int d = 0; d < kDigitsY * G::parts; ++d) {
                uint32_t o[RW];
                const uint32_t addr = tmem_base + G::o_col + (d / kDigitsY) * G::pcols + (d % kDigitsY) * RP + row_base + lane_addr;
                tmem_load<RW>(addr, o);
                tc::tmem_ld_wait<RW>(o);
#pragma unroll
                for (int n = 0; n < RW; ++n) o[n] = __float_as_uint(__uint_as_float(o[n]) * alpha[n]);
                tmem_store<RW>(addr, o);
              }
              tc::tmem_st_wait();
            }
            group_sync();  // (the maxima have been read)
          }
          const float y_scale = v_scale * power_of_two(-unit_e);
          uint32_t y[kDigitsY][RW / 4];   // digits of four rows each
#pragma unroll
          for (int n = 0; n < RW; n += 2) {
            const float a = kv16_exp2(x[n]), b = kv16_exp2(x[n + 1]);
            l[n] += a;
            l[n + 1] += b;
            uint32_t d[kDigitsY];
            weight_digits2(a * y_scale, b * y_scale, d);
#pragma unroll
            for (int g = 0; g < kDigitsY; ++g) y[g][n / 4] = n % 4 == 0 ? d[g] : y[g][n / 4] | d[g] << 16;
          }
          if (tile >= G::p_images) ok &= kv16_wait(&bars[Bars8::pv_done + tile % G::p_images], (tile / G::p_images - 1) & 1, abort_flag);   // (the image has been read)
          // column g RP + n: digit g of row n; 16 columns are 16 bytes of the key's
#pragma unroll
          for (int g = 0; g < kDigitsY; ++g) {
            const int c = g * RP + row_base;
            uint8_t* const to = p_img + tile % G::p_images * G::pimage + (c >> 4) * (kTile * 16) + (c & 15);
            if constexpr (RW == 8) *reinterpret_cast<uint2*>(to) = make_uint2(y[g][0], y[g][1]);
            else *reinterpret_cast<uint4*>(to) = make_uint4(y[g][0], y[g][1], y[g][2], y[g][3]);
          }
          tc::fence_async_smem();
          tc::fence_before_sync();
          mbar_arrive(&bars[Bars8::p_ready + tile % G::p_images]);
        }
        // ---- the piece's rows ----
#pragma unroll
        for (int n = 0; n < RW; ++n) {
          if (n < rows) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) l[n] += __shfl_xor_sync(0xffffffffu, l[n], o);
          }
        }
        if (lane == 0) {
#pragma unroll
          for (int n = 0; n < RW; ++n) wsum[(warp & 3) * RW + n] = l[n];
        }
        group_sync();
        if (key == 0) mbar_arrive(&bars[Bars8::q_empty + (item & 1)]);   // (all of the group have read the factors)
        ++item;
#pragma unroll
        for (int n = 0; n < RW; ++n) l[n] = (wsum[n] + wsum[RW + n]) + (wsum[2 * RW + n] + wsum[3 * RW + n]);
        ok &= kv16_wait(&bars[Bars8::pv_done + (tile - 1) % G::p_images], ((tile - 1) / G::p_images) & 1, abort_flag);
        tc::fence_after_sync();
        const bool whole = it.begins && it.ends;
        float* const slot = partial_slot<HD, RP>(p, (int)blockIdx.x, it.begins);
        const float unit_value = power_of_two(unit_e);
        const bool had_nan = notes->item == item && notes->any != 0;   // (the item has been counted already)
#pragma unroll
        for (int part = 0; part < G::parts; ++part) {
          uint32_t o[kDigitsY][RW];
#pragma unroll
          for (int g = 0; g < kDigitsY; ++g) tmem_load<RW>(tmem_base + G::o_col + part * G::pcols + g * RP + row_base + lane_addr, o[g]);
          tc::tmem_ld_wait();
#pragma unroll
          for (int g = 0; g < kDigitsY; ++g) tc::tmem_landed<RW>(o[g]);
          const int d = part * 128 + key;
          if (d < HD) {
            if (had_nan) {
              const uint32_t nan = nan_rows(p, it, notes, row_base, min(rows, RW), d);
#pragma unroll
              for (int n = 0; n < RW; ++n) o[0][n] = nan >> n & 1 ? 0x7fffffffu : o[0][n];
            }
#pragma unroll
            for (int n = 0; n < RW; ++n) {
              if (n < rows) {
                const float v = fmaf(fmaf(__uint_as_float(o[2][n]), 0.0625f, __uint_as_float(o[1][n])), 0.0625f, __uint_as_float(o[0][n])) * unit_value;
                if (whole) {
                  int token, head;
                  row_of(p, it.first_token, kvh, it.row0 + row_base + n, &token, &head);
                  store_out_elem(p.out + (int64_t)token * p.out_stride_token + (int64_t)head * p.out_stride_head, d, kHalf ? PTH_ATTN_F16 : PTH_ATTN_BF16,
                                 l[n] == 0.f ? 0.f : __fdividef(v, l[n]));
                } else {
                  slot[(row_base + n) * HD + d] = v;
                }
              }
            }
          }
        }
        tc::fence_before_sync();
        if (key == 0) {
#pragma unroll
          for (int n = 0; n < RW; ++n) {
            if (n < rows) {
              if (whole) {
                int token, head;
                row_of(p, it.first_token, kvh, it.row0 + row_base + n, &token, &head);
                if (p.lse != nullptr)
                  p.lse[(int64_t)token * p.num_q_heads + head] = l[n] == 0.f ? -INFINITY : (ref[n] + log2f(l[n])) * kLn2;
              } else {
                slot[RP * HD + row_base + n] = ref[n];
                slot[RP * HD + RP + row_base + n] = l[n];
              }
            }
          }
        }
        if (!whole) {
          const int g0 = it.first_cta, g1 = it.last_cta;   // (groups of CTAs)
          all_sync();
          int* const counter = reinterpret_cast<int*>(p.workspace) + g0 * heads + hslot;
          if (tid == 0) {
            *arrival = arrive_at(counter);
            if (*arrival == g1 - g0) *counter = 0;   // (for the next call)
          }
          all_sync();
          if (*arrival == g1 - g0) merge_pieces<HD, RP, kHalf, 4 * G::groups>(p, it, kvh, g0, g1 - g0 + 1, heads, hslot);
        }
        all_sync();  // (the sums and the arrival have been read)
      }
    }
  } else {
    if constexpr (G::moves) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::other_regs));
  }
  tc::fence_before_sync();
  __syncthreads();
  if (*abort_flag) {   // (the same in all threads) what is in flight comes to its end first: MMAs, and boxes
    if (warp == G::mma_warp && elect_one()) {
      tc::mma_commit(&bars[Bars8::drained]);
      kv16_drain(&bars[Bars8::drained], 0);
      atomicOr(&g_kv8_short_status, 32u);
    }
    if (warp == G::load_warp) {   // (boxes are one warp's)
      for (uint32_t u = asked > G::units ? asked - G::units : 0; u < asked; ++u) kv16_drain(&full[u % G::units], (u / G::units) & 1);
    }
    __syncthreads();
  }
  if (warp == G::mma_warp) {
    tc::tmem_dealloc(tmem_base, G::tmem);
  }
  (void)ok;
}

template <int HD, int RP, bool kHalf, bool kHeld = false>
cudaError_t launch_one(const Kv8Params& p, const CUtensorMap& k_map, const CUtensorMap& v_map, cudaStream_t stream) {
  using G = Geo8<HD, RP, kHalf>;
  static_assert(G::total <= 232448, "shared memory of one CTA");
  static_assert(G::ctas == 1 || G::total <= 115712, "shared memory of two CTAs");
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    cudaFuncAttributes attr;
    err = cudaFuncGetAttributes(&attr, kv8_short_kernel<HD, RP, kHalf, kHeld>);
    if (err == cudaSuccess && G::moves && attr.numRegs < G::start_regs) err = cudaErrorInvalidConfiguration;   // (setmaxnreg would wait without end)
    if (err == cudaSuccess) err = cudaFuncSetAttribute(kv8_short_kernel<HD, RP, kHalf, kHeld>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::total);
    if (err != cudaSuccess) return err;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int sms = sm_count();
  if (sms <= 0) return cudaErrorInvalidDevice;
  return pdl_launch(kv8_short_kernel<HD, RP, kHalf, kHeld>, dim3((unsigned)(sms * G::ctas)), dim3(G::threads), G::total, stream, p, k_map, v_map);
}
template <int HD, int RP>
cudaError_t launch_type(const Kv8Params& p, const CUtensorMap& k_map, const CUtensorMap& v_map, cudaStream_t stream) {
  return p.dtype == PTH_ATTN_F16 ? launch_one<HD, RP, true>(p, k_map, v_map, stream) : launch_one<HD, RP, false>(p, k_map, v_map, stream);
}
template <int HD>
cudaError_t launch_rows(const Kv8Params& p, const CUtensorMap& k_map, const CUtensorMap& v_map, cudaStream_t stream) {
  const int64_t rows = (int64_t)p.max_query_len * p.group;
  if (rows <= 8) return launch_type<HD, 8>(p, k_map, v_map, stream);
  if (rows <= 16) return launch_type<HD, 16>(p, k_map, v_map, stream);
  return launch_type<HD, 32>(p, k_map, v_map, stream);
}

}  // namespace

// Counters, and two partial row tiles per CTA: twice the SMs' number of CTAs with 16 rows, or as many with 32.
int64_t kv8_short_workspace_bytes(int head_size, int num_sms) {
  return kCounterBytes + (int64_t)num_sms * 2 * 2 * 16 * (head_size + 2) * 4;
}

namespace {
// Boxes of 32 slots where pages are whole numbers of them (a piece's tiles begin at multiples of 32 keys), else of 16.
void make_maps(Kv8Params& q, CUtensorMap* k_map, CUtensorMap* v_map) {
  q.box_slots = q.head_size == 64 ? 0 : q.block_size % 32 == 0 ? 32 : 16;
  if (q.box_slots > 0 && (!cell_box_map(q, q.k, q.box_slots, k_map) || !cell_box_map(q, q.v, q.box_slots, v_map))) q.box_slots = 0;
}
}  // namespace

cudaError_t launch_kv8_short_held(const Kv8Params& p, cudaStream_t stream) {
  Kv8Params q = p;
  CUtensorMap k_map{}, v_map{};
  make_maps(q, &k_map, &v_map);
  return launch_one<128, 8, false, true>(q, k_map, v_map, stream);
}
cudaError_t launch_kv8_short(const Kv8Params& p, cudaStream_t stream) {
  Kv8Params q = p;
  CUtensorMap k_map{}, v_map{};
  make_maps(q, &k_map, &v_map);
  switch (p.head_size) {
    case 64:
      return launch_rows<64>(q, k_map, v_map, stream);
    case 128:
      return launch_rows<128>(q, k_map, v_map, stream);
    default:
      return launch_rows<256>(q, k_map, v_map, stream);
  }
}

// Reads and clears this kernel's status word (device must be idle).
cudaError_t read_kv8_short_status(unsigned int* v) {
  unsigned int zero = 0;
  cudaError_t err = cudaMemcpyFromSymbol(v, g_kv8_short_status, sizeof(*v));
  if (err != cudaSuccess) return err;
  return cudaMemcpyToSymbol(g_kv8_short_status, &zero, sizeof(zero));
}

}  // namespace pthb200
