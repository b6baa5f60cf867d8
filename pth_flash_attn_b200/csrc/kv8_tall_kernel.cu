// Attention over the 8-bit paged cache for requests of many query rows: prompts, chunks of prompts, wide verification.
//
// Orientation: query rows on the MMA's M dimension, a thread per row in the softmax:
//   S[row, key] = sum_d Q[row, d] c_K[key, d]    A = digits of Q, B = c_K as it lies in the cache (kind::f8f6f4), accumulator in TMEM
//   O[row, d]  += sum_key Y[row, key] c_V[key, d]  A = Y = P scale_V / U in TMEM over S, B = c_V in fp16 (kind::f16)
// An SM holds two row tiles of 128 rows: of one CTA at 128 dims, where every tile of keys then serves twice, of two CTAs at 64 dims; at
// 256 dims O alone takes half of TMEM: one row tile.  A step is 64 keys; S has two buffers, so that a step's QK and the last
// one's PV run beside its softmax.
//
// Q is a sum of e4m3 digits (two for bf16, three for fp16), all in one accumulator: x = u (d0 + d1 + d2), u a power of two per row that
// puts the row's largest into (224, 448].  A digit is the rounding of what is left, so bf16 numbers are exact down to 2^-10 of their row's
// largest and off by 2^-17 of it at most below.  Two MMAs over 8-bit operands take as long as one over 16-bit ones.
// V passes through registers once per tile: fp16 holds every e4m3 number.  Its scale goes into the weights, in 32 bits, ahead of their one rounding to
// fp16: U is the largest scale that the row has seen so far in the piece (O is rescaled where a step brings a larger one), so weights are at most
// P, and keys that a row does not see change nothing for it, whatever their scale.  (With c_V scale_V / U as operand B and a U for all rows, a scale that is
// no power of two was rounded to 11 bits itself, the same way for all its keys, and a scale 2^25 times the others', under keys that a row did not see,
// left nothing of those that it did.)  So Y needs no digits: one 16-bit number, with 32-bit sums; its rounding by 2^-11 is an eighth of that
// of a bf16 result (fp16 results are off by 2.6e-4 of their norm, by 2.0e-4 with weights of 32 bits).
//
// Softmax in one pass: ref is a running bound of a row's scores (log2 units), P = 2^(s - ref), l = sum P, ref kGain below the maximum of
// a row's first 64 keys.  Later ones need no maximum: the sum of 64 P says whether one of them has outgrown ref too far
// (kMostSum); then ref moves to their maximum, O and l are rescaled and the 64 are computed again.
//
// Warps: softmax (four per row tile), which also ask for a piece's queries, while the last one's rows go out, and make their digits; four
// that widen V; one that works out the pieces and asks for their cells, by TMA boxes of 16 slots (a page holds a whole number of them), and for
// the scales; an MMA warp per row tile.
//
// What bounds it.  A step's softmax, 1,300 to 1,500 clocks of 64 exponentials and their conversions a row, beside 300 to 500 of waiting for S; power
// (the 1,000 W limit) in long calls; a piece's own 8,000 to 10,000 clocks (queries, first S, rows, merge) in short ones.  Measured (bf16 unless
// said, calls behind one another): four chunks of 2,048 tokens over 8,192 keys before them, 32 heads of 8, 128 dims: 1,100 to 1,240 us (1,285 among other
// work), 0.58 to 0.68 of the bf16 rate of a library product (fp16 1,380; 16 heads of 16, 64 dims, 590 to 650).  Twelve prompts of 37 to 2,500 tokens: 16 heads of 16, 64 dims,
// fp16, 164 us; 32 heads of 8, 128 dims, 316 to 336 us.  256 dims, the same chunks: 3,210 to 3,300 us, one row tile per SM.
//
// Schedule: the rows of a request and KV head in row tiles, a first one together with a last one, so that under a causal mask
// these units are about equally long; all units form one sequence in KV tiles of 128 keys, which is cut into equal runs, one per
// CTA.  The pieces of a row tile that a cut divides are merged by the CTA that arrives last.
#include "kv8.cuh"

#include "kv8_boxes.cuh"
#include "pdl.cuh"
#include "umma_rows.cuh"

namespace pthb200 {

__device__ unsigned int g_kv8_tall_status = 0;

namespace {

constexpr float kGainP = 7.f;          // log2 of P of a row's largest score when its reference is set
constexpr float kMostSum = 0x1p15f;    // of 64 P
constexpr int kKeys = 64;              // of a step
constexpr int kWidenWarps = 4;
// KV tiles that a row tile counts besides its own: its queries, its first maximum and its rows' way out.  (With 1, 2, 3, 4 and 6, the twelve
// prompts above: 183, 172, 166, 166, 169 us at 64 dims, 358, 325, 316, 315, 323 at 128.)
constexpr int kItemTiles = 3;

template <int HD, bool kHalf>
struct Tall8 {
  static constexpr int rts = HD == 128 ? 2 : 1;      // row tiles of 128 rows
  static constexpr int ctas = HD == 64 ? 2 : 1;      // per SM
  static constexpr int rows = 128 * rts;
  static constexpr int dims = HD < 128 ? HD : 128;   // of a TMA box, and of a PV accumulator
  static constexpr int parts = HD / dims;
  static constexpr int q_digits = kHalf ? 3 : 2;
  static constexpr int raw = kKeys * HD;             // cells of a step: parts of 64 rows of dims bytes, swizzled
  static constexpr int wide = kKeys * HD * 2;        // W of a step: slabs of 64 dims, 64 rows of 128 bytes, swizzled
  static constexpr int q_digit = 128 * HD;           // column block c of 16 dims at c 2,048, row r at r 16
  static constexpr int q_tile = q_digits * q_digit;
  static constexpr int k_units = HD == 64 ? 4 : HD == 128 ? (kHalf ? 4 : 6) : (kHalf ? 2 : 3);
  // Steps that the loading warp asks for together: with one its own instructions took as long as a step, and the MMAs waited for keys (the chunks 617
  // instead of 553 us at 64 dims, 1,297 instead of 1,196 at 128; 256 dims have no room for two).
  static constexpr int at_once = HD == 256 ? 1 : 2;
  static constexpr int v_units = HD == 64 ? 4 : HD == 128 ? (kHalf ? 3 : 4) : 2;
  static constexpr int w_units = HD == 64 ? 4 : HD == 128 ? 3 : 2;
  // Steps whose scales are kept.  A unit of K that is free again says that QK of its step is complete, which waited for P of two steps before.
  static constexpr int scale_steps = HD == 256 ? 8 : 16;
  static_assert(k_units + at_once + 1 < scale_steps, "scales outlive their readers");
  static constexpr int softmax_warps = 4 * rts;
  static constexpr int widen_warp = softmax_warps, load_warp = widen_warp + kWidenWarps, mma_warp = load_warp + 1;
  static constexpr int threads = (mma_warp + rts) * 32;
  // Registers that a thread starts with (launch_one asks), which setmaxnreg moves from the widening warps to the softmax: as many as leave
  // both without spills.  (Widening and softmax with 64 and 128, 56 and 136, 32 and 160 at 64 dims: 177, 174, 178 us for the twelve prompts, 166, 155,
  // 155 for 512 of 64 tokens; with 64 and 160, 96 and 144, 80 and 152 at 128 dims: 369, 370, 358.)
  static constexpr int start_regs = HD == 256 ? 168 : HD == 128 ? 128 : 96;
  static constexpr int widen_regs = HD == 256 ? 104 : HD == 128 ? 80 : 56, softmax_regs = HD == 256 ? 232 : HD == 128 ? 152 : 136;
  static_assert(softmax_warps * softmax_regs + kWidenWarps * widen_regs <= (softmax_warps + kWidenWarps) * start_regs, "a split that the launch holds");
  static constexpr int s_col = 0, o_col = 2 * rts * kKeys;   // TMEM columns: S(rt, b) at (2 rt + b) 64, O(rt) at o_col + rt HD
  static constexpr int tmem = HD == 64 ? 256 : 512;
  static_assert(o_col + rts * HD <= tmem, "accumulators");
  // shared memory, behind the first 1,024-byte boundary
  static constexpr int v = k_units * raw;
  static constexpr int w = v + v_units * raw;
  static constexpr int q = w + w_units * wide;
  static constexpr int raw_q = q + rts * q_tile;     // query rows as they are (others: in the place of their digits)
  static constexpr int scales = raw_q + (HD == 64 ? 128 * HD * 2 : 0);   // float [kScaleSteps][2][4]: of the keys' runs of 16, of the values'
  static constexpr int bars = scales + scale_steps * 32;
  static constexpr int k_full = 0, k_empty = k_full + k_units, v_full = k_empty + k_units, v_empty = v_full + v_units, w_full = v_empty + v_units,
                       w_empty = w_full + w_units, q_full = w_empty + w_units, s_ready = q_full + rts, p_ready = s_ready + 2 * rts,
                       pv_done = p_ready + 2 * rts, queue = pv_done + 2 * rts, drained = queue + 2 * kQueue,
                       n_bars = drained + rts;
  static constexpr int pieces = bars + n_bars * 8;   // PieceQueue's entries
  // Steps of a piece that some of its rows do not see whole (edges8), at most: in front of the last row's window 4 (of 128 rows) or 6
  // (256), from the first row's own key on 3 or 5.
  static constexpr int nan_steps = rows == 128 ? 8 : 12;
  static constexpr int nan_words = 1 + 2 * nan_steps;
  // Pieces whose notes are kept: these are cleared in front of a piece's entry into the queue, when all warps have begun the piece kQueue + 1 before.
  static constexpr int nan_pieces = kQueue + 2;
  static constexpr int nan = pieces + kQueue * 64;   // uint32_t [nan_pieces][nan_words]: whether there is any; 64 keys of each such step
  static constexpr int misc = nan + (nan_pieces * nan_words + 1) / 2 * 8;   // ints: abort flag, TMEM address, arrivals [2], stop; scratch of find_run
  static constexpr int total = misc + 32 + (threads / 32 + 2) * 8 + 1024;
  static_assert(total <= (ctas == 2 ? 115712 : 232448), "shared memory");
};

// ---- schedule ----

// Keys and length of row tile rt: at least one tile, which then has no visible key.
struct RowTile8 {
  int lo, hi, tiles;
};
template <int RP>
__device__ __forceinline__ RowTile8 row_tile8(const Kv8Params& p, const ReqShape8& s, int rt) {
  RowTile8 t;
  const int rows = s.tokens * p.group;
  t.lo = kv8_low(p, s.pos0 + rt * RP / p.group);
  t.hi = p.causal ? kv8_high(p, s.pos0 + (min(rows, (rt + 1) * RP) - 1) / p.group, 0) : s.hi;
  t.tiles = max(1, (t.hi + kTile - 1) / kTile - t.lo / kTile);
  return t;
}
// Lengths in the sequence, in KV tiles: of a first and a last row tile together, of the one in the middle of an odd number, and of
// all of a KV head.  (Pairs may be longer or shorter than those this goes by: a row tile's last piece takes what is left.  Under a causal mask by some tiles; under a
// window by up to its own length: the longest run of 8,192 fresh tokens with a window of 4,096 is 1.36 of the mean one.)
struct Units8 {
  int pairs, pair, middle;
  long long head;
};
template <int RP>
__device__ __forceinline__ Units8 units8(const Kv8Params& p, const ReqShape8& s) {
  Units8 u{0, 0, 0, 0};
  if (s.tiles == 0) return u;
  const int n = s.row_tiles;
  u.pairs = n / 2;
  if (n >= 2) u.pair = row_tile8<RP>(p, s, 0).tiles + row_tile8<RP>(p, s, n - 1).tiles;
  if (n >= 4) u.pair = max(u.pair, row_tile8<RP>(p, s, 1).tiles + row_tile8<RP>(p, s, n - 2).tiles);
  u.pair += 2 * kItemTiles;
  if (n & 1) u.middle = row_tile8<RP>(p, s, n / 2).tiles + kItemTiles;
  u.head = (long long)u.pairs * u.pair + u.middle;
  return u;
}
// The run of a CTA: a walk over its pieces.
template <int RP>
struct TallWalk8 {
  long long at, end, start;   // position in the sequence, end of the run, start of request r
  int r, runs;                // runs that the sequence is cut into
  long long work;             // length of the sequence
  __device__ __forceinline__ int owner(long long x) const { return (int)(((x + 1) * runs - 1) / work); }
  __device__ __forceinline__ bool next(const Kv8Params& p, Piece* out) {
    for (;;) {
      if (at >= end) return false;
      ReqShape8 s = req_shape<RP>(p, r);
      Units8 u = units8<RP>(p, s);
      while (at >= start + u.head * p.num_kv_heads) {
        start += u.head * p.num_kv_heads;
        ++r;
        s = req_shape<RP>(p, r);
        u = units8<RP>(p, s);
      }
      const int kvh = (int)((at - start) / u.head);
      const long long head = start + (long long)kvh * u.head, off = at - head;
      const bool middle = off >= (long long)u.pairs * u.pair;
      const int pair = middle ? u.pairs : (int)(off / u.pair);
      const long long base = head + (long long)pair * u.pair;   // of the unit
      const int length = middle ? u.middle : u.pair, a = (int)(at - base);
      // the unit's first row tile takes [0, split), the last one what is left
      int rt = pair, from = 0, to = length;
      RowTile8 t = row_tile8<RP>(p, s, rt);
      if (!middle) {
        const int split = min(length - 1, t.tiles + kItemTiles);
        if (a >= split) {
          rt = s.row_tiles - 1 - pair;
          t = row_tile8<RP>(p, s, rt);
          from = split;
        } else {
          to = split;
        }
      }
      const int b = (int)min((long long)to, a + (end - at));
      at += b - a;
      const int tile = max(0, a - from - kItemTiles), stop = b == to ? t.tiles : min(t.tiles, b - from - kItemTiles);
      if (stop <= tile) continue;   // (no keys yet, or none left)
      out->r = r;
      out->kvh = kvh;
      out->row0 = rt * RP;
      out->rows = min(RP, s.tokens * p.group - rt * RP);
      out->first_token = s.first;
      out->key0 = (t.lo / kTile + tile) * kTile;
      out->lo = t.lo;
      out->hi = t.hi;
      out->tiles = stop - tile;
      out->begins = tile == 0;
      out->ends = stop == t.tiles;
      // (the first tile may be in front of the unit's end by less than kItemTiles; the last one belongs to whom the end does at most)
      out->first_cta = owner(base + min(from + kItemTiles, to - 1));
      out->last_cta = owner(base + min(from + kItemTiles + t.tiles, to) - 1);
      out->pos0 = s.pos0;
      return true;
    }
  }
};
// Cuts the sequence.  Every CTA sums the requests' lengths up for itself.  scratch: 64-bit words, warps + 2.
template <int RP, int kThreads>
__device__ __forceinline__ TallWalk8<RP> find_run8(const Kv8Params& p, long long* scratch) {
  constexpr int kWarps = kThreads / 32;
  const int tid = threadIdx.x, per = (p.num_reqs + kThreads - 1) / kThreads, r0 = min(p.num_reqs, tid * per), r1 = min(p.num_reqs, r0 + per);
  TallWalk8<RP> w;
  long long mine = 0;
#pragma unroll 1
  for (int r = r0; r < r1; ++r) mine += units8<RP>(p, req_shape<RP>(p, r)).head * p.num_kv_heads;
  const long long before = scan_threads<kThreads>(mine, scratch, &w.work);
  w.runs = (int)min((long long)gridDim.x, max(w.work, 1ll));   // (none of them empty)
  w.at = (int)blockIdx.x < w.runs ? w.work * blockIdx.x / w.runs : w.work;
  w.end = (int)blockIdx.x < w.runs ? w.work * (blockIdx.x + 1) / w.runs : w.work;
  if (w.at < w.end && before <= w.at && w.at < before + mine) {
    long long start = before;
    int r = r0;
#pragma unroll 1
    for (;; ++r) {
      const long long n = units8<RP>(p, req_shape<RP>(p, r)).head * p.num_kv_heads;
      if (w.at < start + n) break;
      start += n;
    }
    scratch[kWarps] = r;
    scratch[kWarps + 1] = start;
  }
  __syncthreads();
  w.r = (int)scratch[kWarps];
  w.start = scratch[kWarps + 1];
  return w;
}
// Steps of a piece: its keys from key0 on, as far as its row tile sees them; one at least.
__device__ __forceinline__ int steps8(const Piece& it) { return max(1, (min(it.tiles * kTile, it.hi - it.key0) + kKeys - 1) / kKeys); }

// Behind any of a CTA's waits may stand a row tile whose rows are on their way out, merged or not: all have the bound of whole pieces (but
// in the test's instances, which wait for it to pass).
template <bool kHeld>
__device__ __forceinline__ bool piece_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return kv16_wait<kHeld ? 1u : kPieceTimes>(bar, parity, abort_flag);
}

// ---- operands ----

template <bool kAccumulate>
__device__ __forceinline__ void mma_e4m3_words(uint32_t d_tmem, uint32_t alo, uint32_t ahi, uint32_t blo, uint32_t bhi, uint32_t idesc) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %2};\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %5, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "r"(alo), "r"(ahi), "r"(blo), "r"(bhi), "r"(idesc), "n"(kAccumulate ? 1 : 0)
      : "memory");
}
// Swizzled operand descriptor of raw rows: 128 bytes, or 64 bytes in the 64-byte swizzle.
template <int HD>
__device__ __forceinline__ uint64_t raw_desc(uint32_t saddr) {
  if constexpr (HD == 64) return tc::smem_desc(saddr, 16, 512) | (uint64_t)4 << 61;
  return swizzled_desc(saddr, 16, 1024);
}
// Four cells as fp16, which holds them all; NaN stays.
__device__ __forceinline__ uint2 widen4(uint32_t w) { return make_uint2(f16x2_of_e4m3x2(w & 0xffffu), f16x2_of_e4m3x2(w >> 16)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// A run's factor of its scores: never zero, since a hidden score is -inf under a scale of zero too; NaN stays NaN.
__device__ __forceinline__ float score_factor(float scale, float q_factor) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(scale * q_factor), "f"(1e-37f));
  return r;
}
template <int HD, bool kHalf>
__device__ __forceinline__ float* tall8_slot(const Kv8Params& p, int cta, bool begins) {
  // [HD][rows] O, [rows] ref, [rows] l
  return reinterpret_cast<float*>(p.workspace + kCounterBytes) + (int64_t)(2 * cta + (begins ? 1 : 0)) * (Tall8<HD, kHalf>::rows * (HD + 2));
}

// P of 64 scores, 2^(score factor + minus_ref), a factor for every 16 of them, times a weight for every 16 of them, to TMEM as pairs of fp16 numbers; returns
// the sum of P.  (Kept in registers until the step is settled, these and the scores were more than 64 dims' warps have: what spilled went
// round in the first level cache, which shared memory leaves small.)
__device__ __forceinline__ float exponentials8(const uint32_t (&r)[64], const float (&factor)[4], float minus_ref, const float (&weight)[4], uint32_t p_tmem) {
  const f32x2 ref2 = pair(minus_ref, minus_ref);
  f32x2 sum[2] = {0ull, 0ull};
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int n = part * 16 + i;
      float x, y;
      unpair(fma2(pair(__uint_as_float(r[2 * n]), __uint_as_float(r[2 * n + 1])), pair(factor[n / 8], factor[n / 8]), ref2), x, y);
      x = ex2f(x);
      y = ex2f(y);
      sum[n & 1] = add2(sum[n & 1], pair(x, y));
      unpair(mul2(pair(x, y), pair(weight[n / 8], weight[n / 8])), x, y);
      pk[i] = pack_f16(x, y);
    }
    tc::tmem_st16(p_tmem + part * 16, pk);
  }
  return sum_pairs(sum);
}

__device__ __forceinline__ int64_t scale_at(const Kv8Params& p, int kvh, int blk, int slot) {
  return (int64_t)blk * p.scale_stride_block + (int64_t)((uint32_t)slot / (uint32_t)p.scale_tokens) * p.scale_stride_group + (int64_t)kvh * p.scale_stride_head;
}

// Asks for a warp's 32 query rows of a piece, as they are: row n at raw + n 2 HD, its 16-byte pieces swizzled by n.
template <int HD>
__device__ __forceinline__ void copy_rows(const Kv8Params& p, const Piece& it, int row0, uint32_t raw) {
  constexpr int kChunks = HD / 8, kRows = 32 / kChunks;   // pieces of a row, rows at a time
  const int lane = threadIdx.x & 31, chunk = lane % kChunks, sub = lane / kChunks;
  if (it.rows <= row0) return;
  int token, head;
  row_of(p, it.first_token, it.kvh, it.row0 + min(row0 + lane, it.rows - 1), &token, &head);
  const long long off = (long long)token * p.q_stride_token + (long long)head * p.q_stride_head;
#pragma unroll 4
  for (int i = 0; i < 32 / kRows; ++i) {
    const int row = i * kRows + sub;
    copy16(raw + row * (2 * HD) + ((chunk ^ (row & 7)) << 4), p.q + __shfl_sync(0xffffffffu, off, row) + chunk * 16, true);
  }
}
// The digits of a query row, by its thread, to `image`; wait(): all of the row tile have read their rows.  Returns u x softmax scale x log2(e),
// below zero for a row that is not finite.
template <int HD, bool kHalf, class Wait>
__device__ __forceinline__ float stage_row(const Kv8Params& p, const uint8_t* raw, int row, uint8_t* image, Wait wait) {
  using G = Tall8<HD, kHalf>;
  constexpr bool kKept = HD != 64;   // all of the row in registers: its place is the image's
  auto chunk = [&](int c) { return *reinterpret_cast<const uint4*>(raw + ((c ^ (row & 7)) << 4)); };
  uint4 kept[kKept ? HD / 8 : 1];
  uint32_t m = 0;   // largest magnitudes, as 16-bit integers
#pragma unroll
  for (int c = 0; c < HD / 8; ++c) {
    const uint4 w = chunk(c);
    if constexpr (kKept) kept[c] = w;
    m = __vimax3_u16x2(m, w.x & 0x7fff7fffu, w.y & 0x7fff7fffu);
    m = __vimax3_u16x2(m, w.z & 0x7fff7fffu, w.w & 0x7fff7fffu);
  }
  if constexpr (kKept) wait();
  const uint32_t top16 = max(m & 0xffffu, m >> 16);
  const bool finite = top16 < (kHalf ? 0x7c00u : 0x7f80u);
  const float top = kHalf ? __half2float(__ushort_as_half((unsigned short)top16)) : __uint_as_float(top16 << 16);
  const int e = min(119, max(-119, e4m3_exponent(top)));
  const float up = power_of_two(-e);
  // (Rolled at 64 dims: what runs once a piece costs by its instructions, which come from beyond the first caches.  Twelve
  // prompts of 37 to 2,500 tokens, rolled and not, us: 174 / 182 at 64 dims, 402 / 357 at 128.)
#pragma unroll(HD == 64 ? 1 : HD / 16)
  for (int c = 0; c < HD / 16; ++c) {
    const uint4 w0 = kKept ? kept[kKept ? 2 * c : 0] : chunk(2 * c), w1 = kKept ? kept[kKept ? 2 * c + 1 : 0] : chunk(2 * c + 1);
    const uint32_t pairs[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
    uint32_t d[G::q_digits][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float2 f;
      if constexpr (kHalf) f = __half22float2(*reinterpret_cast<const __half2*>(&pairs[i]));
      else f = make_float2(__uint_as_float(pairs[i] << 16), __uint_as_float(pairs[i] & 0xffff0000u));
      __half2 h = __floats2half2_rn(f.x * up, f.y * up);   // (exactly, down to 2^-24, which is far below a digit's last step)
#pragma unroll
      for (int g = 0; g < G::q_digits; ++g) {
        const uint32_t b = e4m3x2_of_f16x2(h);
        if (i & 1) d[g][i / 2] |= b << 16; else d[g][i / 2] = b;
        if (g + 1 < G::q_digits) {
          const uint32_t done = f16x2_of_e4m3x2(b);
          h = __hsub2(h, *reinterpret_cast<const __half2*>(&done));
        }
      }
    }
#pragma unroll
    for (int g = 0; g < G::q_digits; ++g) *reinterpret_cast<uint4*>(image + g * G::q_digit + c * 2048) = make_uint4(d[g][0], d[g][1], d[g][2], d[g][3]);
  }
  return finite ? power_of_two(e) * p.scale_log2 : -1.f;
}

// A value that is NaN under a key that a row does not see would make the row's sum NaN all the same: its weight is zero, but zero times NaN
// is NaN.  So in the steps that some of a piece's rows do not see whole, the widening warps make NaN zero and note the key; at
// the piece's end a row puts NaN where one of those that it sees has it.  Such steps are few, at a piece's ends, so the others' cells
// are not looked at (of all, prompts of 37 to 2,500 tokens took 276 us instead of 237), and what is put in costs by the keys noted.
//
// Piece::edges: steps at its beginning, in front of what the last row sees, + 16 times those at its end, behind what the first row sees.
__device__ __forceinline__ int edges8(const Kv8Params& p, const Piece& it) {
  const int steps = steps8(it), hi = p.causal ? max(0, it.pos0 + it.row0 / p.group + 1) : INT_MAX;
  const int lo = p.window > 0 ? kv8_low(p, it.pos0 + (it.row0 + it.rows - 1) / p.group) : 0;
  const int below = min(steps, (max(0, lo - it.key0) + kKeys - 1) / kKeys), from = min(steps, max(below, max(0, hi - it.key0) / kKeys));
  return below | (steps - from) << 4;
}
struct Edges8 {
  int below, from, notes;   // steps [0, below) and [from, ..), their number
  __device__ __forceinline__ Edges8(const Piece& it, int steps) : below(it.edges & 15), from(steps - (it.edges >> 4)), notes(below + (it.edges >> 4)) {}
  __device__ __forceinline__ bool has(int step) const { return step < below || step >= from; }
  __device__ __forceinline__ int note_of(int step) const { return step < below ? step : below + step - from; }
  __device__ __forceinline__ int step_of(int note) const { return note < below ? note : from + note - below; }
};
// The columns of a row that are NaN by a key that was noted and that the row sees, [lo, hi): 16 to a word.  (A function of its own, which the
// hot code does not run through; only softmax threads call it, who have more registers than the launch gave.)
template <int HD>
__device__ __noinline__ void nan_columns(const Kv8Params& p, const Piece& it, const uint32_t* noted, int lo, int hi, uint32_t* columns) {
  const Edges8 edges(it, steps8(it));
  for (int c = 0; c < HD / 16; ++c) columns[c] = 0u;
#pragma unroll 1
  for (int i = 0; i < 2 * edges.notes; ++i) {
#pragma unroll 1
    for (uint32_t keys = noted[1 + i]; keys != 0; keys &= keys - 1) {
      const int pos = it.key0 + edges.step_of(i / 2) * kKeys + (i & 1) * 32 + __ffs(keys) - 1;
      if (pos < lo || pos >= hi) continue;
      int slot;
      const int blk = block_of(p, it.r, pos, &slot);
      if (blk < 0) continue;
      const uint4* const v = reinterpret_cast<const uint4*>(p.v + (int64_t)blk * p.stride_block + (int64_t)slot * p.stride_slot + (int64_t)it.kvh * p.stride_head);
      auto four = [](uint32_t w) { return (nan_cells(w) >> 7) * 0x01020408u >> 24 & 15u; };   // (bytes' top bits side by side)
#pragma unroll 4
      for (int c = 0; c < HD / 16; ++c) {
        const uint4 w = v[c];
        columns[c] |= four(w.x) | four(w.y) << 4 | four(w.z) << 8 | four(w.w) << 12;
      }
    }
  }
}

template <int HD, bool kHalf, bool kHeld>
__global__ void __launch_bounds__((Tall8<HD, kHalf>::threads), (Tall8<HD, kHalf>::ctas)) kv8_tall_kernel(const __grid_constant__ Kv8Params p, const __grid_constant__ CUtensorMap k_map,
                                                                        const __grid_constant__ CUtensorMap v_map) {
  using G = Tall8<HD, kHalf>;
  constexpr int RP = G::rows;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024u - (tc::smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + G::bars);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + G::misc);
  uint32_t* const tslot = reinterpret_cast<uint32_t*>(smem + G::misc + 4);
  int* const arrival = reinterpret_cast<int*>(smem + G::misc + 8);   // [2]
  int* const stop = arrival + 2;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (warp == G::mma_warp) {
    if (lane == 0) {
      for (int i = 0; i < G::k_units; ++i) {
        tc::mbar_init(&bars[G::k_full + i], 12);        // one arrival per run of 16 keys, and one per scale
        tc::mbar_init(&bars[G::k_empty + i], G::rts);   // one commit per row tile
      }
      for (int i = 0; i < G::v_units; ++i) {
        tc::mbar_init(&bars[G::v_full + i], 4);
        tc::mbar_init(&bars[G::v_empty + i], kWidenWarps);
      }
      for (int i = 0; i < G::w_units; ++i) {
        tc::mbar_init(&bars[G::w_full + i], kWidenWarps);
        tc::mbar_init(&bars[G::w_empty + i], G::rts);
      }
      for (int i = 0; i < G::rts; ++i) {
        tc::mbar_init(&bars[G::q_full + i], 128);
        tc::mbar_init(&bars[G::drained + i], 1);
      }
      for (int i = 0; i < 2 * G::rts; ++i) {
        tc::mbar_init(&bars[G::s_ready + i], 2);        // the MMAs are complete; who issued them has seen the step's scales land
        tc::mbar_init(&bars[G::p_ready + i], 128);
        tc::mbar_init(&bars[G::pv_done + i], 1);
      }
      PieceQueue(nullptr, &bars[G::queue], stop).init(G::threads / 32 - 1);
      *abort_flag = 0;
      tc::mbar_init_fence();
    }
    __syncwarp();
    tc::tmem_alloc(tslot, G::tmem);
    tc::tmem_relinquish();
  }
  pdl_wait();
  const TallWalk8<RP> plan = find_run8<RP, G::threads>(p, reinterpret_cast<long long*>(smem + G::misc + 32));
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem_base = *tslot;
  PieceQueue queue(reinterpret_cast<Piece*>(smem + G::pieces), &bars[G::queue], stop);
  bool ok = true;
  uint32_t asked_k = 0, asked_v = 0;   // steps whose keys, and values, this CTA has asked for (loading warp)

  if (warp == G::load_warp) {
    // =========================== schedule and copies =============================
    // The warp hands a piece to the others, then asks for its cells, kAtOnce steps at a time: a lane for a run of 16 keys, or of their values,
    // and its scale.  (Behind a wait that gave up nothing more is asked for: a unit that is not free may be waiting for its boxes.)
    constexpr int kRuns = G::at_once * (kKeys / 16);
    const int run = lane % kRuns, kind = lane / kRuns, mine = run / 4;   // kind 0: keys, 1: values; the lane's step of those
    const uint32_t k_ring = tc::smem_u32(smem), v_ring = k_ring + G::v, scales = k_ring + G::scales;
    TallWalk8<RP> walk = plan;
    Piece it;
    bool going = true;
    while (going && walk.next(p, &it)) {
      it.edges = edges8(p, it);
      if (kv16_held<kHeld>(p, kHeldSchedule, queue.i)) piece_wait<kHeld>(&bars[G::drained], 0, abort_flag);   // (that nothing arrives on here)
      if (lane < G::nan_words) reinterpret_cast<uint32_t*>(smem + G::nan)[queue.i % G::nan_pieces * G::nan_words + lane] = 0u;
      __syncwarp();   // (ahead of the entry that one lane makes known)
      going = queue.put(it, abort_flag);
      if (!going) break;
      const int n = steps8(it);
      const int32_t* const table = p.block_table + (int64_t)it.r * p.block_table_row_stride;
      auto look_up = [&](int j, int* slot) -> int {   // block of the lane's run: -1, there is none; -2, no row sees it
        const int pos = it.key0 + j * kKeys + run * 16;
        if (pos + 16 <= it.lo || pos >= it.hi) return -2;
        const int page = p.block_shift >= 0 ? pos >> p.block_shift : (int)((uint32_t)pos / (uint32_t)p.block_size);
        *slot = pos - page * p.block_size;
        const int blk = __ldg(table + page);
        return (uint32_t)blk < (uint32_t)p.num_blocks ? blk : -1;
      };
      int slot = 0, next_slot = 0, next_blk = look_up(0, &next_slot);
      auto free_units = [&](int first, int units, uint32_t asked_for, int here) {
        for (int i = 0; i < here; ++i) {
          const uint32_t u = asked_for + i;
          if (u >= (uint32_t)units) ok &= piece_wait<kHeld>(&bars[first + u % units], ((u / units) - 1) & 1, abort_flag);
        }
        ok = __all_sync(0xffffffffu, ok);
        return ok;
      };
#pragma unroll 1
      for (int j = 0; j < n; j += G::at_once) {
        const int blk = next_blk, here = min(G::at_once, n - j);
        slot = next_slot;
        if (j + G::at_once < n) next_blk = look_up(j + G::at_once, &next_slot);
        auto ask = [&](const CUtensorMap& map, uint32_t to, uint64_t* full) {   // the lane's run
          to += (run & 3) * 16 * G::dims;
          if (blk >= 0) {
            mbar_arrive_expect_tx(full, 16 * HD);
#pragma unroll
            for (int part = 0; part < G::parts; ++part) tma_load_4d(to + part * (kKeys * 128), &map, part * 128, it.kvh, slot, blk, full);
          } else {
            if (blk == -1) {   // keys and values of zero
#pragma unroll 1
              for (int i = 0; i < HD; ++i)   // 16 rows of HD bytes, 16 at a time
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(to + i * 16 / (16 * G::dims) * (kKeys * 128) + i * 16 % (16 * G::dims)), "r"(0) : "memory");
              tc::fence_async_smem();
            }
            mbar_arrive(full);
          }
        };
        const bool live = kind < 2 && mine < here;
        const uint32_t step = asked_v + mine, ku = step % G::k_units, vu = step % G::v_units, su = step % G::scale_steps;
        if (kv16_held<kHeld>(p, kHeldCopies, asked_k)) ok = false;
        if (!free_units(G::k_empty, G::k_units, asked_k, here)) break;
        if (live) {
          const float* const base = kind == 0 ? p.k_scale : p.v_scale;
          copy4(scales + su * 32 + kind * 16 + (run & 3) * 4, blk >= 0 ? base + scale_at(p, it.kvh, blk, slot) : base, blk >= 0);
          copies_arrive(&bars[G::k_full + ku]);
          if (kind == 0) ask(k_map, k_ring + ku * G::raw, &bars[G::k_full + ku]);
        }
        asked_k += here;
        __syncwarp();
        if (!free_units(G::v_empty, G::v_units, asked_v, here)) break;
        if (live && kind == 1) ask(v_map, v_ring + vu * G::raw, &bars[G::v_full + vu]);
        asked_v += here;
        __syncwarp();
      }
      if (!ok) break;
    }
    if (going) {
      it.tiles = 0;
      queue.put(it, abort_flag);
    }
    copies_wait_all();
  } else if (warp >= G::widen_warp && warp < G::load_warp) {
    // =========================== V ===============================================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::widen_regs));
    constexpr int kCols = G::dims / 16, kPer = G::parts * kKeys * kCols / 128;   // 16-byte pieces of a thread
    const int thread = tid - G::widen_warp * 32;
    uint32_t step = 0, piece = 0;
    Piece it;
    while (queue.get(&it, abort_flag)) {
      const int n = steps8(it);
      const Edges8 edges(it, n);
      uint32_t* const noted = reinterpret_cast<uint32_t*>(smem + G::nan) + piece++ % G::nan_pieces * G::nan_words;
#pragma unroll 1
      for (int j = 0; j < n; ++j, ++step) {
        const uint32_t vu = step % G::v_units, wu = step % G::w_units;
        ok &= piece_wait<kHeld>(&bars[G::v_full + vu], (step / G::v_units) & 1, abort_flag);
        if (step >= G::w_units) ok &= piece_wait<kHeld>(&bars[G::w_empty + wu], ((step / G::w_units) - 1) & 1, abort_flag);
        const uint8_t* const raw = smem + G::v + vu * G::raw;
        uint8_t* const wide = smem + G::w + wu * G::wide;
        const int key0 = it.key0 + j * kKeys;
        constexpr int kBatch = kPer < 4 ? kPer : 2;
#pragma unroll
        for (int i0 = 0; i0 < kPer; i0 += kBatch) {
        uint4 cells[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int x = (i0 + i) * 128 + thread, part = x / (kKeys * kCols), key = x / kCols % kKeys, c = x % kCols;
          cells[i] = *reinterpret_cast<const uint4*>(raw + part * (kKeys * 128) + key * G::dims + ((HD == 64 ? c ^ ((key >> 1) & 3) : c ^ (key & 7)) << 4));
          if (key0 + key < it.lo || key0 + key >= it.hi) cells[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        if (edges.has(j)) {
          uint32_t nan = 0;
#pragma unroll
          for (int i = 0; i < kBatch; ++i) nan |= nan_cells(cells[i].x) | nan_cells(cells[i].y) | nan_cells(cells[i].z) | nan_cells(cells[i].w);
          if (__builtin_expect(nan != 0, 0)) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
              const int key = ((i0 + i) * 128 + thread) / kCols % kKeys;
              if ((take_nan(cells[i].x) | take_nan(cells[i].y) | take_nan(cells[i].z) | take_nan(cells[i].w)) == 0) continue;
              atomicOr(noted + 1 + 2 * edges.note_of(j) + (key >> 5), 1u << (key & 31));
              *noted = 1u;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int x = (i0 + i) * 128 + thread, part = x / (kKeys * kCols), key = x / kCols % kKeys, c = x % kCols;
          const uint4 v = cells[i];
          const uint2 a = widen4(v.x), b = widen4(v.y), d = widen4(v.z), e = widen4(v.w);
          // dims 16 c .. of slab c / 4: two pieces of 8, in an order that leaves lanes of two slabs on different banks
          uint8_t* const to = wide + (part * 2 + (c >> 2)) * (kKeys * 128) + key * 128;
          const int first = (c >> 2) & 1;
          const uint4 lo = make_uint4(a.x, a.y, b.x, b.y), hi = make_uint4(d.x, d.y, e.x, e.y);
          *reinterpret_cast<uint4*>(to + (((2 * (c & 3) + first) ^ (key & 7)) << 4)) = first ? hi : lo;
          *reinterpret_cast<uint4*>(to + (((2 * (c & 3) + (first ^ 1)) ^ (key & 7)) << 4)) = first ? lo : hi;
        }
        }
        tc::fence_async_smem();   // (W to the tensor core; the raw rows' reads in front of the boxes that come there next)
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars[G::w_full + wu]);
          mbar_arrive(&bars[G::v_empty + vu]);
        }
      }
    }
  } else if (warp >= G::mma_warp) {
    // =========================== MMAs ============================================
    const int rt = warp - G::mma_warp;
    constexpr uint32_t qk_desc = instr_desc_e4m3(128, kKeys, 0, 0);
    constexpr uint32_t pv_desc = tc::instr_desc(128, G::dims, tc::kFmtF16, tc::kFmtF16, 0, 1);
    const uint64_t q_desc = tc::smem_desc(tc::smem_u32(smem + G::q) + rt * G::q_tile, 2048, 128);
    const uint64_t k_desc = raw_desc<HD>(tc::smem_u32(smem));
    const uint64_t w_desc = swizzled_desc(tc::smem_u32(smem + G::w), kKeys * 128, 1024);
    const uint32_t o_tmem = tmem_base + G::o_col + rt * HD, s_tmem = tmem_base + G::s_col + 2 * rt * kKeys;
    uint32_t k_slot = 0, k_phase = 0, w_slot = 0, w_phase = 0;   // of the next step
    auto next_k = [&] {
      if (++k_slot == G::k_units) {
        k_slot = 0;
        k_phase ^= 1;
      }
    };
    auto next_w = [&] {
      if (++w_slot == G::w_units) {
        w_slot = 0;
        w_phase ^= 1;
      }
    };
    uint32_t s_qk = 0, s_pv = 0, pieces = 0;   // steps so far, pieces with live rows
    auto qk = [&](bool first) {
      const uint32_t b = s_qk & 1;
      if (first) ok &= piece_wait<kHeld>(&bars[G::q_full + rt], (pieces - 1) & 1, abort_flag);
      ok &= piece_wait<kHeld>(&bars[G::k_full + k_slot], k_phase, abort_flag);
      if (s_qk > 1) ok &= piece_wait<kHeld>(&bars[G::pv_done + 2 * rt + b], ((s_qk >> 1) - 1) & 1, abort_flag);   // (P of the step before last has been read)
      if (!ok) return;
      tc::fence_after_sync();
#pragma unroll
      for (int part = 0; part < G::parts; ++part) {
#pragma unroll
        for (int kk = 0; kk < G::dims / 32; ++kk) {
          const uint32_t klo = (uint32_t)k_desc + k_slot * (G::raw >> 4) + part * ((kKeys * 128) >> 4) + kk * 2;
#pragma unroll
          for (int g = 0; g < G::q_digits; ++g) {
            const uint32_t qlo = (uint32_t)q_desc + g * (G::q_digit >> 4) + (part * (G::dims / 16) + kk * 2) * (2048 >> 4);
            if (part == 0 && kk == 0 && g == 0) mma_e4m3_words<false>(s_tmem + b * kKeys, qlo, (uint32_t)(q_desc >> 32), klo, (uint32_t)(k_desc >> 32), qk_desc);
            else mma_e4m3_words<true>(s_tmem + b * kKeys, qlo, (uint32_t)(q_desc >> 32), klo, (uint32_t)(k_desc >> 32), qk_desc);
          }
        }
      }
      tc::mma_commit(&bars[G::k_empty + k_slot]);
      tc::mma_commit(&bars[G::s_ready + 2 * rt + b]);
      mbar_arrive(&bars[G::s_ready + 2 * rt + b]);
      next_k();
      ++s_qk;
    };
    auto pv = [&](bool first) {
      const uint32_t b = s_pv & 1;
      ok &= piece_wait<kHeld>(&bars[G::w_full + w_slot], w_phase, abort_flag);
      ok &= piece_wait<kHeld>(&bars[G::p_ready + 2 * rt + b], (s_pv >> 1) & 1, abort_flag);
      if (!ok) return;
      tc::fence_after_sync();
#pragma unroll
      for (int part = 0; part < G::parts; ++part) {
        const uint32_t wlo = (uint32_t)w_desc + w_slot * (G::wide >> 4) + part * ((2 * kKeys * 128) >> 4);
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
          mma_ts_words(o_tmem + part * 128, s_tmem + b * kKeys + kk * 8, wlo + kk * (2048 >> 4), (uint32_t)(w_desc >> 32), pv_desc, !first || kk > 0);
      }
      tc::mma_commit(&bars[G::w_empty + w_slot]);
      tc::mma_commit(&bars[G::pv_done + 2 * rt + b]);
      next_w();
      ++s_pv;
    };
    Piece it;
    const bool leader = elect_one();   // (one lane takes all steps of a piece: the others would only have to be waited for)
    while (queue.get(&it, abort_flag)) {
      if (kv16_held<kHeld>(p, kHeldMma, s_qk)) ok = false;
      if (!leader || !ok) continue;
      const int n = steps8(it);
      if (it.rows <= rt * 128) {   // no rows: free the units as if they had been read
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
          ok &= piece_wait<kHeld>(&bars[G::k_full + k_slot], k_phase, abort_flag);
          ok &= piece_wait<kHeld>(&bars[G::w_full + w_slot], w_phase, abort_flag);
          if (!ok) break;
          mbar_arrive(&bars[G::k_empty + k_slot]);
          mbar_arrive(&bars[G::w_empty + w_slot]);
          next_k();
          next_w();
        }
        continue;
      }
      ++pieces;
      // QK of a step ahead of PV of the one before: the softmax finds the next S when it is done with one
#pragma unroll 1
      for (int j = 0; j <= n && ok; ++j) {
        if (j < n) qk(j == 0);
        if (j > 0 && ok) pv(j == 1);
      }
    }
  } else {
    // =========================== softmax =========================================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::softmax_regs));
    const int rt = warp >> 2;
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_tmem = tmem_base + G::o_col + rt * HD + lane_addr;
    const int row = tid;   // of the CTA's rows
    uint32_t count = 0;    // live steps so far
    uint32_t step = 0;     // steps so far (of all pieces)
    auto rt_sync = [&] { named_barrier(1 + rt, 128); };
    uint8_t* const raw_q = smem + (HD == 64 ? G::raw_q : G::q + rt * G::q_tile);
    const uint32_t raw_rows = tc::smem_u32(raw_q) + (row & 96) * (2 * HD);   // of the warp
    uint32_t piece = 0;    // pieces so far
    bool copied = false;   // the piece's query rows are on their way
    zero_requests<HD, RP, 128 * G::rts>(p);
    {
      Piece it;
      while (queue.get(&it, abort_flag)) {
        const int n_steps = steps8(it);
        const uint32_t* const noted = reinterpret_cast<const uint32_t*>(smem + G::nan) + piece++ % G::nan_pieces * G::nan_words;
        if (it.rows <= rt * 128) {
          step += n_steps;
          copied = false;
          continue;
        }
        const int kvh = it.kvh;
        const bool padding = (row & ~31) >= it.rows;   // (of the whole warp)
        int token, head;
        row_of(p, it.first_token, kvh, it.row0 + min(row, it.rows - 1), &token, &head);
        // (QK has read the last piece's digits: its last S has been waited for)
        float q_factor = 0.f;
        if (!padding) {
          if (!copied) copy_rows<HD>(p, it, row & ~31, raw_rows);
          copies_wait_all();
          __syncwarp();
          q_factor = stage_row<HD, kHalf>(p, raw_q + (row & 127) * (2 * HD), row, smem + G::q + rt * G::q_tile + (row & 127) * 16, rt_sync);
          tc::fence_async_smem();
        } else if constexpr (HD != 64) {
          rt_sync();
        }
        copied = false;
        mbar_arrive(&bars[G::q_full + rt]);
        const int own = it.pos0 + token - it.first_token;
        const int row_lo = kv8_low(p, own), row_hi = p.causal ? min(own + 1, it.hi) : it.hi;
        float ref = -INFINITY, l = 0.f;
        float unit = 0x1p-126f, inverse = 0x1p126f;   // U: the largest scale of values that the row has seen
        const bool not_finite = q_factor < 0.f;
#pragma unroll 1
        for (int t = 0; t < n_steps; ++t, ++count, ++step) {
          const uint32_t b = 2 * rt + (count & 1), use = count >> 1, su = step % G::scale_steps;
          const uint32_t s_tmem = tmem_base + G::s_col + b * kKeys + lane_addr;
          ok &= piece_wait<kHeld>(&bars[G::s_ready + b], use & 1, abort_flag);
          if (padding) {   // (the order of the waits is kept, nothing is computed)
            mbar_arrive(&bars[G::p_ready + b]);
            continue;
          }
          tc::fence_after_sync();
          uint32_t r[64];
          tc::tmem_ld32(s_tmem, r);
          tc::tmem_ld32(s_tmem + 32, r + 32);
          const float4 ks = *reinterpret_cast<const float4*>(smem + G::scales + su * 32);
          const float4 vs = *reinterpret_cast<const float4*>(smem + G::scales + su * 32 + 16);
          float value_scale[4] = {vs.x, vs.y, vs.z, vs.w};
          float factor[4] = {score_factor(ks.x, q_factor), score_factor(ks.y, q_factor), score_factor(ks.z, q_factor), score_factor(ks.w, q_factor)};
          tc::tmem_ld_wait<64>(r);
          const int key0 = it.key0 + t * kKeys;
          if (key0 < row_lo || key0 + kKeys > row_hi) {
            // bit n: key n is seen
            const int lo = min(max(row_lo - key0, 0), 64), hi = min(max(row_hi - key0, 0), 64);
            const uint64_t from = lo < 64 ? ~0ull << lo : 0ull, upto = hi < 64 ? (1ull << hi) - 1 : ~0ull, seen = from & upto;
#pragma unroll
            for (int n = 0; n < 64; ++n)
              r[n] = (uint32_t)(n < 32 ? seen : seen >> 32) >> (n & 31) & 1u ? r[n] : 0xff800000u;  // -inf
#pragma unroll
            for (int g = 0; g < 4; ++g) {   // (scales that the row does not see)
              factor[g] = (uint32_t)(seen >> 16 * g) & 0xffffu ? factor[g] : 1.f;
              value_scale[g] = (uint32_t)(seen >> 16 * g) & 0xffffu ? value_scale[g] : 0.f;
            }
          }
          const float top_scale = max3(fmaxf(value_scale[0], value_scale[1]), value_scale[2], value_scale[3]);
          float total;
          // (One copy of the code for a step's first look and its second: the instruction caches are small.)
          bool move = t == 0;
#pragma unroll 1
          for (bool again = false;; again = true) {
            bool outgrown = true;
            if (!move) {
              const float weight[4] = {value_scale[0] * inverse, value_scale[1] * inverse, value_scale[2] * inverse, value_scale[3] * inverse};
              total = exponentials8(r, factor, ref == -INFINITY ? 0.f : -ref, weight, s_tmem);
              if (again) break;
              outgrown = !(total <= kMostSum) || ref == -INFINITY;
              if (!__any_sync(0xffffffffu, outgrown || top_scale > unit)) break;
            }
            move = false;
            float mx[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              mx[g] = -INFINITY;
#pragma unroll
              for (int n = 0; n < 16; n += 2) mx[g] = max3(mx[g], __uint_as_float(r[16 * g + n]), __uint_as_float(r[16 * g + n + 1]));
              mx[g] *= factor[g];
            }
            const float to = outgrown ? fmaxf(ref, max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) - kGainP) : ref;
            const float to_unit = fmaxf(unit, top_scale);
            const float alpha = to == -INFINITY ? 1.f : ex2f(ref - to);
            asm("rcp.approx.f32 %0, %1;" : "=f"(inverse) : "f"(to_unit));
            const float both = alpha * (unit * inverse);
            ref = to;
            l *= alpha;
            unit = to_unit;
            if (t > 0) {   // (PV of what P holds already is complete first)
              ok &= piece_wait<kHeld>(&bars[G::pv_done + (b ^ 1)], ((count - 1) >> 1) & 1, abort_flag);
              tc::fence_after_sync();
#pragma unroll 1
              for (int d = 0; d < HD / 16; ++d) {
                uint32_t o[16];
                tc::tmem_ld16(o_tmem + d * 16, o);
                tc::tmem_ld_wait<16>(o);
#pragma unroll
                for (int n = 0; n < 16; ++n) o[n] = __float_as_uint(__uint_as_float(o[n]) * both);
                tc::tmem_st16(o_tmem + d * 16, o);
              }
              tc::tmem_st_wait();
            }
          }
          l += total;
          tc::tmem_st_wait();
          tc::fence_before_sync();
          mbar_arrive(&bars[G::p_ready + b]);
        }
        // (QK has read the digits: the next piece's rows can come in the meantime)
        Piece next;
        if (queue.peek(&next)) {
          copy_rows<HD>(p, next, row & ~31, raw_rows);
          copied = true;
        }
        // ---- the piece's rows ----
        ok &= piece_wait<kHeld>(&bars[G::pv_done + 2 * rt + ((count - 1) & 1)], ((count - 1) >> 1) & 1, abort_flag);
        tc::fence_after_sync();
        if (not_finite && max(row_lo, it.key0) < min(row_hi, it.key0 + it.tiles * kTile)) l = NAN;   // (a row that sees no key is zero)
        const bool whole = it.begins && it.ends, live = row < it.rows;
        uint8_t* const out = p.out + (int64_t)token * p.out_stride_token + (int64_t)head * p.out_stride_head;
        float* const lse = p.lse != nullptr ? p.lse + (int64_t)token * p.num_q_heads + head : nullptr;
        auto write16 = [&](const float* o, int d0) {   // 16 columns of the row
          uint32_t w[8];
#pragma unroll
          for (int n = 0; n < 8; ++n) w[n] = pack16<kHalf>(o[2 * n], o[2 * n + 1]);
          uint8_t* const to = out + d0 * 2;
          if (p.out_wide) {
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                         "r"(w[5]), "r"(w[6]), "r"(w[7])
                         : "memory");
          } else {
            *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4*>(to + 16) = make_uint4(w[4], w[5], w[6], w[7]);
          }
        };
        if (!padding) {
          const float factor = whole ? (l == 0.f ? 0.f : unit / l) : unit;
          float* const slot = tall8_slot<HD, kHalf>(p, (int)blockIdx.x, it.begins) + row;
          const bool nan = it.edges != 0 && *noted != 0u;   // (the same in all threads)
          uint32_t columns[HD / 16];
          if (nan) nan_columns<HD>(p, it, noted, row_lo, row_hi, columns);
#pragma unroll 1
          for (int c = 0; c < HD / 16; ++c) {
            uint32_t r[16];
            tc::tmem_ld16(o_tmem + c * 16, r);
            tc::tmem_ld_wait<16>(r);
            if (nan) {
#pragma unroll
              for (int n = 0; n < 16; ++n) r[n] = columns[c] >> n & 1u ? 0x7fffffffu : r[n];
            }
            float o[16];
#pragma unroll
            for (int n = 0; n < 16; ++n) o[n] = __uint_as_float(r[n]) * factor;
            if (whole) {
              if (live) {
                write16(o, c * 16);
              }
            } else {
#pragma unroll
              for (int n = 0; n < 16; ++n) slot[(c * 16 + n) * RP] = o[n];
            }
          }
          if (whole) {
            if (live && lse != nullptr) *lse = l == 0.f ? -INFINITY : ((ref == -INFINITY ? 0.f : ref) + log2f(l)) * kLn2;
          } else {
            slot[HD * RP] = ref;
            slot[(HD + 1) * RP] = l;
          }
        }
        tc::fence_before_sync();
        if (!whole) {
          // (a row tile's pieces are merged by the row tile's own threads: a counter each)
          const int c0 = it.first_cta, c1 = it.last_cta;
          rt_sync();
          int* const counter = reinterpret_cast<int*>(p.workspace) + G::rts * c0 + rt;
          if ((tid & 127) == 0) {
            arrival[rt] = arrive_at(counter) == c1 - c0;
            if (arrival[rt]) *counter = 0;   // (for the next call)
          }
          rt_sync();
          if (arrival[rt] && !padding) {
            auto slot = [&](int c) { return tall8_slot<HD, kHalf>(p, c, c == c0) + row; };
            float top = -INFINITY, sum = 0.f;
            // (the loads of two pieces are in flight together; one that there is not counts nothing)
#pragma unroll 1
            for (int c = c0; c <= c1; c += 2) {
              const bool b = c < c1;
              const float* s = slot(c) + HD * RP;
              const float* t = slot(b ? c + 1 : c) + HD * RP;
              const float ra = __ldcg(s), la = __ldcg(s + RP), rb = b ? __ldcg(t) : -INFINITY, lb = __ldcg(t + RP);
              const float to = max3(top, ra, rb), use = to == -INFINITY ? 0.f : to;
              sum = fmaf(sum, ex2f(top - use), ex2f(ra - use) * la);
              sum += b ? ex2f(rb - use) * lb : 0.f;
              top = to;
            }
            const float use = top == -INFINITY ? 0.f : top, inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll 1
            for (int c = 0; c < HD / 16; ++c) {
              float o[16];
#pragma unroll
              for (int n = 0; n < 16; ++n) o[n] = 0.f;
#pragma unroll 1
              for (int cta = c0; cta <= c1; cta += 2) {
                const bool b = cta < c1;
                const float* s = slot(cta);
                const float* t = slot(b ? cta + 1 : cta);
                const float wa = __ldcg(s + HD * RP), wb = __ldcg(t + HD * RP);
                float v[16], u[16];
#pragma unroll
                for (int n = 0; n < 16; ++n) {
                  v[n] = __ldcg(s + (c * 16 + n) * RP);
                  u[n] = __ldcg(t + (c * 16 + n) * RP);
                }
                const float fa = ex2f(wa - use) * inv, fb = b ? ex2f(wb - use) * inv : 0.f;
#pragma unroll
                for (int n = 0; n < 16; ++n) {
                  o[n] = fmaf(fa, v[n], o[n]);
                  if (b) o[n] = fmaf(fb, u[n], o[n]);
                }
              }
              if (live) write16(o, c * 16);
            }
            if (live && lse != nullptr) *lse = sum == 0.f ? -INFINITY : (use + log2f(sum)) * kLn2;
          }
          rt_sync();   // (the arrival has been read)
        }
      }
      copies_wait_all();
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (*abort_flag) {   // (the same in all threads) what is in flight comes to its end first: MMAs, and boxes
    if (warp >= G::mma_warp && elect_one()) {
      uint64_t* const drained = &bars[G::drained + warp - G::mma_warp];
      tc::mma_commit(drained);
      kv16_drain(drained, 0);
    }
    if (warp == G::load_warp) {
      for (uint32_t u = asked_k > G::k_units ? asked_k - G::k_units : 0; u < asked_k; ++u) kv16_drain(&bars[G::k_full + u % G::k_units], (u / G::k_units) & 1);
      for (uint32_t u = asked_v > G::v_units ? asked_v - G::v_units : 0; u < asked_v; ++u) kv16_drain(&bars[G::v_full + u % G::v_units], (u / G::v_units) & 1);
    }
    if (tid == 0) atomicOr(&g_kv8_tall_status, 64u);
    __syncthreads();
  }
  if (warp == G::mma_warp) tc::tmem_dealloc(tmem_base, G::tmem);
}

template <int HD, bool kHalf, bool kHeld = false>
cudaError_t launch_one(const Kv8Params& p, const CUtensorMap& k_map, const CUtensorMap& v_map, cudaStream_t stream) {
  using G = Tall8<HD, kHalf>;
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    cudaFuncAttributes attr;
    err = cudaFuncGetAttributes(&attr, kv8_tall_kernel<HD, kHalf, kHeld>);
    if (err == cudaSuccess && attr.numRegs < G::start_regs) err = cudaErrorInvalidConfiguration;   // (setmaxnreg would wait without end)
    if (err == cudaSuccess) err = cudaFuncSetAttribute(kv8_tall_kernel<HD, kHalf, kHeld>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::total);
    if (err != cudaSuccess) return err;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int sms = sm_count();
  // (a counter for every CTA's row tiles)
  if (sms <= 0 || sms * G::ctas * G::rts * 4 > kCounterBytes) return cudaErrorInvalidDevice;
  Kv8Params q = p;
  q.out_wide = reinterpret_cast<uintptr_t>(p.out) % 32 == 0 && p.out_stride_token % 32 == 0 && p.out_stride_head % 32 == 0;
  return pdl_launch(kv8_tall_kernel<HD, kHalf, kHeld>, dim3((unsigned)(sms * G::ctas)), dim3(G::threads), G::total, stream, q, k_map, v_map);
}
template <int HD>
cudaError_t launch_type(const Kv8Params& p, const CUtensorMap& k_map, const CUtensorMap& v_map, cudaStream_t stream) {
  return p.dtype == PTH_ATTN_F16 ? launch_one<HD, true>(p, k_map, v_map, stream) : launch_one<HD, false>(p, k_map, v_map, stream);
}

}  // namespace

// Counters, and two partial row tiles per CTA.
int64_t kv8_tall_workspace_bytes(int head_size, int num_sms) {
  const int64_t rows = head_size == 256 ? 128 : 256;   // of an SM's CTAs together
  return kCounterBytes + (int64_t)num_sms * 2 * rows * (head_size + 2) * 4;
}

cudaError_t launch_kv8_tall_held(const Kv8Params& p, cudaStream_t stream) {
  CUtensorMap k_map{}, v_map{};
  if (!cell_box_map(p, p.k, 16, &k_map) || !cell_box_map(p, p.v, 16, &v_map)) return cudaErrorInvalidValue;
  return launch_one<128, false, true>(p, k_map, v_map, stream);
}
cudaError_t launch_kv8_tall(const Kv8Params& p, cudaStream_t stream, bool* taken) {
  CUtensorMap k_map{}, v_map{};
  *taken = cell_box_map(p, p.k, 16, &k_map) && cell_box_map(p, p.v, 16, &v_map);
  if (!*taken) return cudaSuccess;
  switch (p.head_size) {
    case 64:
      return launch_type<64>(p, k_map, v_map, stream);
    case 128:
      return launch_type<128>(p, k_map, v_map, stream);
    default:
      return launch_type<256>(p, k_map, v_map, stream);
  }
}

// Reads and clears this kernel's status word (device must be idle).
cudaError_t read_kv8_tall_status(unsigned int* v) {
  unsigned int zero = 0;
  cudaError_t err = cudaMemcpyFromSymbol(v, g_kv8_tall_status, sizeof(*v));
  if (err != cudaSuccess) return err;
  return cudaMemcpyToSymbol(g_kv8_tall_status, &zero, sizeof(zero));
}

}  // namespace pthb200
