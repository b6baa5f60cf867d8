// Attention over the 16-bit paged cache for requests of many query rows: cross attention of prompts.
//
// Orientation: query rows on the MMA's M dimension, a thread per row in the softmax:
//   S[row, key] = sum_d Q[row, d] K[key, d]       A = Q, B = K as it lies in the cache (K-major), accumulator in TMEM
//   O[row, d]  += sum_key P[row, key] V[key, d]   A = P in TMEM over S, B = V as it lies in the cache (MN-major)
// An SM holds two row tiles of 128 rows, so that the tensor core and one's softmax have work while the other's waits: of one CTA at
// 128 dims, where every K and V tile then serves twice, of two CTAs at 64 dims, whose items may be different ones (a request's
// last rows seldom fill both).  At 256 dims O alone takes half of TMEM: one row tile.
//
// Softmax in one pass: ref is a running bound of a row's scores (log2 units), P = 2^(s - ref), l = sum P.  It is set kGain below the
// maximum of a row's first 64 keys.  Later ones need no maximum: the sum of 64 P, which the row sum takes anyway, says
// whether one of them has outgrown ref too far (kMostSum); then ref moves to their maximum, O and l are rescaled and the
// 64 are computed again.  P is rounded to the cache's type for the MMA (the error of the output is sqrt(2) times that
// of its own rounding), its sum is not.  (A probability below 2^-31 of the row's largest, 2^-102 in bf16, may be
// zero: an infinite value under it gives NaN.)  The steps are of 64 keys (128 at 256 dims) with two S buffers,
// so that a step's QK and the last one's PV run beside its softmax.
//
// What bounds it: a row tile's chain of a step.  Cycles per step of 64 keys at 128 dims, both row tiles at work: 1,380 for the
// exponentials of both (8 of the special function unit for a warp's 32, the conversions beside them), 80 for S to come from TMEM, 160
// for P to go there, some 300 for the two barriers: 2,000 in all, beside 1,350 of MMAs (eight of QK over 64 keys take 400 instead
// of 256: both operands come from shared memory).  Without the exponentials a launch takes 15 % less, with an eighth of QK's MMAs and a
// quarter of PV's 8 %.
// Measured, bf16, behind a flush of L2: 4 x 2,048 tokens over 8,192 states, 32 heads of 8, 128 dims 950 us, 1,157 TFLOP/s (1,084 us, 1,014
// TFLOP/s, in calls behind one another for seconds, at the board's power limit), in fp16 975 us; at 256 dims 2,840 us, 774, and 8 x
// 1,000 over 4,000 1,477 us, 710; 16 heads of 16, 64 dims 510 us, 539.  64 x 16 over 4,000 at 128 dims, one row tile of two, 207 us,
// 5.2 TB/s; 16 x 4-448 over 64-1,500, 16 heads of 16, 64 dims 47 us, of which the start is 3, an item's first maximum and rows' way
// out 3 each, the last merge 4.
// Taken back: steps of 128 keys with one S buffer, a row tile waiting for its MMAs, 1,241; an eighth of the exponentials as a
// polynomial on the FMA pipe 981 against 977, a quarter 1,045; the row tiles' exponentials in turn, or half a step apart (983 against
// 960); P rounded with integer instructions 1,007 against 958; MMAs predicated lane by lane in a warp that stays together 958 against 946.
//
// A warp per row tile issues its MMAs, so neither row tile waits for the other, and nothing relies on the order in which MMAs on
// different accumulators run.
//
// Copies: tiles that are visible as a whole come as boxes (tiled TMA, 64 dims of up to 32 slots of a page) where pages are a
// multiple of 8 slots, others as 16-byte copies, which zero what is not visible.  (All by 16-byte copies: 1,300 cycles a
// unit of 32 KB.  Copies against boxes, us: 4 x 2,048 tokens over 8,192 states 1,049 / 961, 32 x 200 over 8,000 1,035 / 949, 8 x 1,000 over
// 4,000 at 256 dims 2,026 / 1,677, 64 x 256 over 2,000 at 64 dims 303 / 298.)
//
// Schedule: items (row tile, KV head, request), in the order request, head, row tile, so that neighbouring items read the same keys.
// While the keys of a launch fit in the L2 cache, the sequence of all their KV tiles is cut into equal runs, one per CTA (an item
// counts kItemTiles more, which stand in front of its tiles).
// Otherwise all but the last one or two items per CTA go out in waves, CTA c taking items c, c + CTAs, ...: the CTAs then work
// on the same few heads of one request at a time.  The tiles of the rest make up for unequal waves.  Equal runs against waves, us:
// above the bound 4 x 2,048 tokens over 8,192 states 981 / 944, 16 x 10-512 over 64-8,000 314 / 303, 64 x 64 over 64-4,000 at 64 dims
// 166 / 146, 8 x 1,000 over 4,000 at 256 dims 1,641 / 1,487 (100 x 1-100 over 64-1,000 134 / 152); below it 8 x 1,200 over 1,000 at 64
// dims 111 / 115, 16 x 4-448 over 64-1,500 at 128 dims 81 / 83 (30 x 400 over 200 122 / 118).
#include "kv16_sched.cuh"
#include "page_copy.cuh"
#include "pdl.cuh"
#include "umma_rows.cuh"

namespace pthb200 {

__device__ unsigned int g_kv16_tall_status = 0;

namespace {

template <bool kHalf>
constexpr float kMostSum = kHalf ? 0x1p15f : 0x1p-16f;   // of 64 P
constexpr int kLoadWarps = 4;
// KV tiles that an item counts besides its own: its queries, its first maximum and its rows' way out.  With 0, 1, 2, 3, us:
//   16 x 4-448 tokens over 64-1,500 states, 16 heads of 16, 64 dims: 64, 51, 53, 53;  32 of 8, 128 dims: 127, 88, 81, 83;
//   32 of 8, 256 dims: 193, 172, 171, 181;  100 x 1-100 over 64-1,000, 32 of 8, 128 dims: 161, 144, 154, 154.
constexpr int kItemTiles = 2;
constexpr int kPlanReqs = 4096;        // requests up to which a launch may go out in waves
constexpr int kTallSms = 160;
constexpr long long kL2Keys = 48 << 20;   // bytes of keys and values that a launch may spread its CTAs over

template <int HD>
struct Tall {
  static constexpr int rts = HD == 128 ? 2 : 1;      // row tiles of 128 rows
  static constexpr int ctas = HD == 64 ? 2 : 1;      // per SM
  static constexpr int rows = 128 * rts;
  static constexpr int keys = HD == 256 ? 128 : 64;  // of a step, one of the two S buffers of a row tile
  static constexpr int steps = kTile / keys;         // of a KV tile
  static constexpr int halves = keys / 64;           // of a step: P is handed over 64 keys at a time
  static constexpr int dims = HD < 128 ? HD : 128;   // of a unit
  static constexpr int parts = HD / dims;
  static constexpr int unit = kTile * dims * 2;
  static constexpr int qtile = 128 * HD * 2;         // Q of a row tile: slabs of 64 dims, 128 rows of 128 bytes each
  static constexpr int units = 5;
  static constexpr int softmax_warps = 4 * rts;
  static constexpr int load_warp = softmax_warps, mma_warp = load_warp + kLoadWarps, schedule_warp = mma_warp + rts;   // (an MMA warp per row tile)
  static constexpr int threads = (schedule_warp + 1) * 32;
  // Registers that a thread starts with, which setmaxnreg moves from the copies to the softmax.
  static constexpr int start_regs = HD == 256 ? 168 : HD == 128 ? 128 : 96;
  static constexpr int copy_regs = HD == 256 ? 96 : 64, softmax_regs = HD == 256 ? 232 : HD == 128 ? 160 : 128;
  static_assert(softmax_warps * softmax_regs + kLoadWarps * copy_regs <= (softmax_warps + kLoadWarps) * start_regs, "a split that the launch holds");
  static constexpr int s_col = 0, o_col = 2 * rts * keys;   // TMEM columns: S(rt, b) at (2 rt + b) keys, O(rt) at o_col + rt HD
  static constexpr int tmem = HD == 64 ? 256 : 512;
  static_assert(o_col + rts * HD <= tmem, "accumulators");
  // shared memory, behind the first 1,024-byte boundary
  static constexpr int most_ctas = kTallSms * ctas;
  static constexpr int q = units * unit;
  static constexpr int bars = q + rts * qtile;
  static constexpr int n_bars = 2 * units + 2 * rts + 20 + 2 * kQueue + rts;
  static constexpr int pieces = bars + n_bars * 8;   // PieceQueue's entries
  static constexpr int misc = pieces + kQueue * 64;
  static constexpr int bounds = misc + 32;           // the plan's, and its scratch in front
  static constexpr int total = bounds + (most_ctas + 1) * 8 + 1024;
  static_assert(kPlanReqs * 16 + 16 <= units * unit + rts * qtile, "the plan's arrays lie where keys and queries come later");
  static_assert(total <= (ctas == 2 ? 115712 : 232448), "shared memory");
};
template <int HD>
struct TallBars {  // behind [units] full, [units] empty
  static constexpr int q_full = 0, q_empty = Tall<HD>::rts;
  static constexpr int s_ready = 2 * Tall<HD>::rts;  // [4] S buffer 2 rt + b
  static constexpr int p_ready = s_ready + 4;        // [4][2 halves]
  static constexpr int pv_half = p_ready + 8;        // [4] PV of the first of two halves
  static constexpr int pv_done = pv_half + 4;        // [4]
  static constexpr int queue = pv_done + 4;
  static constexpr int drained = queue + 2 * kQueue; // [rts]
};

// Tiled TMA load of one box of a rank-4 tensor map into shared memory.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(tc::smem_u32(bar))
      : "memory");
}

template <int HD>
__device__ __forceinline__ float* tall_slot(const Kv16Params& p, int cta, bool begins) {
  // [HD][rows] O, [rows] ref, [rows] l
  return reinterpret_cast<float*>(p.workspace + kCounterBytes) + (int64_t)(2 * cta + (begins ? 1 : 0)) * (Tall<HD>::rows * (HD + 2));
}

// P of 64 scores as pairs of 16-bit numbers, 2^(score scale + minus_ref); returns the sum of the unrounded ones.
template <bool kHalf>
__device__ __forceinline__ float exponentials(const uint32_t (&r)[64], float scale, float minus_ref, uint32_t (&pk)[32]) {
  const f32x2 scale2 = pair(scale, scale), ref2 = pair(minus_ref, minus_ref);
  f32x2 sum[2] = {0ull, 0ull};
#pragma unroll
  for (int n = 0; n < 32; ++n) {
    float x, y;
    unpair(fma2(pair(__uint_as_float(r[2 * n]), __uint_as_float(r[2 * n + 1])), scale2, ref2), x, y);
    x = ex2f(x);
    y = ex2f(y);
    sum[n & 1] = add2(sum[n & 1], pair(x, y));
    pk[n] = pack16<kHalf>(x, y);
  }
  return sum_pairs(sum);
}

// Steps of a piece: its keys from key0 on, as far as they are visible.
template <int kKeys>
__device__ __forceinline__ int piece_steps(const Piece& it) {
  return (min(it.tiles * kTile, it.hi - it.key0) + kKeys - 1) / kKeys;
}

// Length of an item in the sequence that is cut into runs: its KV tiles, and what its queries and its end take besides.
__device__ __forceinline__ int item_length(const ReqShape& s) { return s.tiles > 0 ? s.tiles + kItemTiles : 0; }

// Walk over the pieces of a CTA: its items of the waves, then its run of the rest.
template <int RP>
struct TallWalk {
  int wave, waves, ctas, item;    // item: of the current wave
  int r, first_item;              // request of the item, items in front of it
  long long at, end;              // the run, in the whole sequence
  int tail_r;
  long long tail_start;           // of request tail_r in the sequence
  long long base, work;           // where the runs begin in the sequence, and how long they are together
  int runs;                       // without waves: that they are cut into, equally
  const long long* bounds;        // with waves: where the CTAs' runs begin, behind `base`
  // CTA that has position x of the sequence in its run.
  __device__ __forceinline__ int owner(long long x) const {
    x -= base;
    if (waves == 0) return (int)(((x + 1) * runs - 1) / work);
    int lo = 0, hi = ctas - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (bounds[mid] <= x) lo = mid; else hi = mid - 1;
    }
    return lo;
  }
  __device__ __forceinline__ bool next(const Kv16Params& p, Piece* out) {
    ReqShape s;
    int it, tile, count;   // item of the request, tiles of it
    if (wave < waves) {
      s = req_shape<RP>(p, r);
      int n = s.tiles > 0 ? s.row_tiles * p.num_kv_heads : 0;
      while (item >= first_item + n) {
        first_item += n;
        ++r;
        s = req_shape<RP>(p, r);
        n = s.tiles > 0 ? s.row_tiles * p.num_kv_heads : 0;
      }
      it = item - first_item;
      tile = 0;
      count = s.tiles;
      out->r = r;
      out->first_cta = out->last_cta = 0;
      ++wave;
      item += ctas;
    } else {
      do {
        if (at >= end) return false;
        s = req_shape<RP>(p, tail_r);
        int n = item_length(s);
        while (at >= tail_start + (long long)n * s.row_tiles * p.num_kv_heads) {
          tail_start += (long long)n * s.row_tiles * p.num_kv_heads;
          ++tail_r;
          s = req_shape<RP>(p, tail_r);
          n = item_length(s);
        }
        const long long off = at - tail_start;
        it = (int)(off / n);
        const int a = (int)(off - (long long)it * n), b = (int)min((long long)n, a + (end - at));   // of the item's length
        tile = max(0, a - kItemTiles);
        count = b - kItemTiles - tile;
        out->first_cta = owner(at - a + kItemTiles);
        out->last_cta = owner(at - a + n - 1);
        at += b - a;
      } while (count <= 0);   // (no keys yet)
      out->r = tail_r;
    }
    const int kvh = (int)((uint32_t)it / (uint32_t)s.row_tiles), rt = it - kvh * s.row_tiles;
    out->kvh = kvh;
    out->row0 = rt * RP;
    out->rows = min(RP, s.tokens * p.group - rt * RP);
    out->first_token = s.first;
    out->key0 = (s.lo / kTile + tile) * kTile;
    out->tiles = count;
    out->lo = s.lo;
    out->hi = s.hi;
    out->begins = tile == 0;
    out->ends = tile + count == s.tiles;
    out->sparse = waves > 0;
    return true;
  }
};

// Who has which items (see the head of this file), worked out by all threads of every CTA.  arrays: room for 16 bytes a request;
// bounds [CTAs + 1].  The result is good in every thread.
template <int HD, int RP, int kThreads, int kMostCtas>
__device__ __forceinline__ TallWalk<RP> make_plan(const Kv16Params& p, uint8_t* arrays, long long* bounds) {
  constexpr int kWarps = kThreads / 32;
  static_assert(3 * kWarps <= kMostCtas, "scratch");
  long long* const scratch = bounds;
  const int R = p.num_reqs, C = (int)gridDim.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per = (R + kThreads - 1) / kThreads, r0 = min(R, tid * per), r1 = min(R, r0 + per);
  // items (0), their lengths (1), KV tiles of the requests' keys (2): in front of this thread's requests, and in all
  long long mine[3] = {0, 0, 0}, before[3], total[3] = {0, 0, 0};
#pragma unroll 1
  for (int r = r0; r < r1; ++r) {
    const ReqShape s = req_shape<RP>(p, r);
    const int n = s.tiles > 0 ? s.row_tiles * p.num_kv_heads : 0;
    mine[0] += n;
    mine[1] += (long long)n * item_length(s);
    mine[2] += s.tiles;
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    long long upto = mine[k];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) scratch[3 * warp + k] = upto;
    before[k] = upto - mine[k];
  }
  __syncthreads();
#pragma unroll 1
  for (int w = 0; w < kWarps; ++w) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const long long x = scratch[3 * w + k];
      if (w < warp) before[k] += x;
      total[k] += x;
    }
  }
  TallWalk<RP> w;
  w.wave = 0;
  w.ctas = C;
  w.item = (int)blockIdx.x;
  w.r = w.first_item = 0;
  w.base = 0;
  w.bounds = bounds;
  const bool waves = total[2] * p.num_kv_heads * ((long long)kTile * HD * 4) > kL2Keys && total[0] >= 2 * C && R <= kPlanReqs;
  w.waves = waves ? (int)(total[0] / C) - 1 : 0;
  if (!waves) {
    w.work = total[1];
    w.runs = (int)min((long long)C, max(w.work, 1ll));   // (none of them empty)
    w.at = (int)blockIdx.x < w.runs ? w.work * blockIdx.x / w.runs : w.work;
    w.end = (int)blockIdx.x < w.runs ? w.work * (blockIdx.x + 1) / w.runs : w.work;
    __syncthreads();   // (the sums have been read)
    if (w.at < w.end && before[1] <= w.at && w.at < before[1] + mine[1]) {
      long long start = before[1];
      int r = r0;
#pragma unroll 1
      for (;; ++r) {
        const ReqShape s = req_shape<RP>(p, r);
        const long long n = (long long)item_length(s) * s.row_tiles * p.num_kv_heads;
        if (w.at < start + n) break;
        start += n;
      }
      scratch[0] = r;
      scratch[1] = start;
    }
    __syncthreads();
    w.tail_r = (int)scratch[0];
    w.tail_start = scratch[1];
    return w;
  }
  // length_first[r] of the sequence and item_first[r] items lie in front of request r, whose items are length[r] long
  long long* const length_first = reinterpret_cast<long long*>(arrays);
  int* const item_first = reinterpret_cast<int*>(length_first + R);
  int* const length = item_first + R;
#pragma unroll 1
  for (int r = r0; r < r1; ++r) {
    const ReqShape s = req_shape<RP>(p, r);
    const int n = s.tiles > 0 ? s.row_tiles * p.num_kv_heads : 0;
    length[r] = item_length(s);
    item_first[r] = (int)before[0];
    length_first[r] = before[1];
    before[0] += n;
    before[1] += (long long)n * length[r];
  }
  __syncthreads();
  // request of an item, or of a position of the sequence: the last that begins at or in front of it
  auto last_of = [&](const auto* first, long long x) {
    int lo = 0, hi = R - 1;
#pragma unroll 1
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= x) lo = mid; else hi = mid - 1;
    }
    return lo;
  };
  const long long f = (long long)w.waves * C;
  const int fr = last_of(item_first, f);
  w.base = length_first[fr] + (f - item_first[fr]) * length[fr];
  w.work = total[1] - w.base;
  w.runs = 0;
  // CTA c has a load of the waves; the rest fills all up to a level: the smallest that holds it
#pragma unroll 1
  for (int c = tid; c < C; c += kThreads) {
    long long load = 0;
#pragma unroll 1
    for (int k = 0; k < w.waves; ++k) load += length[last_of(item_first, c + (long long)k * C)];
    bounds[c] = load;
  }
  __syncthreads();
  if (tid < 32) {
    constexpr int kRows = kMostCtas / 32;   // (CTAs lane + 32 i)
    long long most = 0;
#pragma unroll 1
    for (int c = lane; c < C; c += 32) most = max(most, bounds[c]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    long long lo = total[1] / C, hi = most + w.work / C + 1;   // (at lo there may be too little room, at hi there is enough)
#pragma unroll 1
    while (lo < hi) {
      const long long mid = (lo + hi) >> 1;
      long long room = 0;
#pragma unroll 1
      for (int c = lane; c < C; c += 32) room += max(0ll, mid - bounds[c]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) room += __shfl_xor_sync(0xffffffffu, room, o);
      if (room >= w.work) hi = mid; else lo = mid + 1;
    }
    long long upto = 0;
#pragma unroll 1
    for (int i = 0; i < kRows; ++i) {
      const int c = lane + 32 * i;
      const long long share = c < C ? max(0ll, lo - bounds[c]) : 0;
      long long inc = share;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
      }
      if (c < C) bounds[c] = min(w.work, upto + inc - share);
      upto += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) bounds[C] = w.work;
  }
  __syncthreads();
  w.r = last_of(item_first, w.item);
  w.first_item = item_first[w.r];
  w.at = w.base + bounds[blockIdx.x];
  w.end = w.base + bounds[blockIdx.x + 1];
  w.tail_r = last_of(length_first, w.at);
  w.tail_start = length_first[w.tail_r];
  tc::fence_async_smem();   // (boxes are written where the arrays are, through the other proxy)
  __syncthreads();
  return w;
}

template <int HD, bool kHalf, bool kHeld>
__global__ void __launch_bounds__(Tall<HD>::threads, Tall<HD>::ctas) kv16_tall_kernel(const __grid_constant__ Kv16Params p, const __grid_constant__ CUtensorMap k_map,
                                                                        const __grid_constant__ CUtensorMap v_map) {
  using G = Tall<HD>;
  using B = TallBars<HD>;
  constexpr int RP = G::rows;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024u - (tc::smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* const full = reinterpret_cast<uint64_t*>(smem + G::bars);
  uint64_t* const empty = full + G::units;
  uint64_t* const bars = empty + G::units;
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + G::misc);
  uint32_t* const tslot = reinterpret_cast<uint32_t*>(smem + G::misc + 4);
  int* const arrival = reinterpret_cast<int*>(smem + G::misc + 8);   // [2]
  int* const stop = arrival + 2;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (warp == G::mma_warp) {
    if (lane == 0) {
      for (int i = 0; i < G::units; ++i) {
        tc::mbar_init(&full[i], 32 * kLoadWarps);
        tc::mbar_init(&empty[i], G::rts);   // one commit per row tile
      }
      for (int i = 0; i < G::rts; ++i) {
        tc::mbar_init(&bars[B::q_full + i], 32 * kLoadWarps);
        tc::mbar_init(&bars[B::q_empty + i], 1);
        tc::mbar_init(&bars[B::drained + i], 1);
      }
      for (int i = 0; i < 4; ++i) {
        tc::mbar_init(&bars[B::s_ready + i], 1);
        tc::mbar_init(&bars[B::p_ready + 2 * i], 128);
        tc::mbar_init(&bars[B::p_ready + 2 * i + 1], 128);
        tc::mbar_init(&bars[B::pv_half + i], 1);
        tc::mbar_init(&bars[B::pv_done + i], 1);
      }
      PieceQueue(nullptr, &bars[B::queue], stop).init(G::threads / 32 - 1);
      *abort_flag = 0;
      tc::mbar_init_fence();
    }
    __syncwarp();
    tc::tmem_alloc(tslot, G::tmem);
    tc::tmem_relinquish();
  }
  pdl_wait();
  long long* const bounds = reinterpret_cast<long long*>(smem + G::bounds);
  const TallWalk<RP> plan = make_plan<HD, RP, G::threads, G::most_ctas>(p, smem, bounds);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem_base = *tslot;
  PieceQueue queue(reinterpret_cast<Piece*>(smem + G::pieces), &bars[B::queue], stop);
  bool ok = true;
  int issued = 0;   // units that this thread has had a part in (copying warps)

  if (warp == G::schedule_warp) {
    // =========================== schedule ========================================
    TallWalk<RP> w = plan;
    put_pieces<kHeld>(p, w, queue, &bars[B::drained], abort_flag);
  } else if (warp >= G::load_warp && warp < G::mma_warp) {
    // =========================== copies ==========================================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::copy_regs));
    const int base_key = (warp - G::load_warp) * 32;
    const uint32_t ring = tc::smem_u32(smem);
    uint32_t unit = 0;
    uint32_t q_count[G::rts];
#pragma unroll
    for (int i = 0; i < G::rts; ++i) q_count[i] = 0;
    // A unit: boxes of box_slots slots x 64 dims where pages allow it and the tile is visible as a whole, else 16-byte
    // copies, which leave out what is not visible.
    const int boxes = p.box_slots > 0 ? 32 / p.box_slots : 0;   // of this warp's keys
    const int box_lane = boxes > 0 ? (lane % boxes) * p.box_slots : 0;
    const bool boxing = lane < boxes * (G::dims / 64);
    // (Behind a wait that gave up nothing more is copied: a unit that is not free may be waiting for its boxes.)
    auto load_unit = [&](const CUtensorMap& map, const uint8_t* src, int part, int kvh, bool as_boxes, long long off, int blk, int slot) {
      const uint32_t s = unit % G::units;
      if (unit >= G::units && !kv16_wait(&empty[s], ((unit / G::units) - 1) & 1, abort_flag)) {
        if (ok) issued = (int)unit;
        ok = false;
      }
      if (as_boxes) {
        if (!ok) {
        } else if (boxing) {
          const int slab = lane / boxes;
          mbar_arrive_expect_tx(&full[s], p.box_slots * 128);
          tma_load_4d(ring + s * G::unit + slab * (kTile * 128) + (base_key + box_lane) * 128, &map, part * 128 + slab * 64, kvh, slot, blk, &full[s]);
        } else {
          mbar_arrive(&full[s]);
        }
        __syncwarp();
      } else {
        copy_keys<G::dims>(ring + s * G::unit, base_key, src + part * 256, off);
        if (ok) copies_arrive(&full[s]);
      }
      ++unit;
    };
    {
      KeyLookup keys(p, queue, abort_flag, base_key + lane);
      bool have = keys.fetch();
      while (have) {
        if (warp == G::load_warp && kv16_held<kHeld>(p, kHeldCopies, unit)) break;
        const int kvh = keys.it.kvh;
        const uint8_t* kb = p.k + (int64_t)kvh * p.stride_head;
        const uint8_t* vb = p.v + (int64_t)kvh * p.stride_head;
        const long long off = keys.offset();
        const bool first = keys.fresh, as_boxes = boxes > 0 && keys.key0 >= keys.it.lo && keys.key0 + kTile <= keys.it.hi;
        const int first_token = keys.it.first_token, row0 = keys.it.row0, rows = keys.it.rows;
        const int blk = __shfl_sync(0xffffffffu, keys.blk, box_lane), slot = __shfl_sync(0xffffffffu, keys.slot, box_lane);
        have = keys.fetch();
#pragma unroll
        for (int part = 0; part < G::parts; ++part) load_unit(k_map, kb, part, kvh, as_boxes, off, blk, slot);
        if (first) {
          // the piece's queries, behind its first keys: a row tile's as soon as QK has read the last one's
#pragma unroll
          for (int rt = 0; rt < G::rts; ++rt) {
            if (rows <= rt * 128) continue;
            if (q_count[rt] > 0) kv16_wait(&bars[B::q_empty + rt], (q_count[rt] - 1) & 1, abort_flag);
            ++q_count[rt];
            // a lane looks a row up, the warp copies it
            const int mine = rt * 128 + base_key + lane;
            int token, head;
            row_of(p, first_token, kvh, row0 + min(mine, rows - 1), &token, &head);
            const long long at = mine < rows ? (long long)token * p.q_stride_token + (long long)head * p.q_stride_head : -1ll;
#pragma unroll
            for (int part = 0; part < G::parts; ++part)
              copy_keys<G::dims>(tc::smem_u32(smem + G::q) + rt * G::qtile + part * (2 * kTile * 128), base_key, p.q + part * 256, at);
            copies_arrive(&bars[B::q_full + rt]);
          }
        }
#pragma unroll
        for (int part = 0; part < G::parts; ++part) load_unit(v_map, vb, part, kvh, as_boxes, off, blk, slot);
      }
    }
    copies_wait_all();
    if (ok) issued = (int)unit;
  } else if (warp >= G::mma_warp) {
    // =========================== MMAs ============================================
    const int rt = warp - G::mma_warp;
    constexpr uint32_t fmt = kHalf ? tc::kFmtF16 : tc::kFmtBF16;
    constexpr uint32_t qk_desc = tc::instr_desc(128, G::keys, fmt, fmt, 0, 0);
    constexpr uint32_t pv_desc = tc::instr_desc(128, G::dims, fmt, fmt, 0, 1);
    // (descriptors as two words, of which a step along an operand changes the lower one)
    const uint64_t q_desc = swizzled_desc(tc::smem_u32(smem + G::q) + rt * G::qtile, 16, 1024);
    const uint64_t k_desc = swizzled_desc(tc::smem_u32(smem), 16, 1024);
    const uint64_t v_desc = swizzled_desc(tc::smem_u32(smem), kTile * 128, 1024);
    const uint32_t o_tmem = tmem_base + G::o_col + rt * HD, s_tmem = tmem_base + G::s_col + 2 * rt * G::keys;
    // (this warp's own instructions bound the kernel before its MMAs do: it keeps ring slots and phases instead of dividing,
    // and asks and fences only where there is something to wait for)
    uint32_t k_slot[G::parts], k_phase[G::parts], v_slot[G::parts], v_phase[G::parts];   // of the next tile's units
#pragma unroll
    for (int part = 0; part < G::parts; ++part) {
      k_slot[part] = part;
      v_slot[part] = G::parts + part;
      k_phase[part] = v_phase[part] = 0;
    }
    static_assert(2 * G::parts <= G::units, "a tile's units lap the ring at most once");
    auto next_tile = [&](uint32_t (&slot)[G::parts], uint32_t (&phase)[G::parts]) {
#pragma unroll
      for (int part = 0; part < G::parts; ++part) {
        slot[part] += 2 * G::parts;
        if (slot[part] >= G::units) {
          slot[part] -= G::units;
          phase[part] ^= 1;
        }
      }
    };
    auto landed = [&](const uint32_t (&slot)[G::parts], const uint32_t (&phase)[G::parts], bool copied) {
#pragma unroll
      for (int part = 0; part < G::parts; ++part) ok &= kv16_wait(&full[slot[part]], phase[part], abort_flag);
      if (copied) tc::fence_async_smem();   // (16-byte copies wrote through the generic proxy)
    };
    uint32_t s_qk = 0, s_pv = 0, pieces = 0; // steps so far, pieces with live rows
    auto qk = [&](int sub, bool copied, bool tile_ends, bool first, bool last) {
      const uint32_t b = s_qk & 1;
      if (first) {
        ok &= kv16_wait(&bars[B::q_full + rt], (pieces - 1) & 1, abort_flag);
        tc::fence_async_smem();
      }
      if (sub == 0) landed(k_slot, k_phase, copied);
      if (s_qk > 1) ok &= kv16_wait(&bars[B::pv_done + 2 * rt + b], ((s_qk >> 1) - 1) & 1, abort_flag);   // (P of the step before last has been read)
      {
        tc::fence_after_sync();
#pragma unroll
        for (int part = 0; part < G::parts; ++part) {
          const uint32_t klo = (uint32_t)k_desc + k_slot[part] * (G::unit >> 4) + sub * ((G::keys * 128) >> 4), qlo = (uint32_t)q_desc + part * ((2 * kTile * 128) >> 4);
#pragma unroll
          for (int kk = 0; kk < G::dims / 16; ++kk) {
            constexpr uint32_t slab = (kTile * 128) >> 4;
            const uint32_t at = (kk >> 2) * slab + (kk & 3) * 2;
            if (part == 0 && kk == 0) mma_ss_words<false>(s_tmem + b * G::keys, qlo + at, (uint32_t)(q_desc >> 32), klo + at, (uint32_t)(k_desc >> 32), qk_desc);
            else mma_ss_words<true>(s_tmem + b * G::keys, qlo + at, (uint32_t)(q_desc >> 32), klo + at, (uint32_t)(k_desc >> 32), qk_desc);
          }
          if (tile_ends && ok) tc::mma_commit(&empty[k_slot[part]]);   // (a unit that has not landed is not given back)
        }
        tc::mma_commit(&bars[B::s_ready + 2 * rt + b]);
        if (last) tc::mma_commit(&bars[B::q_empty + rt]);
      }
      if (tile_ends) next_tile(k_slot, k_phase);
      ++s_qk;
    };
    auto pv = [&](int sub, bool copied, bool tile_ends, bool first) {
      const uint32_t b = s_pv & 1;
      if (sub == 0) landed(v_slot, v_phase, copied);
#pragma unroll
      for (int half = 0; half < G::halves; ++half) {
        ok &= kv16_wait(&bars[B::p_ready + 2 * (2 * rt + b) + half], (s_pv >> 1) & 1, abort_flag);
        {
          tc::fence_after_sync();
#pragma unroll
          for (int part = 0; part < G::parts; ++part) {
            const uint32_t vlo = (uint32_t)v_desc + v_slot[part] * (G::unit >> 4) + (sub * G::keys + half * 64) * (128 >> 4);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_ts_words(o_tmem + part * 128, s_tmem + b * G::keys + half * 32 + kk * 8, vlo + kk * (2048 >> 4), (uint32_t)(v_desc >> 32), pv_desc,
                           !first || half > 0 || kk > 0);
            if (tile_ends && half == G::halves - 1 && ok) tc::mma_commit(&empty[v_slot[part]]);
          }
          tc::mma_commit(&bars[(half == G::halves - 1 ? B::pv_done : B::pv_half) + 2 * rt + b]);
        }
      }
      if (tile_ends) next_tile(v_slot, v_phase);
      ++s_pv;
    };
    Piece it;
    const bool leader = elect_one();   // (one lane takes all steps of a piece: the others would only have to be waited for)
    while (queue.get(&it, abort_flag)) {
      if (!leader || !ok) continue;
      if (it.rows <= rt * 128) {   // no rows: free the units as if they had been read
#pragma unroll 1
        for (int i = 0; i < it.tiles; ++i) {
          landed(k_slot, k_phase, false);
          landed(v_slot, v_phase, false);
          if (!ok) break;
#pragma unroll
          for (int part = 0; part < G::parts; ++part) {
            mbar_arrive(&empty[k_slot[part]]);
            mbar_arrive(&empty[v_slot[part]]);
          }
          next_tile(k_slot, k_phase);
          next_tile(v_slot, v_phase);
        }
        continue;
      }
      ++pieces;
      const int n = piece_steps<G::keys>(it);
      auto tile_copied = [&](int j) {   // (as the copying warps decide it)
        const int key0 = it.key0 + j / G::steps * kTile;
        return p.box_slots == 0 || key0 < it.lo || key0 + kTile > it.hi;
      };
      // QK of a step ahead of PV of the one before: the softmax finds the next S when it is done with one
#pragma unroll 1
      for (int j = 0; j <= n; ++j) {
        if (kv16_held<kHeld>(p, kHeldMma, s_qk)) ok = false;
        if (!ok) break;
        if (j < n) qk(j % G::steps, tile_copied(j), j % G::steps == G::steps - 1 || j == n - 1, j == 0, j == n - 1);
        if (j > 0) pv((j - 1) % G::steps, tile_copied(j - 1), (j - 1) % G::steps == G::steps - 1 || j == n, j == 1);
      }
    }
  } else {
    // =========================== softmax =========================================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::softmax_regs));
    const int rt = warp >> 2;
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_tmem = tmem_base + G::o_col + rt * HD + lane_addr;
    const int row = tid;   // of the CTA's rows
    uint32_t count = 0;    // live tiles so far
    auto rt_sync = [&] { named_barrier(1 + rt, 128); };
    zero_requests<HD, RP, 128 * G::rts>(p);
    {
      Piece it;
      while (queue.get(&it, abort_flag)) {
        if (it.rows <= rt * 128) continue;
        const int kvh = it.kvh;
        const bool padding = (row & ~31) >= it.rows;   // (of the whole warp)
        float ref = -INFINITY, l = 0.f;
        const int n_steps = piece_steps<G::keys>(it);
        for (int t = 0; t < n_steps; ++t, ++count) {
          const uint32_t b = 2 * rt + (count & 1), use = count >> 1;
          const uint32_t s_tmem = tmem_base + G::s_col + b * G::keys + lane_addr;
          ok &= kv16_wait(&bars[B::s_ready + b], use & 1, abort_flag);
          if (padding) {   // (the order of the waits is kept, nothing is computed)
#pragma unroll
            for (int half = 0; half < G::halves; ++half) mbar_arrive(&bars[B::p_ready + 2 * b + half]);
            continue;
          }
          tc::fence_after_sync();
          const int key0 = it.key0 + t * G::keys;
          const bool edge = key0 < it.lo || key0 + G::keys > it.hi;
          // (one copy of the code for both halves: the instruction cache is small)
#pragma unroll 1
          for (int half = 0; half < G::halves; ++half) {
            uint32_t r[64];
            tc::tmem_ld32(s_tmem + half * 64, r);
            tc::tmem_ld32(s_tmem + half * 64 + 32, r + 32);
            tc::tmem_ld_wait<64>(r);
            if (edge) {
              const int pos0 = key0 + half * 64;
#pragma unroll
              for (int n = 0; n < 64; ++n)
                if (pos0 + n < it.lo || pos0 + n >= it.hi) r[n] = 0xff800000u;  // -inf
            }
            auto maximum = [&] {
              float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
              for (int n = 0; n < 64; n += 8) {
#pragma unroll
                for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(r[n + 2 * e]), __uint_as_float(r[n + 2 * e + 1]));
              }
              return max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * p.scale_log2 - kGain<kHalf>;
            };
            if (t == 0 && half == 0) ref = maximum();
            uint32_t pk[32];
            float total = exponentials<kHalf>(r, p.scale_log2, ref == -INFINITY ? 0.f : -ref, pk);
            const bool outgrown = !(total <= kMostSum<kHalf>) || ref == -INFINITY;
            if (__any_sync(0xffffffffu, outgrown)) {
              const float to = outgrown ? fmaxf(ref, maximum()) : ref;
              const float alpha = to == -INFINITY ? 1.f : ex2f(ref - to);
              ref = to;
              l *= alpha;
              if (t > 0 || half > 0) {   // (PV of what P holds already is complete first)
                if (half > 0) {
                  ok &= kv16_wait(&bars[B::pv_half + b], use & 1, abort_flag);
                } else {
                  ok &= kv16_wait(&bars[B::pv_done + (b ^ 1)], ((count - 1) >> 1) & 1, abort_flag);
                }
                tc::fence_after_sync();
#pragma unroll 1
                for (int d = 0; d < HD / 16; ++d) {
                  uint32_t o[16];
                  tc::tmem_ld16(o_tmem + d * 16, o);
                  tc::tmem_ld_wait<16>(o);
#pragma unroll
                  for (int n = 0; n < 16; ++n) o[n] = __float_as_uint(weighed(__uint_as_float(o[n]), alpha));
                  tc::tmem_st16(o_tmem + d * 16, o);
                }
                tc::tmem_st_wait();
              }
              total = exponentials<kHalf>(r, p.scale_log2, ref == -INFINITY ? 0.f : -ref, pk);
            }
            l += total;
            tc::tmem_st32(s_tmem + half * 32, pk);
            tc::tmem_st_wait();
            tc::fence_before_sync();
            mbar_arrive(&bars[B::p_ready + 2 * b + half]);
          }
        }
        // ---- the piece's rows ----
        {
          ok &= kv16_wait(&bars[B::pv_done + 2 * rt + ((count - 1) & 1)], ((count - 1) >> 1) & 1, abort_flag);
          tc::fence_after_sync();
        }
        const bool whole = it.begins && it.ends, live = row < it.rows;
        int token, head;
        row_of(p, it.first_token, kvh, it.row0 + min(row, it.rows - 1), &token, &head);
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
          const float inv = l == 0.f ? 0.f : 1.f / l;
          float* const slot = tall_slot<HD>(p, (int)blockIdx.x, it.begins) + row;
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t r[32];
            tc::tmem_ld32(o_tmem + c * 32, r);
            tc::tmem_ld_wait<32>(r);
            if (whole) {
              float o[32];
#pragma unroll
              for (int n = 0; n < 32; ++n) o[n] = __uint_as_float(r[n]) * inv;
              if (live) {
                write16(o, c * 32);
                write16(o + 16, c * 32 + 16);
              }
            } else {
#pragma unroll
              for (int n = 0; n < 32; ++n) slot[(c * 32 + n) * RP] = __uint_as_float(r[n]);
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
          auto none = [&](int c) { return it.sparse != 0 && bounds[c] == bounds[c + 1]; };   // (a CTA with much of the waves may have none of the rest)
          rt_sync();
          int* const counter = reinterpret_cast<int*>(p.workspace) + G::rts * c0 + rt;
          if ((tid & 127) == 0) {
            int pieces = 0;
            for (int c = c0; c <= c1; ++c) pieces += none(c) ? 0 : 1;
            arrival[rt] = arrive_at(counter) == pieces - 1;
            if (arrival[rt]) *counter = 0;   // (for the next call)
          }
          rt_sync();
          if (arrival[rt] && !padding) {
            auto slot = [&](int c) { return tall_slot<HD>(p, c, c == c0) + row; };
            float top = -INFINITY, sum = 0.f;
            // (the loads of two pieces are in flight together; one that there is not counts nothing)
#pragma unroll 1
            for (int c = c0; c <= c1; c += 2) {
              const bool a = !none(c), b = c < c1 && !none(c + 1);
              const float* s = slot(a ? c : c0) + HD * RP;
              const float* t = slot(b ? c + 1 : c0) + HD * RP;
              const float ra = a ? __ldcg(s) : -INFINITY, la = __ldcg(s + RP), rb = b ? __ldcg(t) : -INFINITY, lb = __ldcg(t + RP);
              const float to = max3(top, ra, rb), use = to == -INFINITY ? 0.f : to;
              sum = fmaf(sum, ex2f(top - use), a ? ex2f(ra - use) * la : 0.f);
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
                const bool a = !none(cta), b = cta < c1 && !none(cta + 1);
                const float* s = slot(a ? cta : c0);
                const float* t = slot(b ? cta + 1 : c0);
                const float wa = __ldcg(s + HD * RP), wb = __ldcg(t + HD * RP);
                float v[16], u[16];
#pragma unroll
                for (int n = 0; n < 16; ++n) {
                  v[n] = __ldcg(s + (c * 16 + n) * RP);
                  u[n] = __ldcg(t + (c * 16 + n) * RP);
                }
                const float fa = a ? ex2f(wa - use) * inv : 0.f, fb = b ? ex2f(wb - use) * inv : 0.f;
                if (__any_sync(0xffffffffu, (a && fa == 0.f) || (b && fb == 0.f))) {   // a piece far below the others: its infinities count
#pragma unroll
                  for (int n = 0; n < 16; ++n) {
                    if (a) o[n] += weighed(v[n], fa);
                    if (b) o[n] += weighed(u[n], fb);
                  }
                  continue;
                }
#pragma unroll
                for (int n = 0; n < 16; ++n) {
                  if (a) o[n] = fmaf(fa, v[n], o[n]);
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
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (*abort_flag) {   // (the same in all threads) what is in flight comes to its end first: MMAs, and boxes
    if (warp >= G::mma_warp && warp < G::schedule_warp && elect_one()) {
      uint64_t* const drained = &bars[B::drained + warp - G::mma_warp];
      tc::mma_commit(drained);
      kv16_drain(drained, 0);
    }
    // (the copying threads stopped at units of their own: who has stopped short of another arrives without a copy, so that
    // the units' last phases end with what has been asked for)
    int* const most = arrival;
    if (tid == 0) *most = 0;
    __syncthreads();
    atomicMax(most, issued);
    __syncthreads();
    if (warp >= G::load_warp && warp < G::mma_warp) {
      for (; issued < *most; ++issued) mbar_arrive(&full[issued % G::units]);
      for (int u = max(0, issued - G::units); u < issued; ++u) kv16_drain(&full[u % G::units], (u / G::units) & 1);
    }
    if (tid == 0) atomicOr(&g_kv16_tall_status, 16u);
    __syncthreads();
  }
  if (warp == G::mma_warp) tc::tmem_dealloc(tmem_base, G::tmem);
}

// Tensor map over one of the caches, [dims][heads][slots][blocks], a box being 64 dims of box_slots slots of one head, in the
// 128-byte swizzle.  False: the driver refuses the view.  (Encoded for every call: a microsecond of the host.)
bool page_box_map(const Kv16Params& p, const uint8_t* base, CUtensorMap* map) {
  const EncodeTiledFn fn = encode_tiled_fn();
  const cuuint64_t dims[4] = {(cuuint64_t)p.head_size, (cuuint64_t)p.num_kv_heads, (cuuint64_t)p.block_size, (cuuint64_t)p.num_blocks};
  const cuuint64_t strides[3] = {(cuuint64_t)p.stride_head, (cuuint64_t)p.stride_slot, (cuuint64_t)p.stride_block};
  const cuuint32_t box[4] = {64, 1, (cuuint32_t)p.box_slots, 1}, elem[4] = {1, 1, 1, 1};
  return fn != nullptr && fn(map, p.dtype == PTH_ATTN_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                             const_cast<uint8_t*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, bool kHalf, bool kHeld = false>
cudaError_t launch_one(const Kv16Params& p, cudaStream_t stream) {
  using G = Tall<HD>;
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    err = cudaFuncSetAttribute(kv16_tall_kernel<HD, kHalf, kHeld>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::total);
    if (err != cudaSuccess) return err;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int sms = sm_count();
  if (sms <= 0 || sms > kTallSms) return cudaErrorInvalidDevice;
  // Boxes take pages of a multiple of 8 slots: the swizzle repeats every 8 rows.
  Kv16Params q = p;
  q.box_slots = 0;
  q.out_wide = reinterpret_cast<uintptr_t>(p.out) % 32 == 0 && p.out_stride_token % 32 == 0 && p.out_stride_head % 32 == 0;
  for (int slots = 32; slots >= 8 && q.box_slots == 0; slots >>= 1)
    if (p.block_size % slots == 0) q.box_slots = slots;
  CUtensorMap k_map{}, v_map{};
  if (q.box_slots > 0 && !(page_box_map(q, p.k, &k_map) && page_box_map(q, p.v, &v_map))) q.box_slots = 0;
  return pdl_launch(kv16_tall_kernel<HD, kHalf, kHeld>, dim3((unsigned)(sms * G::ctas)), dim3(G::threads), G::total, stream, q, k_map, v_map);
}
template <int HD>
cudaError_t launch_type(const Kv16Params& p, cudaStream_t stream) {
  return p.dtype == PTH_ATTN_F16 ? launch_one<HD, true>(p, stream) : launch_one<HD, false>(p, stream);
}

}  // namespace

// Counters, and two partial row tiles per CTA.
int64_t kv16_tall_workspace_bytes(int head_size, int num_sms) {
  const int64_t rows = head_size == 256 ? 128 : 256;   // of an SM's CTAs together
  return kCounterBytes + (int64_t)num_sms * 2 * rows * (head_size + 2) * 4;
}

cudaError_t launch_kv16_tall(const Kv16Params& p, cudaStream_t stream) {
  switch (p.head_size) {
    case 64:
      return launch_type<64>(p, stream);
    case 128:
      return launch_type<128>(p, stream);
    default:
      return launch_type<256>(p, stream);
  }
}

cudaError_t launch_kv16_tall_held(const Kv16Params& p, cudaStream_t stream) { return launch_one<128, false, true>(p, stream); }

// Reads and clears this kernel's status word (device must be idle).
cudaError_t read_kv16_tall_status(unsigned int* v) {
  unsigned int zero = 0;
  cudaError_t err = cudaMemcpyFromSymbol(v, g_kv16_tall_status, sizeof(*v));
  if (err != cudaSuccess) return err;
  return cudaMemcpyToSymbol(g_kv16_tall_status, &zero, sizeof(zero));
}

}  // namespace pthb200
