// Attention over the 16-bit paged cache for requests of few query rows (a row is a query token and head): one-token decode,
// cross attention of a few tokens.
//
// Orientation: the 128 keys of a tile sit on the MMA's M dimension, the rows of a KV head on N, so tensor work goes
// into keys and not into padding:
//   S^T[key, row] = sum_d K[key, d] Q[row, d]         A = K as it lies in the cache (K-major), B = Q
//   O^T[d, row]  += sum_key V[key, d] P[key, row]     A = V as it lies in the cache (MN-major), B = P
// Both operands A are the cache's own bytes: no element of K or V passes through a register.
//
// Softmax in one pass: ref is a running bound of a row's scores (log2 units), P = 2^(s - ref), l = sum P.  ref is a row's
// maximum less kGain when it is set, and moves (with l and O rescaled) only when a score outgrows it by kSlack, so that most
// tiles need no maximum at all, only a vote of the 128 threads.  P goes into the MMA as the sum of two 16-bit
// numbers (hi + lo: 2 x 8 or 2 x 11 bits), side by side on N: at the instruction's minimum of 16 columns that costs
// eight rows nothing, and the outputs' error is their own rounding (with one: 1.4 times it).
//
// What bounds it: the cache's bytes, 4 D per key and KV head at 4 D G flops.  The tile's parts (128 keys x 128 dims of K, of
// V) are units of one ring of shared memory, K of the next tile ahead of V of this one, which is the order in which they are
// used; four warps fill it with 16-byte copies that go to their swizzled place, zero where a key is not visible (so what lies
// there in memory, NaN included, is never read).  Two CTAs per SM keep 192 KB in flight.  Copies of pages instead (tiled
// TMA, boxes of 16 slots x 64 dims, 64 requests x 8,192 keys x 8 heads x 128 dims) moved 6.83 TB/s, with boxes of 4 KB 7.06, 16-byte
// copies 7.17, which also take pages of any size and place.
//
// Measured, bf16, one call behind another: 64 requests x 8,192 keys, 32 heads of 8, 128 dims 321 us, 6.7 TB/s; 61 x 4,096-12,288, 12 of
// 2, 256 dims 161 us, 6.5 TB/s; one request of 131,072 keys 91 us, 5.9 TB/s, of which the last arriver's merge of 37 pieces and
// the start are 9; 8 requests of up to 4,095 keys 22.1 us for 79 MB, some 5 in front of the first tile (the launch, the
// lengths, the block table, the first keys: one after the other) and 5 behind the last (the merge).
//
// Schedule: the keys of all (request, row tile) form one sequence, which is cut into equal runs, one for every group of Hkv CTAs;
// CTA h of a group reads head h, so that the heads of a page are read at the same time.  The pieces of a row tile that a cut
// divides are merged by the CTA that arrives last: one launch, and the same bits whoever is last.
#include "kv16_sched.cuh"
#include "page_copy.cuh"
#include "pdl.cuh"

namespace pthb200 {

__device__ unsigned int g_kv16_status = 0;

namespace {

constexpr int kSoftmaxThreads = 128;   // warps 0-3: thread t is key t of a tile, then dim t of the output
constexpr int kLoadWarp = 4;           // warps 4-7
constexpr int kMmaWarp = 8, kScheduleWarp = 9;
constexpr int kThreads = 320;
// The sequence is counted in grains of 32 keys; a row tile counts kPieceGrains more, what its queries and its end take.  (With 0, 4
// and 8, us: 200 requests of up to 500 keys 65.5, 61.4, 61.5; 300 of up to 300 at 256 dims 47.1, 41.0, 38.9; 8 of up to 4,095 32.8,
// 30.7, 30.7; 2,000 of 100 260, 258, 256.  Grains of 128 keys: 4 requests of 500 18.4 instead of 16.4.)
constexpr int kGrain = 32, kPieceGrains = 4;
// Length of a run at least, so that few keys are not spread over pieces that cost more to merge: with 1, 4 and 16, us, one request
// of 2,000 keys 24.6, 18.5, 18.4, four of 500 16.4, 16.4, 18.4.
constexpr int kRunMin = 4;
constexpr float kSlack = 8.f;

template <int HD, int RP>
struct Geo {
  static constexpr int dims = HD < 128 ? HD : 128;   // of a unit
  static constexpr int parts = HD / dims;            // units of a tile's K, and of its V
  static constexpr int unit = kTile * dims * 2;
  static constexpr int cols = RP < 16 ? 16 : RP;     // N of QK (its rows past RP repeat the first)
  static constexpr int qimage = RP * HD * 2;
  static constexpr int pimage = 2 * RP * kTile * 2;
  static constexpr int fixed = 2 * qimage + pimage + 4 * RP * 4 * 2 + 768;
  // Two CTAs per SM where three units fit, else one: one's softmax and merge beside the other's copies.  (One against two, us: 64 requests
  // x 8,192 keys 348 / 329, 64 x 2,000 109 / 104, 64 x 64-1,500 at 64 dims 70 / 57.)
  static constexpr int units2 = (115712 - fixed - 1024) / unit;
  static constexpr int ctas = units2 >= 3 && RP <= 16 ? 2 : 1;
  static constexpr int most = 98304 * (3 - ctas) / unit;
  static constexpr int fit = ctas == 2 ? units2 : (232448 - fixed - 1024) / unit;
  static constexpr int units = fit < most ? fit : most;
  static_assert(units >= 3, "K and V of a tile, and the next K");
  // Registers that the copies hand to the softmax from what a thread starts with (168 with one CTA per SM, 96 with two); with 8
  // rows nothing spills as it is.
  static constexpr bool moves = RP == 32 || (RP == 16 && ctas == 2);
  static constexpr int softmax_regs = RP == 32 ? 232 : 128, copy_regs = RP == 32 ? 72 : 64, start_regs = RP == 32 ? 168 : 96;
  static_assert(!moves || 4 * softmax_regs + 4 * copy_regs <= 8 * start_regs, "a split that the launch holds");
  static constexpr int s_col = 0, o_col = 2 * cols;  // TMEM columns: S twice, O of every part (hi, lo)
  static constexpr int tmem_need = 2 * cols + parts * 2 * RP;
  static constexpr int tmem = tmem_need <= 64 ? 64 : tmem_need <= 128 ? 128 : 256;
  static_assert(tmem_need <= 256, "two CTAs share the SM's columns");
  // shared memory, behind the first 1,024-byte boundary
  static constexpr int q = units * unit;
  static constexpr int p = q + 2 * qimage;
  static constexpr int wmax = p + pimage;            // float [4 warps][RP]
  static constexpr int wsum = wmax + 4 * RP * 4;     // float [4 warps][RP]
  static constexpr int pieces = wsum + 4 * RP * 4;   // PieceQueue's entries
  static constexpr int bars = pieces + kQueue * 64;
  static constexpr int n_bars = 2 * units + 2 + 2 + 1 + 1 + 2 * kQueue + 1;
  static constexpr int misc = bars + n_bars * 8;     // ints: abort flag, TMEM address, arrival, stop; scratch of find_run
  static constexpr int total = misc + 160 + 1024;
  static_assert(kQueue * 64 + n_bars * 8 + 160 <= 768, "fixed part");
};

struct Bars {  // offsets behind [units] full, [units] empty
  static constexpr int q_empty = 0, s_ready = 2, p_ready = 4, pv_done = 5, queue = 6, drained = queue + 2 * kQueue;
};

// Length of a row tile in the sequence: its keys in grains, and what a piece costs besides.
template <int RP>
__device__ __forceinline__ int row_tile_length(const ReqShape& s) {
  return s.tiles > 0 ? (s.hi - s.lo / kGrain * kGrain + kGrain - 1) / kGrain + kPieceGrains : 0;
}
// The run of a CTA: a walk over its pieces.
template <int RP>
struct ShortWalk {
  long long at, end, start;   // position in the sequence, end of the run, start of request r
  int r, kvh;
  long long begin, first_start;   // where the run begins, for further KV heads
  int first_r, heads;
  long long work;             // length of the sequence
  int groups;                 // that it is cut among
  // Group that has position x of the sequence.
  __device__ __forceinline__ int owner(long long x) const { return (int)(((x + 1) * groups - 1) / work); }
  __device__ __forceinline__ bool next(const Kv16Params& p, Piece* out) {
    for (;;) {
      if (at >= end) {
        kvh += heads;
        if (begin >= end || kvh >= p.num_kv_heads) return false;
        at = begin;
        start = first_start;
        r = first_r;
      }
      ReqShape s = req_shape<RP>(p, r);
      int n = row_tile_length<RP>(s);
      while (at >= start + (long long)n * s.row_tiles) {
        start += (long long)n * s.row_tiles;
        ++r;
        s = req_shape<RP>(p, r);
        n = row_tile_length<RP>(s);
      }
      const long long off = at - start;
      const int rt = s.row_tiles == 1 ? 0 : (int)(off / n), a = (int)(off - (long long)rt * n);
      const int b = (int)min((long long)n, a + (end - at));
      at += b - a;
      if (b <= kPieceGrains) continue;   // (no keys yet)
      const int base = s.lo / kGrain * kGrain;
      out->r = r;
      out->kvh = kvh;
      out->row0 = rt * RP;
      out->rows = min(RP, s.tokens * p.group - rt * RP);
      out->first_token = s.first;
      out->key0 = base + max(0, a - kPieceGrains) * kGrain;
      out->lo = max(s.lo, out->key0);
      out->hi = min(s.hi, base + (b - kPieceGrains) * kGrain);
      out->tiles = (out->hi - out->key0 + kTile - 1) / kTile;
      out->begins = a <= kPieceGrains;
      out->ends = b == n;
      out->first_cta = owner(start + (long long)rt * n + kPieceGrains);
      out->last_cta = owner(start + (long long)rt * n + n - 1);
      return true;
    }
  }
};
// Cuts the sequence, of which [before, before + mine) are requests from r0 on.  Returns whether this CTA's run begins among
// them, and where.
template <int RP>
__device__ __forceinline__ bool begin_run(const Kv16Params& p, ShortWalk<RP>& w, int group, int r0, long long before, long long mine, int* r, long long* start) {
  w.groups = (int)min((long long)((int)gridDim.x / w.heads), max(w.work / kRunMin, 1ll));
  w.begin = group < w.groups ? w.work * group / w.groups : 0;
  w.end = group < w.groups ? w.work * (group + 1) / w.groups : 0;
  if (w.begin >= w.end || w.begin < before || w.begin >= before + mine) return false;
  *start = before;
#pragma unroll 1
  for (*r = r0;; ++*r) {
    const ReqShape s = req_shape<RP>(p, *r);
    const long long n = (long long)row_tile_length<RP>(s) * s.row_tiles;
    if (w.begin < *start + n) return true;
    *start += n;
  }
}
// Every CTA sums the requests' lengths up for itself, with all its threads (its scheduling warp alone, while the others go
// on: 0.2 us less at 8 and 64 requests, twice the code).  scratch: 64-bit words, warps + 2.
template <int RP>
__device__ __forceinline__ ShortWalk<RP> find_run(const Kv16Params& p, long long* scratch) {
  constexpr int kWarps = kThreads / 32;
  const int tid = threadIdx.x;
  ShortWalk<RP> w;
  w.heads = min(p.num_kv_heads, (int)gridDim.x);   // KV heads that a group reads at the same time
  w.kvh = (int)blockIdx.x % w.heads;
  const int group = (int)blockIdx.x / w.heads;
  const int per = (p.num_reqs + kThreads - 1) / kThreads, r0 = min(p.num_reqs, tid * per), r1 = min(p.num_reqs, r0 + per);
  long long mine = 0;
#pragma unroll 1
  for (int r = r0; r < r1; ++r) {
    const ReqShape s = req_shape<RP>(p, r);
    mine += (long long)row_tile_length<RP>(s) * s.row_tiles;
  }
  const long long before = scan_threads<kThreads>(mine, scratch, &w.work);
  int r = 0;
  long long start = 0;
  if (begin_run<RP>(p, w, group, r0, before, mine, &r, &start)) {
    scratch[kWarps] = r;
    scratch[kWarps + 1] = start;
  }
  __syncthreads();
  w.at = w.begin;
  w.first_r = w.r = (int)scratch[kWarps];
  w.first_start = w.start = scratch[kWarps + 1];
  return w;
}

// Barrier of the softmax warps that tells whether any of them has seen `x`.
__device__ __forceinline__ bool softmax_any(bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t"
      "}\n"
      : "=r"(r)
      : "r"((uint32_t)x)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void softmax_sync() { named_barrier(1, kSoftmaxThreads); }

template <int N>
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t* r) {
  if constexpr (N == 8) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr)
                 : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 16) tc::tmem_ld16(addr + i, r + i);
  }
}
template <int N>
__device__ __forceinline__ void tmem_store(uint32_t addr, const uint32_t* r) {
  if constexpr (N == 8) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 16) tc::tmem_st16(addr + i, r + i);
  }
}

// Two numbers as 16-bit parts: hi is their rounding, but the type's smallest normal number at least, lo the rounding of what is
// left.  So hi is above zero for every key, and an infinite value makes its part of the output infinite: that part says so,
// whatever the sign of lo is (a hi of zero, or hi and lo together, would make it NaN).  Keys that are not visible have values of zero.
template <bool kHalf>
__device__ __forceinline__ void split2(float a, float b, uint32_t* hi, uint32_t* lo) {
  if constexpr (kHalf) {
    const __half2 h = __hmax2_nan(__floats2half2_rn(a, b), __floats2half2_rn(0x1p-14f, 0x1p-14f));
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    *hi = *reinterpret_cast<const uint32_t*>(&h);
    *lo = *reinterpret_cast<const uint32_t*>(&l);
  } else {
    const __nv_bfloat162 h = __hmax2_nan(__floats2bfloat162_rn(a, b), __floats2bfloat162_rn(0x1p-126f, 0x1p-126f));
    const uint32_t w = *reinterpret_cast<const uint32_t*>(&h);
    const __nv_bfloat162 l = __floats2bfloat162_rn(a - __uint_as_float(w << 16), b - __uint_as_float(w & 0xffff0000u));
    *hi = w;
    *lo = *reinterpret_cast<const uint32_t*>(&l);
  }
}

template <int HD, int RP>
__device__ __forceinline__ float* partial_slot(const Kv16Params& p, int cta, bool begins) {
  float* base = reinterpret_cast<float*>(p.workspace + kCounterBytes);
  return base + (int64_t)(2 * cta + (begins ? 1 : 0)) * (RP * (HD + 2));  // [RP][HD] O, [RP] ref, [RP] l
}

// Merges the pieces of a row tile, left by the CTAs of groups g0 .. g0 + pieces - 1, and writes its rows: a warp per row, a lane per
// four columns.  The statistics and columns of eight pieces (four at 256 dims) are loaded together; the running sums are rescaled when a later piece has the
// larger ref.
template <int HD, int RP, bool kHalf>
__device__ __forceinline__ void merge_pieces(const Kv16Params& p, const Piece& it, int kvh, int g0, int pieces, int heads, int hslot) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kVec = HD >= 128 ? HD / 128 : 1, kBatch = 8 / kVec;
  const int d0 = (HD == 64 ? lane & 15 : lane) * 4;
#pragma unroll 1
  for (int n = warp; n < it.rows; n += 4) {
    float top = -INFINITY, l = 0.f, acc[kVec][4];
#pragma unroll
    for (int v = 0; v < kVec; ++v) acc[v][0] = acc[v][1] = acc[v][2] = acc[v][3] = 0.f;
#pragma unroll 1
    for (int k0 = 0; k0 < pieces; k0 += kBatch) {
      float4 o[kBatch][kVec];
      float ref[kBatch], sum[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int k = min(k0 + b, pieces - 1);
        const float* s = partial_slot<HD, RP>(p, (g0 + k) * heads + hslot, k == 0);
        ref[b] = __ldcg(s + RP * HD + n);
        sum[b] = __ldcg(s + RP * HD + RP + n);
#pragma unroll
        for (int v = 0; v < kVec; ++v) o[b][v] = __ldcg(reinterpret_cast<const float4*>(s + n * HD + v * 128 + d0));
      }
      float to = top;
#pragma unroll
      for (int b = 0; b < kBatch; ++b) to = fmaxf(to, ref[b]);
      const float use = to == -INFINITY ? 0.f : to, alpha = kv16_exp2(top - use);
      top = to;
      l *= alpha;
      if (alpha == 0.f) {   // (the same in all lanes) out of exponents
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[v][e] = weighed(acc[v][e], alpha);
        }
      } else {
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[v][e] *= alpha;
        }
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (k0 + b >= pieces) break;
        const float f = kv16_exp2(ref[b] - use);
        l = fmaf(f, sum[b], l);
        if (f == 0.f) {   // (the same in all lanes)
#pragma unroll
          for (int v = 0; v < kVec; ++v) {
            acc[v][0] += weighed(o[b][v].x, 0.f);
            acc[v][1] += weighed(o[b][v].y, 0.f);
            acc[v][2] += weighed(o[b][v].z, 0.f);
            acc[v][3] += weighed(o[b][v].w, 0.f);
          }
        } else {
#pragma unroll
          for (int v = 0; v < kVec; ++v) {
            acc[v][0] = fmaf(f, o[b][v].x, acc[v][0]);
            acc[v][1] = fmaf(f, o[b][v].y, acc[v][1]);
            acc[v][2] = fmaf(f, o[b][v].z, acc[v][2]);
            acc[v][3] = fmaf(f, o[b][v].w, acc[v][3]);
          }
        }
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    int token, head;
    row_of(p, it.first_token, kvh, it.row0 + n, &token, &head);
    uint8_t* out = p.out + (int64_t)token * p.out_stride_token + (int64_t)head * p.out_stride_head;
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      const uint2 w = make_uint2(pack16<kHalf>(acc[v][0] * inv, acc[v][1] * inv), pack16<kHalf>(acc[v][2] * inv, acc[v][3] * inv));
      if (HD >= 128 || lane < 16) *reinterpret_cast<uint2*>(out + (v * 128 + d0) * 2) = w;
    }
    if (lane == 0 && p.lse != nullptr)
      p.lse[(int64_t)token * p.num_q_heads + head] = l == 0.f ? -INFINITY : ((top == -INFINITY ? 0.f : top) + log2f(l)) * kLn2;
  }
}

template <int HD, int RP, bool kHalf, bool kHeld>
__global__ void __launch_bounds__(kThreads, (Geo<HD, RP>::ctas)) kv16_short_kernel(const __grid_constant__ Kv16Params p) {
  using G = Geo<HD, RP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024u - (tc::smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* const full = reinterpret_cast<uint64_t*>(smem + G::bars);
  uint64_t* const empty = full + G::units;
  uint64_t* const bars = empty + G::units;
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + G::misc);
  uint32_t* const tslot = reinterpret_cast<uint32_t*>(smem + G::misc + 4);
  int* const arrival = reinterpret_cast<int*>(smem + G::misc + 8);
  int* const stop = arrival + 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (warp == kMmaWarp) {
    if (lane == 0) {
      for (int i = 0; i < G::units; ++i) {
        tc::mbar_init(&full[i], 128);
        tc::mbar_init(&empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        tc::mbar_init(&bars[Bars::q_empty + i], 1);
        tc::mbar_init(&bars[Bars::s_ready + i], 1);
      }
      tc::mbar_init(&bars[Bars::p_ready], kSoftmaxThreads);
      tc::mbar_init(&bars[Bars::pv_done], 1);
      tc::mbar_init(&bars[Bars::drained], 1);
      PieceQueue(nullptr, &bars[Bars::queue], stop).init(kThreads / 32 - 1);
      *abort_flag = 0;
      tc::mbar_init_fence();
    }
    __syncwarp();
    tc::tmem_alloc(tslot, G::tmem);
    tc::tmem_relinquish();
  }
  pdl_wait();
  ShortWalk<RP> walk = find_run<RP>(p, reinterpret_cast<long long*>(smem + G::misc + 16));
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem_base = *tslot;
  PieceQueue queue(reinterpret_cast<Piece*>(smem + G::pieces), &bars[Bars::queue], stop);
  bool ok = true;

  if (warp == kScheduleWarp) {
    // =========================== schedule ========================================
    put_pieces<kHeld>(p, walk, queue, &bars[Bars::drained], abort_flag);
  } else if (warp >= kLoadWarp && warp < kMmaWarp) {
    // =========================== copies ==========================================
    // A warp owns 32 keys of every tile: lane l knows where key l of them lies.
    if constexpr (G::moves) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::copy_regs));
    const int base_key = (warp - kLoadWarp) * 32;
    const uint32_t ring = tc::smem_u32(smem);
    uint32_t unit = 0, item = 0;
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
        if (warp == kLoadWarp && kv16_held<kHeld>(p, kHeldCopies, unit)) break;
        const bool now = have;
        long long off = 0;
        int64_t head_k = 0;
        if (now) {
          off = keys.offset();
          const int kvh = keys.it.kvh;
          head_k = (int64_t)kvh * p.stride_head;
          const bool first = keys.fresh;
          const int first_token = keys.it.first_token, row0 = keys.it.row0, rows = keys.it.rows;
          have = keys.fetch();
#pragma unroll
          for (int part = 0; part < G::parts; ++part) {
            const uint32_t s = next_unit();
            if (part == 0 && first) {
              // the rows of Q come with the piece's first unit: chunk c of row n at c (RP 16) + n 16
              if (item >= 2) ok &= kv16_wait(&bars[Bars::q_empty + (item & 1)], ((item >> 1) - 1) & 1, abort_flag);
              const uint32_t dst = tc::smem_u32(smem + G::q) + (item & 1) * G::qimage;
              for (int i = tid - kLoadWarp * 32; i < RP * (HD / 8); i += 128) {
                const int n = i / (HD / 8), c = i % (HD / 8);
                int token, head;
                row_of(p, first_token, kvh, row0 + min(n, rows - 1), &token, &head);
                copy16(dst + c * (RP * 16) + n * 16, p.q + (int64_t)token * p.q_stride_token + (int64_t)head * p.q_stride_head + c * 16, n < rows);
              }
              ++item;
            }
            copy_keys<G::dims>(ring + s * G::unit, base_key, p.k + head_k + part * 256, off);
            copies_arrive(&full[s]);
          }
        }
        if (have_v) {
#pragma unroll
          for (int part = 0; part < G::parts; ++part) {
            const uint32_t s = next_unit();
            copy_keys<G::dims>(ring + s * G::unit, base_key, p.v + head_v + part * 256, off_v);
            copies_arrive(&full[s]);
          }
        }
        off_v = off;
        head_v = head_k;
        have_v = now;
      }
    }
    copies_wait_all();
  } else if (warp == kMmaWarp) {
    // =========================== MMAs ============================================
    // QK of a tile is issued ahead of PV of the one before, in the order in which the units arrive.
    constexpr uint32_t fmt = kHalf ? tc::kFmtF16 : tc::kFmtBF16;
    constexpr uint32_t qk_desc = tc::instr_desc(128, G::cols, fmt, fmt, 0, 0);
    constexpr uint32_t pv_desc = tc::instr_desc(128, 2 * RP, fmt, fmt, 1, 1);
    const uint32_t ring = tc::smem_u32(smem), q_s = tc::smem_u32(smem + G::q), p_s = tc::smem_u32(smem + G::p);
    uint32_t unit = 0, tile = 0, item = 0;
    auto arrived = [&]() -> uint32_t {
      const uint32_t s = unit % G::units;
      ok &= kv16_wait(&full[s], (unit / G::units) & 1, abort_flag);
      tc::fence_async_smem();   // (the copies wrote through the generic proxy)
      ++unit;
      return s;
    };
    auto qk = [&](bool last_of_item) {
#pragma unroll
      for (int part = 0; part < G::parts; ++part) {
        const uint32_t s = arrived();
        if (elect_one()) {
          tc::fence_after_sync();
#pragma unroll
          for (int kk = 0; kk < G::dims / 16; ++kk) {
            const uint64_t a = swizzled_desc(ring + s * G::unit + (kk >> 2) * (kTile * 128) + (kk & 3) * 32, 16, 1024);
            const uint64_t b = tc::smem_desc(q_s + (item & 1) * G::qimage + (part * (G::dims / 8) + kk * 2) * (RP * 16), RP * 16, RP == 8 ? 0 : 128);
            tc::mma_ss(tmem_base + G::s_col + (tile & 1) * G::cols, a, b, qk_desc, part > 0 || kk > 0);
          }
          tc::mma_commit(&empty[s]);
          if (part == G::parts - 1) {
            tc::mma_commit(&bars[Bars::s_ready + (tile & 1)]);
            if (last_of_item) tc::mma_commit(&bars[Bars::q_empty + (item & 1)]);
          }
        }
        __syncwarp();
      }
      ++tile;
      if (last_of_item) ++item;
    };
    uint32_t pv_tile = 0;
    auto pv = [&](bool first_of_item) {
      ok &= kv16_wait(&bars[Bars::p_ready], pv_tile & 1, abort_flag);
#pragma unroll
      for (int part = 0; part < G::parts; ++part) {
        const uint32_t s = arrived();
        if (elect_one()) {
          tc::fence_after_sync();
#pragma unroll
          for (int kk = 0; kk < kTile / 16; ++kk) {
            // (64 dims: the instruction's other 64 rows are the same bytes again, which nothing reads)
            const uint64_t a = swizzled_desc(ring + s * G::unit + kk * 2048, HD == 64 ? 0 : kTile * 128, 1024);
            const uint64_t b = tc::smem_desc(p_s + kk * 256, 128, kTile * 16);
            tc::mma_ss(tmem_base + G::o_col + part * 2 * RP, a, b, pv_desc, !first_of_item || kk > 0);
          }
          tc::mma_commit(&empty[s]);
          if (part == G::parts - 1) tc::mma_commit(&bars[Bars::pv_done]);
        }
        __syncwarp();
      }
      ++pv_tile;
    };
    Piece it;
    bool pending = false, pending_first = false;
    while (queue.get(&it, abort_flag)) {
      for (int t = 0; t < it.tiles; ++t) {
        if (kv16_held<kHeld>(p, kHeldMma, tile)) break;
        qk(t == it.tiles - 1);
        if (pending) pv(pending_first);
        pending = true;
        pending_first = t == 0;
      }
    }
    if (pending) pv(pending_first);
  } else if (warp < kLoadWarp) {
    // =========================== softmax =========================================
    if constexpr (G::moves) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::softmax_regs));
    const uint32_t lane_addr = (uint32_t)(warp * 32) << 16;
    float* const wmax = reinterpret_cast<float*>(smem + G::wmax);
    float* const wsum = reinterpret_cast<float*>(smem + G::wsum);
    uint8_t* const p_img = smem + G::p + tid * 16;
    uint32_t tile = 0;
    zero_requests<HD, RP, kSoftmaxThreads>(p);
    {
      const int heads = min(p.num_kv_heads, (int)gridDim.x), hslot = (int)blockIdx.x % heads;
      Piece it;
      while (queue.get(&it, abort_flag)) {
        const int kvh = it.kvh;
        float ref[RP], l[RP];
#pragma unroll
        for (int n = 0; n < RP; ++n) {
          ref[n] = -INFINITY;
          l[n] = 0.f;
        }
        for (int t = 0; t < it.tiles; ++t, ++tile) {
          ok &= kv16_wait(&bars[Bars::s_ready + (tile & 1)], (tile >> 1) & 1, abort_flag);
          tc::fence_after_sync();
          uint32_t sr[RP];
          tmem_load<RP>(tmem_base + G::s_col + (tile & 1) * G::cols + lane_addr, sr);
          tc::tmem_ld_wait<RP>(sr);
          const int pos = it.key0 + t * kTile + tid;
          if (pos < it.lo || pos >= it.hi) {
#pragma unroll
            for (int n = 0; n < RP; ++n) sr[n] = 0xff800000u;  // -inf
          }
          float x[RP];
          bool outgrown = false;
#pragma unroll
          for (int n = 0; n < RP; ++n) {
            x[n] = fmaf(__uint_as_float(sr[n]), p.scale_log2, -ref[n]);
            outgrown |= n < it.rows && !(x[n] <= kGain<kHalf> + kSlack);   // (also where ref is not set yet)
          }
          if (softmax_any(outgrown)) {
#pragma unroll
            for (int n = 0; n < RP; ++n) {
              const float m = redux_max(__uint_as_float(sr[n]));
              if (lane == 0) wmax[warp * RP + n] = m * p.scale_log2;
            }
            softmax_sync();
            float alpha[RP];
            bool moved = false;
#pragma unroll
            for (int n = 0; n < RP; ++n) {
              const float m = fmaxf(fmaxf(wmax[n], wmax[RP + n]), fmaxf(wmax[2 * RP + n], wmax[3 * RP + n])) - kGain<kHalf>;
              const float to = fmaxf(ref[n], m);
              alpha[n] = to == -INFINITY ? 1.f : kv16_exp2(ref[n] - to);
              moved |= alpha[n] != 1.f;
              ref[n] = to;
              l[n] *= alpha[n];
              x[n] = fmaf(__uint_as_float(sr[n]), p.scale_log2, to == -INFINITY ? 0.f : -to);
            }
            if (t > 0 && moved) {   // (the same in all threads)
              ok &= kv16_wait(&bars[Bars::pv_done], (tile - 1) & 1, abort_flag);
              tc::fence_after_sync();
#pragma unroll
              for (int half = 0; half < 2 * G::parts; ++half) {   // hi and lo of every part
                uint32_t o[RP];
                const uint32_t addr = tmem_base + G::o_col + half * RP + lane_addr;
                tmem_load<RP>(addr, o);
                tc::tmem_ld_wait<RP>(o);
#pragma unroll
                for (int n = 0; n < RP; ++n) o[n] = __float_as_uint(weighed(__uint_as_float(o[n]), alpha[n]));
                tmem_store<RP>(addr, o);
              }
              tc::tmem_st_wait();
            }
            softmax_sync();  // (the maxima have been read)
          }
          uint32_t hi[RP / 2], lo[RP / 2];
#pragma unroll
          for (int n = 0; n < RP; n += 2) {
            const float a = kv16_exp2(x[n]), b = kv16_exp2(x[n + 1]);
            l[n] += a;
            l[n + 1] += b;
            split2<kHalf>(a, b, &hi[n / 2], &lo[n / 2]);
          }
          if (tile > 0) ok &= kv16_wait(&bars[Bars::pv_done], (tile - 1) & 1, abort_flag);  // (P of the last tile has been read)
#pragma unroll
          for (int j = 0; j < RP / 8; ++j) {
            *reinterpret_cast<uint4*>(p_img + j * (kTile * 16)) = make_uint4(hi[4 * j], hi[4 * j + 1], hi[4 * j + 2], hi[4 * j + 3]);
            *reinterpret_cast<uint4*>(p_img + (RP / 8 + j) * (kTile * 16)) = make_uint4(lo[4 * j], lo[4 * j + 1], lo[4 * j + 2], lo[4 * j + 3]);
          }
          tc::fence_async_smem();
          tc::fence_before_sync();
          mbar_arrive(&bars[Bars::p_ready]);
        }
        // ---- the piece's rows ----
#pragma unroll
        for (int n = 0; n < RP; ++n) {
          if (n < it.rows) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) l[n] += __shfl_xor_sync(0xffffffffu, l[n], o);
          }
        }
        if (lane == 0) {
#pragma unroll
          for (int n = 0; n < RP; ++n) wsum[warp * RP + n] = l[n];
        }
        softmax_sync();
#pragma unroll
        for (int n = 0; n < RP; ++n) l[n] = (wsum[n] + wsum[RP + n]) + (wsum[2 * RP + n] + wsum[3 * RP + n]);
        ok &= kv16_wait(&bars[Bars::pv_done], (tile - 1) & 1, abort_flag);
        tc::fence_after_sync();
        const bool whole = it.begins && it.ends;
        float* const slot = partial_slot<HD, RP>(p, (int)blockIdx.x, it.begins);
#pragma unroll
        for (int part = 0; part < G::parts; ++part) {
          uint32_t o[2 * RP];
          tmem_load<2 * RP>(tmem_base + G::o_col + part * 2 * RP + lane_addr, o);
          tc::tmem_ld_wait<2 * RP>(o);
          const int d = part * 128 + tid;
          if (d < HD) {
#pragma unroll
            for (int n = 0; n < RP; ++n) {
              if (n < it.rows) {
                const float hi = __uint_as_float(o[n]), v = isinf(hi) ? hi : hi + __uint_as_float(o[RP + n]);
                if (whole) {
                  int token, head;
                  row_of(p, it.first_token, kvh, it.row0 + n, &token, &head);
                  store_out_elem(p.out + (int64_t)token * p.out_stride_token + (int64_t)head * p.out_stride_head, d, kHalf ? PTH_ATTN_F16 : PTH_ATTN_BF16,
                                 l[n] == 0.f ? 0.f : __fdividef(v, l[n]));
                } else {
                  slot[n * HD + d] = v;
                }
              }
            }
          }
        }
        tc::fence_before_sync();
        if (tid == 0) {
#pragma unroll
          for (int n = 0; n < RP; ++n) {
            if (n < it.rows) {
              if (whole) {
                int token, head;
                row_of(p, it.first_token, kvh, it.row0 + n, &token, &head);
                if (p.lse != nullptr)
                  p.lse[(int64_t)token * p.num_q_heads + head] = l[n] == 0.f ? -INFINITY : ((ref[n] == -INFINITY ? 0.f : ref[n]) + log2f(l[n])) * kLn2;
              } else {
                slot[RP * HD + n] = ref[n];
                slot[RP * HD + RP + n] = l[n];
              }
            }
          }
        }
        if (!whole) {
          const int g0 = it.first_cta, g1 = it.last_cta;   // (groups)
          softmax_sync();
          int* const counter = reinterpret_cast<int*>(p.workspace) + g0 * heads + hslot;
          if (tid == 0) {
            *arrival = arrive_at(counter);
            if (*arrival == g1 - g0) *counter = 0;   // (for the next call)
          }
          softmax_sync();
          if (*arrival == g1 - g0) {
            merge_pieces<HD, RP, kHalf>(p, it, kvh, g0, g1 - g0 + 1, heads, hslot);
          }
        }
        softmax_sync();  // (the sums and the arrival have been read)
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    if (*abort_flag) {   // (copies have landed, MMAs may be in flight)
      if (elect_one()) {
        tc::mma_commit(&bars[Bars::drained]);
        kv16_drain(&bars[Bars::drained], 0);
        atomicOr(&g_kv16_status, 8u);
      }
      __syncwarp();
    }
    tc::tmem_dealloc(tmem_base, G::tmem);
  }
  (void)ok;
}

template <int HD, int RP, bool kHalf, bool kHeld = false>
cudaError_t launch_one(const Kv16Params& p, cudaStream_t stream) {
  using G = Geo<HD, RP>;
  static_assert(G::total <= 232448, "shared memory of one CTA");
  static_assert(G::ctas == 1 || G::total <= 115712, "shared memory of two CTAs");
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    err = cudaFuncSetAttribute(kv16_short_kernel<HD, RP, kHalf, kHeld>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::total);
    if (err != cudaSuccess) return err;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int sms = sm_count();
  if (sms <= 0) return cudaErrorInvalidDevice;
  return pdl_launch(kv16_short_kernel<HD, RP, kHalf, kHeld>, dim3((unsigned)(sms * G::ctas)), dim3(kThreads), G::total, stream, p);
}
template <int HD, int RP>
cudaError_t launch_type(const Kv16Params& p, cudaStream_t stream) {
  return p.dtype == PTH_ATTN_F16 ? launch_one<HD, RP, true>(p, stream) : launch_one<HD, RP, false>(p, stream);
}
template <int HD>
cudaError_t launch_rows(const Kv16Params& p, cudaStream_t stream) {
  const int64_t rows = (int64_t)p.max_query_len * p.group;
  if (rows <= 8) return launch_type<HD, 8>(p, stream);
  if (rows <= 16) return launch_type<HD, 16>(p, stream);
  return launch_type<HD, 32>(p, stream);
}

}  // namespace

// Counters, and two partial row tiles per CTA: twice the SMs' number of CTAs with 16 rows, or as many with 32.
int64_t kv16_short_workspace_bytes(int head_size, int num_sms) {
  return kCounterBytes + (int64_t)num_sms * 2 * 2 * 16 * (head_size + 2) * 4;
}

cudaError_t launch_kv16_short(const Kv16Params& p, cudaStream_t stream) {
  switch (p.head_size) {
    case 64:
      return launch_rows<64>(p, stream);
    case 128:
      return launch_rows<128>(p, stream);
    default:
      return launch_rows<256>(p, stream);
  }
}

cudaError_t launch_kv16_short_held(const Kv16Params& p, cudaStream_t stream) { return launch_one<128, 8, false, true>(p, stream); }

// Reads and clears this kernel's status word (device must be idle).
cudaError_t read_kv16_status(unsigned int* v) {
  unsigned int zero = 0;
  cudaError_t err = cudaMemcpyFromSymbol(v, g_kv16_status, sizeof(*v));
  if (err != cudaSuccess) return err;
  return cudaMemcpyToSymbol(g_kv16_status, &zero, sizeof(zero));
}

}  // namespace pthb200
