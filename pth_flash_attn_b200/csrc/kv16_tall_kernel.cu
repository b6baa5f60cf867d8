// Attention over the 16-bit paged cache for requests of many query rows: cross attention of prompts.
//
// Orientation: query rows on the MMA's M dimension, a thread per row in the softmax:
//   S[row, key] = sum_d Q[row, d] K[key, d]       A = Q, B = K as it lies in the cache (K-major), accumulator in TMEM
//   O[row, d]  += sum_key P[row, key] V[key, d]   A = P in TMEM over S, B = V as it lies in the cache (MN-major)
// A CTA owns 256 rows (two MMA row tiles of 128) at 64 and 128 dims, so that every K and V tile serves twice and the tensor core
// works on one row tile while the other's softmax runs; at 256 dims, where O alone takes half of TMEM, 128 rows with
// two S buffers, which do the same for two tiles of keys.
//
// Softmax: ref is a running bound of the row's scores (log2 units) that moves, with l and O rescaled, only when the largest
// score of a tile outgrows it by kSlack; P = 2^(s - ref) is rounded to the cache's type for the MMA (the error of the output
// is sqrt(2) times that of its own rounding), its sum l is not.  P lands in two halves of 64 keys, each of
// which the MMA takes as soon as it is complete.
//
// One warp issues the MMAs.  The two row tiles are two programs (QK of tile i, PV of tile i in halves, ...) that it polls in
// turn: whichever has its operands goes next, so neither waits for the other, and nothing relies on the order in which MMAs on
// different accumulators run.
//
// Copies, schedule and merging of pieces: kv16_sched.cuh, as for the short kernel; a CTA per SM.
#include "kv16_sched.cuh"
#include "page_copy.cuh"
#include "pdl.cuh"
#include "umma_rows.cuh"

namespace pthb200 {

__device__ unsigned int g_kv16_tall_status = 0;

namespace {

constexpr float kGain = 7.f, kSlack = 8.f;
constexpr int kLoadWarps = 4;

template <int HD>
struct Tall {
  static constexpr int rts = HD == 256 ? 1 : 2;      // row tiles of 128 rows
  static constexpr int rows = 128 * rts;
  static constexpr int bufs = HD == 256 ? 2 : 1;     // S buffers of a row tile
  static constexpr int dims = HD < 128 ? HD : 128;   // of a unit
  static constexpr int parts = HD / dims;
  static constexpr int unit = kTile * dims * 2;
  static constexpr int qtile = 128 * HD * 2;         // Q of a row tile: slabs of 64 dims, 128 rows of 128 bytes each
  static constexpr int units = HD == 64 ? 8 : 5;
  static constexpr int softmax_warps = 4 * rts;
  static constexpr int load_warp = softmax_warps, mma_warp = load_warp + kLoadWarps;
  static constexpr int threads = (mma_warp + 1) * 32;
  // Registers: 13 warps start with 128 each (9 with 168), which setmaxnreg moves from the copies to the softmax.
  static constexpr int start_regs = HD == 256 ? 168 : 128, copy_regs = HD == 256 ? 72 : 56, softmax_regs = HD == 256 ? 232 : 160;
  static_assert(softmax_warps * softmax_regs + kLoadWarps * copy_regs + start_regs <= (threads / 32) * start_regs, "a split that the launch holds");
  static constexpr int s_col = 0, o_col = 256;       // S(rt, b) at 128 (rt + b), O(rt) at 256 + rt HD
  // shared memory, behind the first 1,024-byte boundary
  static constexpr int q = units * unit;
  static constexpr int bars = q + rts * qtile;
  static constexpr int n_bars = 2 * units + 2 * rts + 4 * 2 + 2;
  static constexpr int misc = bars + n_bars * 8;
  static constexpr int total = misc + 256 + 1024;
  static_assert(total <= 232448, "shared memory of one CTA");
};
template <int HD>
struct TallBars {  // behind [units] full, [units] empty
  static constexpr int q_full = 0, q_empty = Tall<HD>::rts;
  static constexpr int s_ready = 2 * Tall<HD>::rts;  // [2] S buffer (rt + b)
  static constexpr int p_ready = s_ready + 2;        // [2][2 halves]
  static constexpr int pv_done = p_ready + 4;        // [2]
};

__device__ __forceinline__ bool test_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}\n"
      : "=r"(ok)
      : "r"(tc::smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, bool accumulate) {
  mma_ts_words(d_tmem, a_tmem, (uint32_t)b_desc, (uint32_t)(b_desc >> 32), idesc, accumulate);
}
template <bool kHalf>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (kHalf) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

template <int HD>
__device__ __forceinline__ float* tall_slot(const Kv16Params& p, int cta, bool begins) {
  // [HD][rows] O, [rows] ref, [rows] l
  return reinterpret_cast<float*>(p.workspace + kCounterBytes) + (int64_t)(2 * cta + (begins ? 1 : 0)) * (Tall<HD>::rows * (HD + 2));
}

template <int HD, bool kHalf>
__global__ void __launch_bounds__(Tall<HD>::threads, 1) kv16_tall_kernel(const __grid_constant__ Kv16Params p) {
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
  int* const arrival = reinterpret_cast<int*>(smem + G::misc + 8);
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
      }
      for (int i = 0; i < 2; ++i) {
        tc::mbar_init(&bars[B::s_ready + i], 1);
        tc::mbar_init(&bars[B::p_ready + 2 * i], 128);
        tc::mbar_init(&bars[B::p_ready + 2 * i + 1], 128);
        tc::mbar_init(&bars[B::pv_done + i], 1);
      }
      *abort_flag = 0;
      tc::mbar_init_fence();
    }
    __syncwarp();
    tc::tmem_alloc(tslot, 512);
    tc::tmem_relinquish();
  }
  pdl_wait();
  const Run<RP> run = find_run<RP, G::threads>(p, reinterpret_cast<long long*>(smem + G::misc + 16));
  zero_requests<HD, RP, G::threads>(p);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem_base = *tslot;
  const int heads = run.heads, hslot = run.hslot;
  const bool works = run.start.at < run.start.end;
  bool ok = true;

  if (warp >= G::load_warp && warp < G::mma_warp) {
    // =========================== copies ==========================================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::copy_regs));
    const int base_key = (warp - G::load_warp) * 32;
    const uint32_t ring = tc::smem_u32(smem);
    uint32_t unit = 0;
    uint32_t q_count[G::rts];
#pragma unroll
    for (int i = 0; i < G::rts; ++i) q_count[i] = 0;
    auto load_unit = [&](const uint8_t* src, long long off) {
      const uint32_t s = unit % G::units;
      if (unit >= G::units) ok &= wait_or_abort(&empty[s], ((unit / G::units) - 1) & 1, abort_flag);
      copy_keys<G::dims>(ring + s * G::unit, base_key, src, off);
      copies_arrive(&full[s]);
      ++unit;
    };
    for (int kvh = hslot; kvh < p.num_kv_heads && works; kvh += heads) {
      const uint8_t* kb = p.k + (int64_t)kvh * p.stride_head;
      const uint8_t* vb = p.v + (int64_t)kvh * p.stride_head;
      KeyLookup<RP> keys(p, run.start, base_key + lane);
      bool have = keys.fetch();
      while (have) {
        const long long off = keys.offset();
        const bool first = keys.fresh;
        const int first_token = keys.it.first_token, row0 = keys.it.row0, rows = keys.it.rows;
        have = keys.fetch();
#pragma unroll
        for (int part = 0; part < G::parts; ++part) load_unit(kb + part * 256, off);
        if (first) {
          // the piece's queries, behind its first keys: a row tile's as soon as QK has read the last one's
#pragma unroll
          for (int rt = 0; rt < G::rts; ++rt) {
            if (rows <= rt * 128) continue;
            if (q_count[rt] > 0) ok &= wait_or_abort(&bars[B::q_empty + rt], (q_count[rt] - 1) & 1, abort_flag);
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
        for (int part = 0; part < G::parts; ++part) load_unit(vb + part * 256, off);
      }
    }
    copies_wait_all();
  } else if (warp == G::mma_warp) {
    // =========================== MMAs ============================================
    constexpr uint32_t fmt = kHalf ? tc::kFmtF16 : tc::kFmtBF16;
    constexpr uint32_t qk_desc = tc::instr_desc(128, 128, fmt, fmt, 0, 0);
    constexpr uint32_t pv_desc = tc::instr_desc(128, G::dims, fmt, fmt, 0, 1);
    const uint32_t ring = tc::smem_u32(smem), q_s = tc::smem_u32(smem + G::q);
    // A row tile's program over the pieces of this CTA's run.
    struct Program {
      Walk<RP> w;
      Piece it;
      int kvh, qk, pv, half, tiles;   // next QK and PV of the piece
      bool done, live;
      uint32_t tile0;                 // of the piece in the order of all tiles of the CTA (units of the ring)
      uint32_t s_qk, s_pv;            // live tiles so far: use of the S buffers
      uint32_t q_used;
    };
    Program prog[G::rts];
#pragma unroll
    for (int rt = 0; rt < G::rts; ++rt) {
      prog[rt].w = run.start;
      prog[rt].kvh = hslot;
      prog[rt].qk = prog[rt].pv = prog[rt].half = prog[rt].tiles = 0;
      prog[rt].done = !works;
      prog[rt].live = false;
      prog[rt].tile0 = prog[rt].s_qk = prog[rt].s_pv = prog[rt].q_used = 0;
    }
    auto landed = [&](uint32_t u) { return test_wait(&full[u % G::units], (u / G::units) & 1); };
    // (a row tile without rows frees the units as if it had read them)
    auto pass = [&](uint32_t u) {
      if (elect_one()) {
        for (int part = 0; part < G::parts; ++part) mbar_arrive(&empty[(u + part) % G::units]);
      }
      __syncwarp();
    };
    auto try_qk = [&](Program& g, int rt) -> bool {
      const uint32_t u = (g.tile0 + g.qk) * 2 * G::parts;
      const uint32_t b = rt + g.s_qk % G::bufs, use = g.s_qk / G::bufs;
      if (g.live && g.qk == 0 && !test_wait(&bars[B::q_full + rt], g.q_used & 1)) return false;
      if (g.live && use > 0 && !test_wait(&bars[B::pv_done + b], (use - 1) & 1)) return false;
#pragma unroll
      for (int part = 0; part < G::parts; ++part) {
        if (!landed(u + part)) return false;
      }
      if (!g.live) {
        pass(u);
        ++g.qk;
        return true;
      }
      tc::fence_async_smem();   // (the copies wrote through the generic proxy)
      if (elect_one()) {
        tc::fence_after_sync();
#pragma unroll
        for (int part = 0; part < G::parts; ++part) {
          const uint32_t s = (u + part) % G::units;
#pragma unroll
          for (int kk = 0; kk < G::dims / 16; ++kk) {
            const uint32_t at = (kk >> 2) * (kTile * 128) + (kk & 3) * 32;
            tc::mma_ss(tmem_base + G::s_col + b * 128, swizzled_desc(q_s + rt * G::qtile + part * (2 * kTile * 128) + at, 16, 1024),
                       swizzled_desc(ring + s * G::unit + at, 16, 1024), qk_desc, part > 0 || kk > 0);
          }
          tc::mma_commit(&empty[s]);
        }
        tc::mma_commit(&bars[B::s_ready + b]);
        if (g.qk == g.tiles - 1) tc::mma_commit(&bars[B::q_empty + rt]);
      }
      __syncwarp();
      if (g.qk == 0) ++g.q_used;
      ++g.qk;
      ++g.s_qk;
      return true;
    };
    auto try_pv = [&](Program& g, int rt) -> bool {
      const uint32_t u = (g.tile0 + g.pv) * 2 * G::parts + G::parts;
      const uint32_t b = rt + g.s_pv % G::bufs, use = g.s_pv / G::bufs;
      if (g.live && !test_wait(&bars[B::p_ready + 2 * b + g.half], use & 1)) return false;
#pragma unroll
      for (int part = 0; part < G::parts; ++part) {
        if (!landed(u + part)) return false;
      }
      if (!g.live) {
        pass(u);
        ++g.pv;
        return true;
      }
      tc::fence_async_smem();
      if (elect_one()) {
        tc::fence_after_sync();
#pragma unroll
        for (int part = 0; part < G::parts; ++part) {
          const uint32_t s = (u + part) % G::units;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_ts(tmem_base + G::o_col + rt * HD + part * 128, tmem_base + G::s_col + b * 128 + g.half * 32 + kk * 8,
                   swizzled_desc(ring + s * G::unit + (g.half * 4 + kk) * 2048, kTile * 128, 1024), pv_desc, g.pv > 0 || g.half > 0 || kk > 0);
          if (g.half == 1) tc::mma_commit(&empty[s]);
        }
        if (g.half == 1) tc::mma_commit(&bars[B::pv_done + b]);
      }
      __syncwarp();
      g.half ^= 1;
      if (g.half == 0) {
        ++g.pv;
        ++g.s_pv;
      }
      return true;
    };
    auto step = [&](Program& g, int rt) -> bool {
      if (g.pv == g.tiles) {   // next piece
        g.tile0 += (uint32_t)g.tiles;
        while (!next_piece<RP>(p, g.w, &g.it)) {
          g.kvh += heads;
          if (g.kvh >= p.num_kv_heads) {
            g.done = true;
            return true;
          }
          g.w = run.start;
        }
        g.tiles = g.it.tiles;
        g.qk = g.pv = g.half = 0;
        g.live = g.it.rows > rt * 128;
        return true;
      }
      if (g.qk < g.tiles && g.qk < g.pv + G::bufs && try_qk(g, rt)) return true;
      return g.pv < g.qk && try_pv(g, rt);
    };
    long long deadline = clock64() + (1ll << 32);
    uint32_t idle = 0;
    for (;;) {
      bool all_done = true, moved = false;
#pragma unroll
      for (int rt = 0; rt < G::rts; ++rt) {
        if (prog[rt].done) continue;
        all_done = false;
        moved |= step(prog[rt], rt);
      }
      if (all_done) break;
      if (moved) {
        idle = 0;
      } else if ((++idle & 1023u) == 0) {
        if (idle == 1024u) deadline = clock64() + (1ll << 32);
        if (*abort_flag || clock64() > deadline) {
          *abort_flag = 1;
          ok = false;
          break;
        }
      }
    }
    __syncwarp();
  } else {
    // =========================== softmax =========================================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::softmax_regs));
    const int rt = warp >> 2;
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_tmem = tmem_base + G::o_col + rt * HD + lane_addr;
    const int row = tid;   // of the CTA's rows
    uint32_t count = 0;    // live tiles so far
    auto rt_sync = [&] { named_barrier(1 + rt, 128); };
    for (int kvh = hslot; kvh < p.num_kv_heads && works; kvh += heads) {
      Walk<RP> w = run.start;
      Piece it;
      while (next_piece<RP>(p, w, &it)) {
        if (it.rows <= rt * 128) continue;
        const bool padding = (row & ~31) >= it.rows;   // (of the whole warp)
        float ref = -INFINITY, l = 0.f;
        for (int t = 0; t < it.tiles; ++t, ++count) {
          const uint32_t b = rt + count % G::bufs, use = count / G::bufs;
          const uint32_t s_tmem = tmem_base + G::s_col + b * 128 + lane_addr;
          ok &= wait_or_abort(&bars[B::s_ready + b], use & 1, abort_flag);
          if (padding) {   // (the order of the waits is kept, nothing is computed)
            mbar_arrive(&bars[B::p_ready + 2 * b]);
            mbar_arrive(&bars[B::p_ready + 2 * b + 1]);
            continue;
          }
          tc::fence_after_sync();
          uint32_t r[128];
#pragma unroll
          for (int c = 0; c < 4; ++c) tc::tmem_ld32(s_tmem + c * 32, r + c * 32);
          tc::tmem_ld_wait<128>(r);
          const int key0 = it.key0 + t * kTile;
          if (key0 < it.lo || key0 + kTile > it.hi) {
#pragma unroll
            for (int n = 0; n < 128; ++n)
              if (key0 + n < it.lo || key0 + n >= it.hi) r[n] = 0xff800000u;  // -inf
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int n = 0; n < 128; n += 8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(r[n + 2 * e]), __uint_as_float(r[n + 2 * e + 1]));
          }
          const float top = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * p.scale_log2 - kGain;
          const bool need = !(top <= ref + kSlack);   // (also where ref is not set yet)
          if (__any_sync(0xffffffffu, need)) {
            const float to = need ? fmaxf(ref, top) : ref;
            const float alpha = to == -INFINITY ? 1.f : ex2f(ref - to);
            ref = to;
            l *= alpha;
            if (t > 0) {
              const uint32_t b1 = rt + (count - 1) % G::bufs, use1 = (count - 1) / G::bufs;
              ok &= wait_or_abort(&bars[B::pv_done + b1], use1 & 1, abort_flag);
              tc::fence_after_sync();
#pragma unroll 1
              for (int c = 0; c < HD / 16; ++c) {
                uint32_t o[16];
                tc::tmem_ld16(o_tmem + c * 16, o);
                tc::tmem_ld_wait<16>(o);
#pragma unroll
                for (int n = 0; n < 16; ++n) o[n] = __float_as_uint(__uint_as_float(o[n]) * alpha);
                tc::tmem_st16(o_tmem + c * 16, o);
              }
              tc::tmem_st_wait();
            }
          }
          const float use_ref = ref == -INFINITY ? 0.f : -ref;
          const f32x2 scale2 = pair(p.scale_log2, p.scale_log2), ref2 = pair(use_ref, use_ref);
          f32x2 sum[2] = {0ull, 0ull};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int n = 0; n < 16; ++n) {
              float x, y;
              unpair(fma2(pair(__uint_as_float(r[c * 32 + 2 * n]), __uint_as_float(r[c * 32 + 2 * n + 1])), scale2, ref2), x, y);
              x = ex2f(x);
              y = ex2f(y);
              sum[n & 1] = add2(sum[n & 1], pair(x, y));
              pk[n] = pack16<kHalf>(x, y);
            }
            tc::tmem_st16(s_tmem + c * 16, pk);
            if (c & 1) {
              tc::tmem_st_wait();
              tc::fence_before_sync();
              mbar_arrive(&bars[B::p_ready + 2 * b + (c >> 1)]);
            }
          }
          l += sum_pairs(sum);
        }
        // ---- the piece's rows ----
        {
          const uint32_t b1 = rt + (count - 1) % G::bufs, use1 = (count - 1) / G::bufs;
          ok &= wait_or_abort(&bars[B::pv_done + b1], use1 & 1, abort_flag);
          tc::fence_after_sync();
        }
        const bool whole = it.begins && it.ends, live = row < it.rows;
        int token, head;
        row_of(p, it.first_token, kvh, it.row0 + min(row, it.rows - 1), &token, &head);
        uint8_t* const out = p.out + (int64_t)token * p.out_stride_token + (int64_t)head * p.out_stride_head;
        float* const lse = p.lse != nullptr ? p.lse + (int64_t)token * p.num_q_heads + head : nullptr;
        auto write32 = [&](const float* o, int d0) {   // 32 columns of the row
#pragma unroll
          for (int c = 0; c < 4; ++c)
            *reinterpret_cast<uint4*>(out + (d0 + c * 8) * 2) =
                make_uint4(pack16<kHalf>(o[c * 8], o[c * 8 + 1]), pack16<kHalf>(o[c * 8 + 2], o[c * 8 + 3]),
                           pack16<kHalf>(o[c * 8 + 4], o[c * 8 + 5]), pack16<kHalf>(o[c * 8 + 6], o[c * 8 + 7]));
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
              if (live) write32(o, c * 32);
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
          const int g0 = run.owner(it.start), g1 = run.owner(it.start + it.row_tiles_keys - 1);
          __threadfence();
          rt_sync();
          int* const counter = reinterpret_cast<int*>(p.workspace) + 2 * (g0 * heads + hslot) + rt;
          if ((tid & 127) == 0) arrival[rt] = atomicAdd(counter, 1);
          rt_sync();
          if (arrival[rt] == g1 - g0) {
            __threadfence();
            if ((tid & 127) == 0) *counter = 0;   // (for the next call)
            const int pieces = g1 - g0 + 1;
            auto slot = [&](int k) { return tall_slot<HD>(p, (g0 + k) * heads + hslot, k == 0) + row; };
            float top = -INFINITY, sum = 0.f;
            for (int k = 0; k < pieces; ++k) top = fmaxf(top, __ldcg(slot(k) + HD * RP));
            const float use = top == -INFINITY ? 0.f : top;
            for (int k = 0; k < pieces; ++k) {
              const float* s = slot(k) + HD * RP;
              sum = fmaf(ex2f(__ldcg(s) - use), __ldcg(s + RP), sum);
            }
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            if (!padding) {
#pragma unroll 1
              for (int c = 0; c < HD / 32; ++c) {
                float o[32];
#pragma unroll
                for (int n = 0; n < 32; ++n) o[n] = 0.f;
#pragma unroll 1
                for (int k = 0; k < pieces; ++k) {
                  const float* s = slot(k);
                  const float f = ex2f(__ldcg(s + HD * RP) - use);
                  float v[32];
#pragma unroll
                  for (int n = 0; n < 32; ++n) v[n] = __ldcg(s + (c * 32 + n) * RP);
#pragma unroll
                  for (int n = 0; n < 32; ++n) o[n] = fmaf(f, v[n], o[n]);
                }
#pragma unroll
                for (int n = 0; n < 32; ++n) o[n] *= inv;
                if (live) write32(o, c * 32);
              }
              if (live && lse != nullptr) *lse = sum == 0.f ? -INFINITY : (use + log2f(sum)) * kLn2;
            }
          }
          rt_sync();   // (the arrival has been read)
        }
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == G::mma_warp) tc::tmem_dealloc(tmem_base, 512);
  if (tid == 0 && *abort_flag) atomicOr(&g_kv16_tall_status, 16u);
  (void)ok;
}

template <int HD, bool kHalf>
cudaError_t launch_one(const Kv16Params& p, cudaStream_t stream) {
  using G = Tall<HD>;
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    err = cudaFuncSetAttribute(kv16_tall_kernel<HD, kHalf>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::total);
    if (err != cudaSuccess) return err;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int sms = sm_count();
  if (sms <= 0) return cudaErrorInvalidDevice;
  return pdl_launch(kv16_tall_kernel<HD, kHalf>, dim3((unsigned)sms), dim3(G::threads), G::total, stream, p);
}
template <int HD>
cudaError_t launch_type(const Kv16Params& p, cudaStream_t stream) {
  return p.dtype == PTH_ATTN_F16 ? launch_one<HD, true>(p, stream) : launch_one<HD, false>(p, stream);
}

}  // namespace

// Counters, and two partial row tiles per CTA.
int64_t kv16_tall_workspace_bytes(int head_size, int num_sms) {
  const int64_t rows = head_size == 256 ? 128 : 256;
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

// Reads and clears this kernel's status word (device must be idle).
cudaError_t read_kv16_tall_status(unsigned int* v) {
  unsigned int zero = 0;
  cudaError_t err = cudaMemcpyFromSymbol(v, g_kv16_tall_status, sizeof(*v));
  if (err != cudaSuccess) return err;
  return cudaMemcpyToSymbol(g_kv16_tall_status, &zero, sizeof(zero));
}

}  // namespace pthb200
