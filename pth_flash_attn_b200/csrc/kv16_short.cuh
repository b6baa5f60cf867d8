// What the attention kernels with the keys on the MMA's M dimension share (the 16-bit and the 8-bit paged cache): the walk over a
// CTA's run of the sequence of all keys, the softmax warps' barriers, and the merge of a row tile's pieces.
//
// Schedule: the keys of all (request, row tile) form one sequence, which is cut into equal runs, one for every group of Hkv CTAs;
// CTA h of a group reads head h, so that the heads of a page are read at the same time.  The pieces of a row tile that a cut
// divides are merged by the CTA that arrives last: one launch, and the same bits whoever is last.
#pragma once

#include "kv16_sched.cuh"
#include "page_copy.cuh"

namespace pthb200 {
namespace {

constexpr int kSoftmaxThreads = 128;   // warps 0-3: thread t is key t of a tile, then dim t of the output
// The sequence is counted in grains of 32 keys; a row tile counts kPieceGrains more, what its queries and its end take.  (With 0, 4
// and 8, us: 200 requests of up to 500 keys 65.5, 61.4, 61.5; 300 of up to 300 at 256 dims 47.1, 41.0, 38.9; 8 of up to 4,095 32.8,
// 30.7, 30.7; 2,000 of 100 260, 258, 256.  Grains of 128 keys: 4 requests of 500 18.4 instead of 16.4.)
constexpr int kGrain = 32, kPieceGrains = 4;
// Length of a run at least, so that few keys are not spread over pieces that cost more to merge: with 1, 4 and 16, us, one request
// of 2,000 keys 24.6, 18.5, 18.4, four of 500 16.4, 16.4, 18.4.
constexpr int kRunMin = 4;

// Length of a row tile in the sequence: its keys in grains, and what a piece costs besides.
template <class Shape>
__device__ __forceinline__ int row_tile_length(const Shape& s) {
  return s.tiles > 0 ? (s.hi - s.lo / kGrain * kGrain + kGrain - 1) / kGrain + kPieceGrains : 0;
}
// The run of a CTA: a walk over its pieces.
template <int RP, class Params>
struct ShortWalk {
  long long at, end, start;   // position in the sequence, end of the run, start of request r
  int r, kvh;
  long long begin, first_start;   // where the run begins, for further KV heads
  int first_r, heads;
  long long work;             // length of the sequence
  int groups;                 // that it is cut among
  // Group that has position x of the sequence.
  __device__ __forceinline__ int owner(long long x) const { return (int)(((x + 1) * groups - 1) / work); }
  __device__ __forceinline__ bool next(const Params& p, Piece* out) {
    for (;;) {
      if (at >= end) {
        kvh += heads;
        if (begin >= end || kvh >= p.num_kv_heads) return false;
        at = begin;
        start = first_start;
        r = first_r;
      }
      auto s = req_shape<RP>(p, r);
      int n = row_tile_length(s);
      while (at >= start + (long long)n * s.row_tiles) {
        start += (long long)n * s.row_tiles;
        ++r;
        s = req_shape<RP>(p, r);
        n = row_tile_length(s);
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
      place_piece(out, s);
      return true;
    }
  }
};
// Cuts the sequence, of which [before, before + mine) are requests from r0 on.  Returns whether this CTA's run begins among
// them, and where.
template <int RP, class Params>
__device__ __forceinline__ bool begin_run(const Params& p, ShortWalk<RP, Params>& w, int group, int r0, long long before, long long mine, int* r, long long* start) {
  w.groups = (int)min((long long)((int)gridDim.x / w.heads), max(w.work / kRunMin, 1ll));
  w.begin = group < w.groups ? w.work * group / w.groups : 0;
  w.end = group < w.groups ? w.work * (group + 1) / w.groups : 0;
  if (w.begin >= w.end || w.begin < before || w.begin >= before + mine) return false;
  *start = before;
#pragma unroll 1
  for (*r = r0;; ++*r) {
    const auto s = req_shape<RP>(p, *r);
    const long long n = (long long)row_tile_length(s) * s.row_tiles;
    if (w.begin < *start + n) return true;
    *start += n;
  }
}
// Every CTA sums the requests' lengths up for itself, with all its threads (its scheduling warp alone, while the others go
// on: 0.2 us less at 8 and 64 requests, twice the code).  scratch: 64-bit words, warps + 2.
template <int RP, int kThreads, class Params>
__device__ __forceinline__ ShortWalk<RP, Params> find_run(const Params& p, long long* scratch) {
  constexpr int kWarps = kThreads / 32;
  const int tid = threadIdx.x;
  ShortWalk<RP, Params> w;
  w.heads = min(p.num_kv_heads, (int)gridDim.x);   // KV heads that a group reads at the same time
  w.kvh = (int)blockIdx.x % w.heads;
  const int group = (int)blockIdx.x / w.heads;
  const int per = (p.num_reqs + kThreads - 1) / kThreads, r0 = min(p.num_reqs, tid * per), r1 = min(p.num_reqs, r0 + per);
  long long mine = 0;
#pragma unroll 1
  for (int r = r0; r < r1; ++r) {
    const auto s = req_shape<RP>(p, r);
    mine += (long long)row_tile_length(s) * s.row_tiles;
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

template <int HD, int RP>
__device__ __forceinline__ float* partial_slot(const Kv16Params& p, int cta, bool begins) {
  float* base = reinterpret_cast<float*>(p.workspace + kCounterBytes);
  return base + (int64_t)(2 * cta + (begins ? 1 : 0)) * (RP * (HD + 2));  // [RP][HD] O, [RP] ref, [RP] l
}

// Merges the pieces of a row tile, left by the CTAs of groups g0 .. g0 + pieces - 1, and writes its rows: a warp per row, a lane per
// four columns.  The statistics and columns of eight pieces (four at 256 dims) are loaded together; the running sums are rescaled when a later piece has the
// larger ref.
template <int HD, int RP, bool kHalf, int kWarps = 4>
__device__ __forceinline__ void merge_pieces(const Kv16Params& p, const Piece& it, int kvh, int g0, int pieces, int heads, int hslot) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kVec = HD >= 128 ? HD / 128 : 1, kBatch = 8 / kVec;
  const int d0 = (HD == 64 ? lane & 15 : lane) * 4;
#pragma unroll 1
  for (int n = warp; n < it.rows; n += kWarps) {
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

}  // namespace
}  // namespace pthb200
