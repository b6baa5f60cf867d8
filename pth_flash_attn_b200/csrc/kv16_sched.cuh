// What the attention kernels of the 16-bit paged cache share: the pieces they work in, and how keys get to shared memory.
//
// A request's query rows (a row is a query token and head of one KV head, token-major) are cut into row tiles of RP; a row tile
// reads all KV tiles (128 keys) that the request sees.  A row tile that the schedule divides is computed in pieces, runs of
// its KV tiles, by several CTAs; they leave partial results in the workspace, each CTA in a slot for the piece that begins a
// row tile or in one for a piece that goes on with one, and count their arrivals on a counter of the CTA that holds the
// first piece.  The last to arrive merges them, in the pieces' order.
#pragma once

#include <climits>

#include "kv16.cuh"

namespace pthb200 {
namespace {

constexpr int kTile = 128;             // keys
constexpr int kCounterBytes = 4096;    // arrival counters at the start of the workspace, one per CTA

// 2^kGain is P of a row's largest score when its reference is set; scores that come later take P further up, by 2^8 at most.  fp16:
// P, and the second half of a P in two halves, stay within its numbers, 2^-24 .. 65,504.  bf16 has the exponents of the 32-bit
// sums: P is at most 2^-16, so that P times values of any size, summed over 65,536 keys, stays below 2^128 as the result does.
// (On the other side a product below 2^-126 may be lost: 2^-102 of the output.)
template <bool kHalf>
constexpr float kGain = kHalf ? 7.f : -24.f;

// One piece of a row tile: the keys [lo, hi) from key0 on, in `tiles` KV tiles.
struct Piece {
  int r, kvh;
  int row0, rows;             // rows row0 .. row0 + rows of the request's q_len x G
  int first_token;
  int key0, tiles, lo, hi;
  int begins, ends;           // the row tile's first piece, its last
  int first_cta, last_cta;    // that have its pieces (in the counting of the kernel's schedule)
  int sparse;                 // CTAs between them may have none
  int pos0;                   // position of the request's first query token (8-bit cache)
  int edges;                  // its steps at either end that some rows do not see whole (kv8_tall_kernel.cu)
};
static_assert(sizeof(Piece) == 64, "queue entry");

// The pieces of a CTA go from the warp that works them out to the others through a queue in shared memory, so the others
// neither carry the schedule's state nor wait for the lengths it reads.  An entry without tiles ends it.
//
// All warps take the same pieces, also when a wait of the CTA gives up: lanes shuffle and warps share named barriers, so one that
// left while another found its piece would be waited for without end.  Therefore the scheduling warp alone ends the queue: where
// its own wait gives up, or another has, it names the first piece that it has not entered, and an entry is not overwritten
// before all have read it.  Its waits are bounded, and with them those for an entry.
constexpr int kQueue = 4;
constexpr uint32_t kPieceTimes = 16;   // (of the bound on other waits)
struct PieceQueue {
  Piece* entry;      // [kQueue]
  uint64_t* full;    // [kQueue]: one arrival
  uint64_t* empty;   // [kQueue]: one per reading warp
  volatile int* stop;   // pieces that there are, once that is decided before the end
  uint32_t i = 0;
  __device__ __forceinline__ PieceQueue(Piece* entries, uint64_t* bars, int* stop_at) : entry(entries), full(bars), empty(bars + kQueue), stop(stop_at) {}
  __device__ __forceinline__ void init(int readers) {
    *stop = INT_MAX;
    for (int k = 0; k < kQueue; ++k) {
      tc::mbar_init(&full[k], 1);
      tc::mbar_init(&empty[k], readers);
    }
  }
  __device__ __forceinline__ bool put(const Piece& x, volatile int* abort_flag) {
    const uint32_t k = i % kQueue;
    if (!__all_sync(0xffffffffu, *abort_flag == 0 && (i < kQueue || kv16_wait<kPieceTimes>(&empty[k], ((i / kQueue) - 1) & 1, abort_flag)))) {
      if ((threadIdx.x & 31) == 0) *stop = (int)i;
      return false;
    }
    if ((threadIdx.x & 31) == 0) {
      entry[k] = x;
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::smem_u32(&full[k])) : "memory");
    }
    __syncwarp();
    ++i;
    return true;
  }
  // The entry that get takes next, if it is there already.
  __device__ __forceinline__ bool peek(Piece* x) const {
    const uint32_t k = i % kQueue;
    if (!__all_sync(0xffffffffu, tc::mbar_test_wait(&full[k], (i / kQueue) & 1))) return false;
    *x = entry[k];
    return x->tiles > 0;
  }
  __device__ __forceinline__ bool get(Piece* x, volatile int* abort_flag) {
    const uint32_t k = i % kQueue;
    if (!tc::mbar_test_wait(&full[k], (i / kQueue) & 1)) {
#pragma unroll 1
      for (uint32_t n = 0; !tc::mbar_try_wait_hint(&full[k], (i / kQueue) & 1, 1000u); ++n) {
        if (*stop <= (int)i || n == 2 * kPieceTimes * kWaitTries) return false;
        if (n == kPieceTimes * kWaitTries) *abort_flag = 1;
      }
    }
    *x = entry[k];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::smem_u32(&empty[k])) : "memory");
    ++i;
    return x->tiles > 0;
  }
};

// The scheduling warp: the pieces of `walk`, and the end.  never: a barrier that nothing arrives on.
template <bool kHeld, class Params, class Walk>
__device__ __forceinline__ void put_pieces(const Params& p, Walk& walk, PieceQueue& queue, uint64_t* never, volatile int* abort_flag) {
  Piece it;
  while (walk.next(p, &it)) {
    if (kv16_held<kHeld>(p, kHeldSchedule, queue.i)) kv16_wait(never, 0, abort_flag);
    if (!queue.put(it, abort_flag)) return;
  }
  it.tiles = 0;
  queue.put(it, abort_flag);
}

struct ReqShape {
  int tokens, first, lo, hi, tiles, row_tiles;
};
template <int RP>
__device__ __forceinline__ ReqShape req_shape(const Kv16Params& p, int r) {
  ReqShape s;
  kv16_visible(p, r, &s.lo, &s.hi);
  s.tokens = kv16_tokens(p, r, &s.first);
  const int rows = s.tokens * p.group;
  s.row_tiles = (rows + RP - 1) / RP;
  s.tiles = s.hi > s.lo && rows > 0 ? (s.hi + kTile - 1) / kTile - s.lo / kTile : 0;
  return s;
}
// What a walk says of a piece besides: nothing here.
__device__ __forceinline__ void place_piece(Piece*, const ReqShape&) {}
// Counts an arrival behind everything that this CTA's threads have written in front of a barrier that this thread has passed,
// and ahead of what they read behind the next one: the partial results of all who arrived before.
__device__ __forceinline__ int arrive_at(int* counter) {
  int before;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
  return before;
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
// Token and query head of a row of a request.
__device__ __forceinline__ void row_of(const Kv16Params& p, int first_token, int kvh, int row, int* token, int* head) {
  const int t = p.query_start_loc == nullptr ? 0 : (int)((uint32_t)row / (uint32_t)p.group);
  *token = first_token + t;
  *head = kvh * p.group + row - t * p.group;
}

__device__ __forceinline__ float redux_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

// Sum of `mine` over the threads in front of this one, and over all of them.  scratch: a 64-bit word per warp, free again
// behind the caller's next barrier.
template <int kThreads>
__device__ __forceinline__ long long scan_threads(long long mine, long long* scratch, long long* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) scratch[warp] = upto;
  __syncthreads();
  long long before = upto - mine;
  *total = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += scratch[w];
    *total += scratch[w];
  }
  return before;
}

// Rows of requests without a visible key: zero, -inf.
template <int HD, int RP, int kThreads, class Params>
__device__ __forceinline__ void zero_requests(const Params& p) {
  for (int r = (int)blockIdx.x; r < p.num_reqs; r += (int)gridDim.x) {
    const auto s = req_shape<RP>(p, r);
    if (s.tiles > 0 || s.tokens == 0) continue;
#pragma unroll 1
    for (int64_t i = threadIdx.x; i < (int64_t)s.tokens * p.num_q_heads * (HD / 8); i += kThreads) {
      const int64_t row = i / (HD / 8);
      const int token = s.first + (int)(row / p.num_q_heads), head = (int)(row % p.num_q_heads), c = (int)(i % (HD / 8));
      *reinterpret_cast<uint4*>(p.out + (int64_t)token * p.out_stride_token + (int64_t)head * p.out_stride_head + c * 16) = make_uint4(0u, 0u, 0u, 0u);
      if (c == 0 && p.lse != nullptr) p.lse[(int64_t)token * p.num_q_heads + head] = -INFINITY;
    }
  }
}

// The KV tiles of a CTA's pieces, one after the other, for the lane of a copying warp that looks key `key` of every tile up in
// the block table.  The entry of the next tile is on its way while the copies of this one are issued.
struct KeyLookup {
  const Kv16Params& p;
  PieceQueue queue;
  volatile int* abort_flag;
  Piece it;            // of the tile looked up last
  int key, left = 0, key0 = 0, blk = -1, slot = 0;
  bool fresh = false;  // the tile is its piece's first
  __device__ __forceinline__ KeyLookup(const Kv16Params& params, const PieceQueue& q, volatile int* abort, int lane_key)
      : p(params), queue(q), abort_flag(abort), key(lane_key) {}
  __device__ __forceinline__ bool fetch() {
    fresh = left == 0;
    if (fresh) {
      if (!queue.get(&it, abort_flag)) return false;
      left = it.tiles;
      key0 = it.key0;
    } else {
      key0 += kTile;
    }
    --left;
    const int pos = key0 + key;
    blk = -1;
    if (pos >= it.lo && pos < it.hi) {
      int page;
      if (p.block_shift >= 0) {
        page = pos >> p.block_shift;
        slot = pos & (p.block_size - 1);
      } else {
        page = (int)((uint32_t)pos / (uint32_t)p.block_size);
        slot = pos - page * p.block_size;
      }
      blk = __ldg(p.block_table + (int64_t)it.r * p.block_table_row_stride + page);
      if ((uint32_t)blk >= (uint32_t)p.num_blocks) blk = -1;
    }
    return true;
  }
  // Byte offset of the key's row inside a KV head's stream; -1: there is none to read.
  __device__ __forceinline__ long long offset() const { return blk >= 0 ? (long long)blk * p.stride_block + (long long)slot * p.stride_slot : -1ll; }
};

// The 32 keys of a warp, from `base_key` of a tile on: rows of `kDims` dims from off (the lane's key's) into a swizzled unit.
template <int kDims>
__device__ __forceinline__ void copy_keys(uint32_t unit, int base_key, const uint8_t* src, long long off) {
  constexpr int kChunks = kDims / 8, kRows = 32 / kChunks;   // 16-byte chunks of a row, rows at a time
  const int lane = threadIdx.x & 31, chunk = lane % kChunks, sub = lane / kChunks;
  const uint32_t dst = unit + (chunk >> 3) * (kTile * 128) + base_key * 128;
#pragma unroll
  for (int i = 0; i < 32 / kRows; ++i) {
    const int row = i * kRows + sub;
    const long long o = __shfl_sync(0xffffffffu, off, row);
    copy16(dst + row * 128 + (((chunk & 7) ^ (row & 7)) << 4), o >= 0 ? src + o + chunk * 16 : src, o >= 0);
  }
}

}  // namespace
}  // namespace pthb200
