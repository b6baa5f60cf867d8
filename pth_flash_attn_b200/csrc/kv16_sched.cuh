// Schedule of the attention kernels of the 16-bit paged cache.
//
// A request's query rows (a row is a query token and head of one KV head, token-major) are cut into row tiles of RP; a row tile
// reads all KV tiles (128 keys) that the request sees.  The tiles of all (request, row tile) form one sequence, which
// is cut into equal runs, one for every group of Hkv CTAs; CTA h of a group reads KV head h, so that the heads of a page
// are read at the same time.  A row tile that a cut divides is computed in pieces by the CTAs of neighbouring groups;
// they leave partial results in the workspace, a slot of the CTA for the piece that begins a row tile and one for the piece
// that goes on with one, and count their arrivals on the counter of the CTA that holds the first piece.
#pragma once

#include "kv16.cuh"

namespace pthb200 {
namespace {

constexpr int kTile = 128;             // keys
constexpr int kCounterBytes = 4096;    // arrival counters at the start of the workspace, one per CTA
constexpr int kRunMin = 1;             // KV tiles a run holds at least

// One piece of a request's row tile: keys [key0, key0 + 128 tiles) of those visible, [lo, hi).
struct Piece {
  int r, row0, rows;          // rows row0 .. row0 + rows of the request's q_len x G
  int first_token;
  int key0, tiles, lo, hi;
  bool begins, ends;
  long long start;            // of the row tile in the sequence
  int row_tiles_keys;         // KV tiles of the whole row tile
};

template <int RP>
struct Walk {
  long long at, end, start;   // position in the sequence, end of the run, start of request r
  int r;
};

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
template <int RP>
__device__ __forceinline__ bool next_piece(const Kv16Params& p, Walk<RP>& w, Piece* out) {
  if (w.at >= w.end) return false;
  ReqShape s = req_shape<RP>(p, w.r);
  long long n = (long long)s.tiles * s.row_tiles;
  while (w.at >= w.start + n) {
    w.start += n;
    ++w.r;
    s = req_shape<RP>(p, w.r);
    n = (long long)s.tiles * s.row_tiles;
  }
  const long long off = w.at - w.start;
  const int rt = s.row_tiles == 1 ? 0 : (int)(off / s.tiles);
  const int tile = (int)(off - (long long)rt * s.tiles);
  out->r = w.r;
  out->row0 = rt * RP;
  out->rows = min(RP, s.tokens * p.group - rt * RP);
  out->first_token = s.first;
  out->lo = s.lo;
  out->hi = s.hi;
  out->key0 = (s.lo / kTile + tile) * kTile;
  out->tiles = (int)min((long long)(s.tiles - tile), w.end - w.at);
  out->begins = tile == 0;
  out->ends = tile + out->tiles == s.tiles;
  out->start = w.start + (long long)rt * s.tiles;
  out->row_tiles_keys = s.tiles;
  w.at += out->tiles;
  return true;
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

// The run of a CTA, and what the pieces' owners are found with: tile x of the sequence belongs to group
// ((x + 1) groups - 1) / work.
template <int RP>
struct Run {
  Walk<RP> start;       // at == end: the CTA has none
  long long work;       // tiles of the sequence
  int groups, heads, hslot;
  __device__ __forceinline__ int owner(long long x) const { return (int)(((x + 1) * groups - 1) / work); }
};
// Every CTA sums the tiles of all requests up for itself.  scratch: 64-bit words, warps + 2.  Ends with a CTA barrier in front
// of which the first piece's request is written.
template <int RP, int kThreads>
__device__ __forceinline__ Run<RP> find_run(const Kv16Params& p, long long* scratch) {
  constexpr int kWarps = kThreads / 32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  Run<RP> run;
  run.heads = min(p.num_kv_heads, (int)gridDim.x);   // KV heads that a group reads at the same time
  run.hslot = (int)blockIdx.x % run.heads;
  const int group = (int)blockIdx.x / run.heads;
  const int per = (p.num_reqs + kThreads - 1) / kThreads, r0 = min(p.num_reqs, tid * per), r1 = min(p.num_reqs, r0 + per);
  long long mine = 0;
  for (int r = r0; r < r1; ++r) {
    const ReqShape s = req_shape<RP>(p, r);
    mine += (long long)s.tiles * s.row_tiles;
  }
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) scratch[warp] = upto;
  __syncthreads();
  long long before = upto - mine;
  run.work = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += scratch[w];
    run.work += scratch[w];
  }
  const long long most = run.work / kRunMin > 0 ? run.work / kRunMin : 1;
  run.groups = (int)min((long long)((int)gridDim.x / run.heads), most);
  run.start.at = group < run.groups ? run.work * group / run.groups : 0;
  run.start.end = group < run.groups ? run.work * (group + 1) / run.groups : 0;
  if (run.start.at < run.start.end && before <= run.start.at && run.start.at < before + mine) {
    long long start = before;
    int r = r0;
    for (;; ++r) {
      const ReqShape s = req_shape<RP>(p, r);
      const long long n = (long long)s.tiles * s.row_tiles;
      if (run.start.at < start + n) break;
      start += n;
    }
    scratch[kWarps] = r;
    scratch[kWarps + 1] = start;
  }
  __syncthreads();
  const bool works = run.start.at < run.start.end;
  run.start.r = works ? (int)scratch[kWarps] : 0;
  run.start.start = works ? scratch[kWarps + 1] : 0;
  return run;
}

// Rows of requests without a visible key: zero, -inf.
template <int HD, int RP, int kThreads>
__device__ __forceinline__ void zero_requests(const Kv16Params& p) {
  for (int r = (int)blockIdx.x; r < p.num_reqs; r += (int)gridDim.x) {
    const ReqShape s = req_shape<RP>(p, r);
    if (s.tiles > 0 || s.tokens == 0) continue;
    for (int64_t i = threadIdx.x; i < (int64_t)s.tokens * p.num_q_heads * (HD / 8); i += kThreads) {
      const int64_t row = i / (HD / 8);
      const int token = s.first + (int)(row / p.num_q_heads), head = (int)(row % p.num_q_heads), c = (int)(i % (HD / 8));
      *reinterpret_cast<uint4*>(p.out + (int64_t)token * p.out_stride_token + (int64_t)head * p.out_stride_head + c * 16) = make_uint4(0u, 0u, 0u, 0u);
      if (c == 0 && p.lse != nullptr) p.lse[(int64_t)token * p.num_q_heads + head] = -INFINITY;
    }
  }
}

// Tiles of a run, one after the other, for the lane of a copying warp that looks key `key` of every tile up in the block
// table.  The entry of the next tile is on its way while the copies of this one are issued.
template <int RP>
struct KeyLookup {
  const Kv16Params& p;
  Walk<RP> w;
  Piece it;            // of the tile looked up last
  int key, left = 0, key0 = 0, blk = -1, slot = 0;
  bool fresh = false;  // the tile is its piece's first
  __device__ __forceinline__ KeyLookup(const Kv16Params& params, const Walk<RP>& walk, int lane_key) : p(params), w(walk), key(lane_key) {}
  __device__ __forceinline__ bool fetch() {
    fresh = left == 0;
    if (fresh) {
      if (!next_piece<RP>(p, w, &it)) return false;
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
    }
    return true;
  }
  // Byte offset of the key's row inside a KV head's stream; -1: the request does not see the key.
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
