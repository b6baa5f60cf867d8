// Rotary positions: pairs of a head's dimensions turned by position x frequency, queries and keys in one launch.  Bytes bound it: q and
// k are read and written once.
//
// The angle is a product in 64 bits, taken to [-pi, pi] there (a position of 10^6 has 20 bits in front of the point, which 32 bits
// would take from the angle), and its sine and cosine have 32 bits, near their zeros too: they are those of the angle's rounding to 32 bits, corrected by what
// that left.  A CTA works them out once for a few tokens and all their heads, in shared memory.
//
// A thread turns the pairs of two vectors of 16 bytes at a time where the rows' places allow it, else pair by pair.
// Both of a pair are read before either is written, so a tensor may be turned in place.  8,192 tokens of 32 + 8 heads, 128 dims, bf16, 0.17 GB:
// 33 to 36 us, 0.72 to 0.78 of the copy bandwidth.
#include "kv8.cuh"

#include "page_copy.cuh"
#include "pdl.cuh"

namespace pthb200 {
namespace {

constexpr int kThreads = 256;

struct RotaryParams {
  const uint8_t* src[2];
  uint8_t* dst[2];
  int64_t src_stride_token[2], src_stride_head[2], dst_stride_token[2], dst_stride_head[2];
  int32_t heads[2];
  const int64_t* positions;
  const void* frequencies;
  int32_t frequencies_64, num_tokens, head_size, half, inverse;
  float scale;
};

template <int kDtype>
__device__ __forceinline__ float get(const uint8_t* row, int i) {
  if constexpr (kDtype == PTH_ATTN_F32) return reinterpret_cast<const float*>(row)[i];
  if constexpr (kDtype == PTH_ATTN_F16) return __half2float(reinterpret_cast<const __half*>(row)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[i]);
}
template <int kDtype>
__device__ __forceinline__ void put(uint8_t* row, int i, float x) {
  if constexpr (kDtype == PTH_ATTN_F32) reinterpret_cast<float*>(row)[i] = x;
  else if constexpr (kDtype == PTH_ATTN_F16) reinterpret_cast<__half*>(row)[i] = __float2half_rn(x);
  else reinterpret_cast<__nv_bfloat16*>(row)[i] = __float2bfloat16_rn(x);
}
// The numbers of 16 bytes.
template <int kDtype>
struct Vec {
  static constexpr int n = kDtype == PTH_ATTN_F32 ? 4 : 8;
  float x[n];
  __device__ __forceinline__ void load(const uint8_t* at) {
    const uint4 v = *reinterpret_cast<const uint4*>(at);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kDtype == PTH_ATTN_F32) {
        x[i] = __uint_as_float(w[i]);
      } else if constexpr (kDtype == PTH_ATTN_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      } else {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
  // Turns the pair (this i, y j) by t.
  __device__ __forceinline__ void turn(int i, Vec& y, int j, float2 t) {
    const float u = x[i], v = y.x[j];
    x[i] = u * t.x - v * t.y;
    y.x[j] = u * t.y + v * t.x;
  }
  __device__ __forceinline__ void store(uint8_t* at) const {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kDtype == PTH_ATTN_F32) w[i] = __float_as_uint(x[i]);
      else w[i] = pack16<kDtype == PTH_ATTN_F16>(x[2 * i], x[2 * i + 1]);
    }
    *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// Cosine and sine, times the scale, of pair i of the token at `position`.
__device__ __forceinline__ float2 turn_of(const RotaryParams& p, long long position, int i) {
  const double f = p.frequencies_64 ? __ldg(static_cast<const double*>(p.frequencies) + i) : (double)__ldg(static_cast<const float*>(p.frequencies) + i);
  const double a = (double)position * f;
  // less the nearest multiple of 2 pi (in two parts: the quotient has up to 31 bits)
  const double turns = rint(a * 0.15915494309189533577);
  const double r = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.28318530717958623, a));
  const float near = (float)r, rest = (float)(r - (double)near);
  float sn, cn;
  sincosf(near, &sn, &cn);
  const float s = fmaf(rest, cn, sn), c = fmaf(-rest, sn, cn);
  return make_float2(c * p.scale, (p.inverse ? -s : s) * p.scale);
}

// Where piece x of a CTA's tokens lies: of a head's pairs, then of the dimensions that are copied.
template <int kDtype, bool kInterleaved, bool kVector>
struct Place {
  const uint8_t* src;
  uint8_t* dst;
  int i, turning;      // piece of the head; pieces that turn
  int token;           // of the CTA
  __device__ __forceinline__ Place(const RotaryParams& p, int token0, uint32_t x) {
    constexpr int kVec = Vec<kDtype>::n;
    turning = kVector ? p.half / kVec : p.half;
    const uint32_t per = kVector ? (p.head_size - p.half) / kVec : p.head_size - p.half, heads = p.heads[0] + p.heads[1];
    const uint32_t row = x / per;
    i = (int)(x - row * per);
    token = (int)(row / heads);
    const int h = (int)(row - token * heads), k = h >= p.heads[0] ? 1 : 0, head = h - (k ? p.heads[0] : 0);
    src = p.src[k] + (int64_t)(token0 + token) * p.src_stride_token[k] + (int64_t)head * p.src_stride_head[k];
    dst = p.dst[k] + (int64_t)(token0 + token) * p.dst_stride_token[k] + (int64_t)head * p.dst_stride_head[k];
  }
  // byte offsets of a vector piece's two halves (of a copied one: the same twice)
  __device__ __forceinline__ int2 halves(const RotaryParams& p) const {
    constexpr int kVec = Vec<kDtype>::n, kSize = 16 / kVec;
    if (i >= turning) {
      const int at = (2 * p.half + (i - turning) * kVec) * kSize;
      return make_int2(at, at);
    }
    const int a = (kInterleaved ? 2 * i * kVec : i * kVec) * kSize;
    return make_int2(a, kInterleaved ? a + 16 : a + p.half * kSize);
  }
};

template <int kDtype, bool kInterleaved, bool kVector>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryParams p, int per_cta) {
  extern __shared__ float2 turns[];   // [tokens of the CTA][half]
  constexpr int kVec = Vec<kDtype>::n;
  using At = Place<kDtype, kInterleaved, kVector>;
  const int token0 = (int)blockIdx.x * per_cta, tokens = min(per_cta, p.num_tokens - token0), half = p.half;
  const uint32_t pieces = (uint32_t)tokens * (uint32_t)((p.heads[0] + p.heads[1]) * (kVector ? (p.head_size - half) / kVec : p.head_size - half));
  pdl_wait();
  for (int i = threadIdx.x; i < tokens * half; i += kThreads) {
    const int t = i / half, pair = i - t * half;
    // (vectors: the e-th pairs of all pieces side by side, so that lanes read from banks of their own)
    turns[kVector ? t * half + pair % kVec * (half / kVec) + pair / kVec : i] = turn_of(p, __ldg(reinterpret_cast<const long long*>(p.positions) + token0 + t), pair);
  }
  __syncthreads();
  if constexpr (kVector) {
    const int step = half / kVec;
#pragma unroll 1
    for (uint32_t x = threadIdx.x; x < pieces; x += kThreads) {
      const At at(p, token0, x);
      const int2 to = at.halves(p);
      Vec<kDtype> a, b;
      a.load(at.src + to.x);
      b.load(at.src + to.y);   // (a copied piece twice)
      if (at.i < at.turning) {
        const float2* const t = turns + at.token * half + at.i;
        if constexpr (kInterleaved) {
#pragma unroll
          for (int e = 0; e < kVec / 2; ++e) {
            a.turn(2 * e, a, 2 * e + 1, t[e * step]);
            b.turn(2 * e, b, 2 * e + 1, t[(kVec / 2 + e) * step]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < kVec; ++e) a.turn(e, b, e, t[e * step]);
        }
        b.store(at.dst + to.y);
      }
      a.store(at.dst + to.x);
    }
  } else {
#pragma unroll 1
    for (uint32_t x = threadIdx.x; x < pieces; x += kThreads) {
      const At at(p, token0, x);
      if (at.i >= at.turning) {
        put<kDtype>(at.dst, half + at.i, get<kDtype>(at.src, half + at.i));   // (dimension 2 half + i - half)
        continue;
      }
      const int ia = kInterleaved ? 2 * at.i : at.i, ib = kInterleaved ? 2 * at.i + 1 : at.i + half;
      const float2 t = turns[at.token * half + at.i];
      const float x0 = get<kDtype>(at.src, ia), y0 = get<kDtype>(at.src, ib);
      put<kDtype>(at.dst, ia, x0 * t.x - y0 * t.y);
      put<kDtype>(at.dst, ib, x0 * t.y + y0 * t.x);
    }
  }
}

template <int kDtype>
cudaError_t launch_for(const RotaryParams& p, bool interleaved, bool vector, cudaStream_t stream) {
  // tokens of a CTA: one where there are too few to give every SM several CTAs of four
  const int per_cta = p.num_tokens >= 4 * sm_count() * 4 ? 4 : 1;
  const dim3 grid((unsigned)((p.num_tokens + per_cta - 1) / per_cta));
  const size_t smem = (size_t)per_cta * p.half * sizeof(float2);
  if (interleaved) return pdl_launch(vector ? rotary_kernel<kDtype, true, true> : rotary_kernel<kDtype, true, false>, grid, kThreads, smem, stream, p, per_cta);
  return pdl_launch(vector ? rotary_kernel<kDtype, false, true> : rotary_kernel<kDtype, false, false>, grid, kThreads, smem, stream, p, per_cta);
}

}  // namespace

cudaError_t launch_rotary(const PthB200RotaryArgs& a, cudaStream_t stream) {
  RotaryParams p{};
  p.src[0] = static_cast<const uint8_t*>(a.q);
  p.src[1] = static_cast<const uint8_t*>(a.k);
  p.dst[0] = static_cast<uint8_t*>(a.q_out);
  p.dst[1] = static_cast<uint8_t*>(a.k_out);
  p.src_stride_token[0] = a.q_stride_token;
  p.src_stride_token[1] = a.k_stride_token;
  p.src_stride_head[0] = a.q_stride_head;
  p.src_stride_head[1] = a.k_stride_head;
  p.dst_stride_token[0] = a.q_out_stride_token;
  p.dst_stride_token[1] = a.k_out_stride_token;
  p.dst_stride_head[0] = a.q_out_stride_head;
  p.dst_stride_head[1] = a.k_out_stride_head;
  p.heads[0] = a.num_q_heads;
  p.heads[1] = a.num_k_heads;
  p.positions = a.positions;
  p.frequencies = a.frequencies;
  p.frequencies_64 = a.frequencies_64;
  p.num_tokens = a.num_tokens;
  p.head_size = a.head_size;
  p.half = a.num_frequencies;
  p.inverse = a.inverse;
  p.scale = a.scale;
  // whole vectors: rows on 16-byte boundaries, both halves and the rest multiples of 16 bytes
  const int vec = a.dtype == PTH_ATTN_F32 ? 4 : 8;
  bool vector = a.num_frequencies % vec == 0 && a.head_size % vec == 0;
  for (int k = 0; k < 2; ++k) {
    if (p.heads[k] == 0) continue;
    vector = vector && reinterpret_cast<uintptr_t>(p.src[k]) % 16 == 0 && reinterpret_cast<uintptr_t>(p.dst[k]) % 16 == 0 && p.src_stride_token[k] % 16 == 0 &&
             p.src_stride_head[k] % 16 == 0 && p.dst_stride_token[k] % 16 == 0 && p.dst_stride_head[k] % 16 == 0;
  }
  if (a.dtype == PTH_ATTN_F32) return launch_for<PTH_ATTN_F32>(p, a.interleaved != 0, vector, stream);
  if (a.dtype == PTH_ATTN_F16) return launch_for<PTH_ATTN_F16>(p, a.interleaved != 0, vector, stream);
  return launch_for<PTH_ATTN_BF16>(p, a.interleaved != 0, vector, stream);
}

}  // namespace pthb200
