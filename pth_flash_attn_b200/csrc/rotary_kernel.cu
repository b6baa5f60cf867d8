// Rotary positions: pairs of a head's dimensions turned by position x frequency, queries and keys in one launch.  Bytes bound it: q and
// k are read and written once.
//
// The angle is a product in 64 bits, taken to [-pi, pi] there (a position of 10^6 has 20 bits in front of the point, which 32 bits
// would take from the angle), and its sine and cosine have 32 bits.  A CTA works them out once for a token and all its heads, in
// shared memory.
//
// A thread turns kVec pairs of a head: vectors of 16 bytes where the rows' places allow it, else pair by pair.  Both of a pair are
// read before either is written, so a tensor may be turned in place.
#include "kv8.cuh"

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
  const float r = (float)fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.28318530717958623, a));
  float s, c;
  sincosf(r, &s, &c);
  return make_float2(c * p.scale, (p.inverse ? -s : s) * p.scale);
}

template <int kDtype, bool kInterleaved, bool kVector>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  extern __shared__ float2 turns[];   // [half]
  constexpr int kVec = Vec<kDtype>::n, kSize = kDtype == PTH_ATTN_F32 ? 4 : 2;
  const int token = (int)blockIdx.x, heads = p.heads[0] + p.heads[1], half = p.half;
  pdl_wait();
  const long long position = __ldg(reinterpret_cast<const long long*>(p.positions) + token);
  for (int i = threadIdx.x; i < half; i += kThreads) turns[i] = turn_of(p, position, i);
  __syncthreads();
  // pieces of a head: of its pairs, then of the dimensions that are copied
  const int turning = kVector ? 2 * half / (2 * kVec) : half, copied = kVector ? (p.head_size - 2 * half) / kVec : p.head_size - 2 * half;
  const int per = turning + copied;
  for (int x = threadIdx.x; x < heads * per; x += kThreads) {
    const int h = x / per, i = x - h * per, k = h >= p.heads[0] ? 1 : 0, head = h - (k ? p.heads[0] : 0);
    const uint8_t* const src = p.src[k] + (int64_t)token * p.src_stride_token[k] + (int64_t)head * p.src_stride_head[k];
    uint8_t* const dst = p.dst[k] + (int64_t)token * p.dst_stride_token[k] + (int64_t)head * p.dst_stride_head[k];
    if (i >= turning) {
      if constexpr (kVector) {
        const int at = (2 * half + (i - turning) * kVec) * kSize;
        *reinterpret_cast<uint4*>(dst + at) = *reinterpret_cast<const uint4*>(src + at);
      } else {
        put<kDtype>(dst, 2 * half + i - turning, get<kDtype>(src, 2 * half + i - turning));
      }
    } else if constexpr (kVector) {
      // kVec pairs: 16 bytes of either half, or 32 bytes of pairs side by side
      const int a0 = (kInterleaved ? 2 * i * kVec : i * kVec) * kSize, b0 = kInterleaved ? a0 + 16 : a0 + half * kSize;
      Vec<kDtype> a, b;
      a.load(src + a0);
      b.load(src + b0);
      if constexpr (kInterleaved) {
#pragma unroll
        for (int e = 0; e < kVec / 2; ++e) {
          const float2 t = turns[i * kVec + e], u = turns[i * kVec + kVec / 2 + e];
          const float ax = a.x[2 * e], ay = a.x[2 * e + 1], bx = b.x[2 * e], by = b.x[2 * e + 1];
          a.x[2 * e] = ax * t.x - ay * t.y;
          a.x[2 * e + 1] = ax * t.y + ay * t.x;
          b.x[2 * e] = bx * u.x - by * u.y;
          b.x[2 * e + 1] = bx * u.y + by * u.x;
        }
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float2 t = turns[i * kVec + e];
          const float ax = a.x[e], bx = b.x[e];
          a.x[e] = ax * t.x - bx * t.y;
          b.x[e] = ax * t.y + bx * t.x;
        }
      }
      a.store(dst + a0);
      b.store(dst + b0);
    } else {
      const int ia = kInterleaved ? 2 * i : i, ib = kInterleaved ? 2 * i + 1 : i + half;
      const float2 t = turns[i];
      const float a = get<kDtype>(src, ia), b = get<kDtype>(src, ib);
      put<kDtype>(dst, ia, a * t.x - b * t.y);
      put<kDtype>(dst, ib, a * t.y + b * t.x);
    }
  }
}

template <int kDtype>
cudaError_t launch_for(const RotaryParams& p, bool interleaved, bool vector, cudaStream_t stream) {
  const dim3 grid((unsigned)p.num_tokens);
  const size_t smem = (size_t)p.half * sizeof(float2);
  if (interleaved) return pdl_launch(vector ? rotary_kernel<kDtype, true, true> : rotary_kernel<kDtype, true, false>, grid, kThreads, smem, stream, p);
  return pdl_launch(vector ? rotary_kernel<kDtype, false, true> : rotary_kernel<kDtype, false, false>, grid, kThreads, smem, stream, p);
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
