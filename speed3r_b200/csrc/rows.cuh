// Rows of fp32, bf16 or fp16 elements: vectors of W elements (all of them begin at a multiple of their own size), their
// conversion, and sums over the threads that share a row.  The type is an argument, the same for the whole grid: a branch on
// it costs nothing next to a load, and one kernel serves all combinations of types.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace s3r {

__host__ __device__ constexpr int type_bytes(int type) { return type == S3R_F32 ? 4 : 2; }
inline bool known_type(int type) { return type == S3R_F32 || type == S3R_BF16 || type == S3R_F16; }

// The largest vector that rows of `channels` elements at these addresses can be read in: 8, 4 or 1 elements (fp32 vectors of 8
// are two loads of 16 bytes).
inline int row_vector(int channels, const void* const* pointers, const int* types, int n) {
  int w = channels % 8 == 0 ? 8 : channels % 4 == 0 ? 4 : 1;
  for (int i = 0; i < n; ++i)
    while (w > 1 && pointers[i] && reinterpret_cast<uintptr_t>(pointers[i]) % (w * type_bytes(types[i]) < 16 ? w * type_bytes(types[i]) : 16)) w = w == 8 ? 4 : 1;
  return w;
}

#ifdef __CUDACC__
template <int W>
struct Raw {
  uint32_t v[W];          // 16-bit types fill half of it
};

template <int W>
__device__ __forceinline__ void load_raw(Raw<W>& r, const void* p, int type, int64_t i) {
  if (type == S3R_F32) {
    const float* q = static_cast<const float*>(p) + i;
    if constexpr (W >= 4) {
#pragma unroll
      for (int k = 0; k < W; k += 4) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(q + k));
        r.v[k] = u.x, r.v[k + 1] = u.y, r.v[k + 2] = u.z, r.v[k + 3] = u.w;
      }
    } else {
      r.v[0] = __ldg(reinterpret_cast<const uint32_t*>(q));
    }
  } else {
    const uint16_t* q = static_cast<const uint16_t*>(p) + i;
    if constexpr (W == 8) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(q));
      r.v[0] = u.x, r.v[1] = u.y, r.v[2] = u.z, r.v[3] = u.w;
    } else if constexpr (W == 4) {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(q));
      r.v[0] = u.x, r.v[1] = u.y;
    } else {
      r.v[0] = __ldg(q);
    }
  }
}

__device__ __forceinline__ float half_lo(uint32_t v) { return __half2float(__ushort_as_half(static_cast<uint16_t>(v))); }
__device__ __forceinline__ float half_hi(uint32_t v) { return __half2float(__ushort_as_half(static_cast<uint16_t>(v >> 16))); }

template <int W>
__device__ __forceinline__ void unpack(float (&f)[W], const Raw<W>& r, int type) {
  if (type == S3R_F32) {
#pragma unroll
    for (int k = 0; k < W; ++k) f[k] = __uint_as_float(r.v[k]);
  } else if (type == S3R_BF16) {
    if constexpr (W == 1) {
      f[0] = bf16_lo(r.v[0]);
    } else {
#pragma unroll
      for (int k = 0; k < W; k += 2) f[k] = bf16_lo(r.v[k / 2]), f[k + 1] = bf16_hi(r.v[k / 2]);
    }
  } else {
    if constexpr (W == 1) {
      f[0] = half_lo(r.v[0]);
    } else {
#pragma unroll
      for (int k = 0; k < W; k += 2) f[k] = half_lo(r.v[k / 2]), f[k + 1] = half_hi(r.v[k / 2]);
    }
  }
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// to nearest even; what W values become in memory
template <int W>
__device__ __forceinline__ void pack(Raw<W>& r, const float (&f)[W], int type) {
  if (type == S3R_F32) {
#pragma unroll
    for (int k = 0; k < W; ++k) r.v[k] = __float_as_uint(f[k]);
  } else if constexpr (W == 1) {
    r.v[0] = (type == S3R_BF16 ? pack_bf16(f[0], 0.f) : pack_half(f[0], 0.f)) & 0xffffu;
  } else {
#pragma unroll
    for (int k = 0; k < W; k += 2) r.v[k / 2] = type == S3R_BF16 ? pack_bf16(f[k], f[k + 1]) : pack_half(f[k], f[k + 1]);
  }
}
template <int W>
__device__ __forceinline__ void store_raw(const Raw<W>& r, void* p, int type, int64_t i) {
  if (type == S3R_F32) {
    float* q = static_cast<float*>(p) + i;
    if constexpr (W >= 4) {
#pragma unroll
      for (int k = 0; k < W; k += 4) *reinterpret_cast<uint4*>(q + k) = make_uint4(r.v[k], r.v[k + 1], r.v[k + 2], r.v[k + 3]);
    } else {
      *reinterpret_cast<uint32_t*>(q) = r.v[0];
    }
  } else {
    uint16_t* q = static_cast<uint16_t*>(p) + i;
    if constexpr (W == 8) *reinterpret_cast<uint4*>(q) = make_uint4(r.v[0], r.v[1], r.v[2], r.v[3]);
    else if constexpr (W == 4) *reinterpret_cast<uint2*>(q) = make_uint2(r.v[0], r.v[1]);
    else *q = static_cast<uint16_t>(r.v[0]);
  }
}

__device__ __forceinline__ float load_one(const void* p, int type, int64_t i) {
  Raw<1> r;
  load_raw<1>(r, p, type, i);
  float f[1];
  unpack<1>(f, r, type);
  return f[0];
}
template <int W>
__device__ __forceinline__ void load_vector(float (&f)[W], const void* p, int type, int64_t i) {
  Raw<W> r;
  load_raw<W>(r, p, type, i);
  unpack<W>(f, r, type);
}

// max that keeps NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// A quotient of 8 bits per element and one scale per row: what 127 is worth, and its inverse.  Rows whose largest magnitude is
// below 2^-119 (127 / big would be infinite) become zeros.
struct RowScale {
  float scale, inverse;
};
__device__ __forceinline__ RowScale row_scale(float big) {
  return {__fdiv_rn(big, 127.f), big < 1.5046328e-36f ? 0.f : __fdiv_rn(127.f, big)};
}
// to nearest even, NaN to 0
__device__ __forceinline__ uint32_t to_s8(float v, float inverse) {
  int q;
  asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(q) : "f"(__fmul_rn(v, inverse)));
  return static_cast<uint32_t>(q) & 0xffu;
}

// Sums of N values over the G threads of a row, in a fixed order.  Rows of more than a warp exchange their warps' sums through
// `red` (2 x N x G / 32 floats, the halves in turn, so that one barrier per sum is enough: a half is written again only behind
// the barrier of the sum in between).  `bar`: number of the barrier of these threads.
template <int G, int N>
__device__ __forceinline__ void row_sum(float (&s)[N], float* red, uint32_t& turn, int t, int bar) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) s[k] += __shfl_xor_sync(0xffffffffu, s[k], o);
  if constexpr (G > 32) {
    constexpr int kWarps = G / 32;
    float* half = red + turn * (4 * kWarps);
    turn ^= 1u;
    if ((t & 31) == 0)
#pragma unroll
      for (int k = 0; k < N; ++k) half[k * kWarps + (t >> 5)] = s[k];
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(G) : "memory");
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float a = half[k * kWarps];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) a += half[k * kWarps + w];
      s[k] = a;
    }
  }
}
template <int G>
__device__ __forceinline__ float row_max(float s, float* red, uint32_t& turn, int t, int bar) {
#pragma unroll
  for (int o = 16; o; o >>= 1) s = max_nan(s, __shfl_xor_sync(0xffffffffu, s, o));
  if constexpr (G > 32) {
    constexpr int kWarps = G / 32;
    float* half = red + turn * (4 * kWarps);
    turn ^= 1u;
    if ((t & 31) == 0) half[t >> 5] = s;
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(G) : "memory");
    s = half[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) s = max_nan(s, half[w]);
  }
  return s;
}
#endif  // __CUDACC__

}  // namespace s3r
