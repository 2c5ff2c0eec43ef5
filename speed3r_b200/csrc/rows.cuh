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

// The vector at element i, where `in`.  Predicated, not branched around: a branch per vector, with the same registers written on
// both sides of it, makes loads wait for one another (64 512 rows of 1024: 160 us, this way 132).
template <int W>
__device__ __forceinline__ void load_raw(Raw<W>& r, const void* p, int type, int64_t i, bool in = true) {
  const char* at = static_cast<const char*>(p) + i * type_bytes(type);
  const int wide = in && type == S3R_F32, narrow = in && type != S3R_F32;
  if constexpr (W == 8) {
    asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.s32 a, %9, 0;\n\tsetp.ne.s32 b, %10, 0;\n\t"
                 "@a ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%8];\n\t@b ld.global.nc.v4.b32 {%4, %5, %6, %7}, [%8 + 16];\n\t}"
                 : "=r"(r.v[0]), "=r"(r.v[1]), "=r"(r.v[2]), "=r"(r.v[3]), "=r"(r.v[4]), "=r"(r.v[5]), "=r"(r.v[6]), "=r"(r.v[7])
                 : "l"(at), "r"(static_cast<int>(in)), "r"(wide));
  } else if constexpr (W == 4) {
    asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.s32 a, %5, 0;\n\tsetp.ne.s32 b, %6, 0;\n\t"
                 "@a ld.global.nc.v2.b32 {%0, %1}, [%4];\n\t@b ld.global.nc.v2.b32 {%2, %3}, [%4 + 8];\n\t}"
                 : "=r"(r.v[0]), "=r"(r.v[1]), "=r"(r.v[2]), "=r"(r.v[3]) : "l"(at), "r"(static_cast<int>(in)), "r"(wide));
  } else {
    asm volatile("{\n\t.reg .pred a, b;\n\t.reg .b16 h;\n\tsetp.ne.s32 a, %2, 0;\n\tsetp.ne.s32 b, %3, 0;\n\t"
                 "@a ld.global.nc.b32 %0, [%1];\n\t@b ld.global.nc.b16 h, [%1];\n\t@b mov.b32 %0, {h, h};\n\t}"
                 : "=r"(r.v[0]) : "l"(at), "r"(wide), "r"(narrow));
  }
}

__device__ __forceinline__ float half_lo(uint32_t v) { return __half2float(__ushort_as_half(static_cast<uint16_t>(v))); }
__device__ __forceinline__ float half_hi(uint32_t v) { return __half2float(__ushort_as_half(static_cast<uint16_t>(v >> 16))); }

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <int W>
__device__ __forceinline__ void unpack_as(float* f, const Raw<W>& r, int type) {       // type: a constant
  if (type == S3R_F32) {
#pragma unroll
    for (int k = 0; k < W; ++k) f[k] = __uint_as_float(r.v[k]);
  } else if (W == 1) {
    f[0] = type == S3R_BF16 ? bf16_lo(r.v[0]) : half_lo(r.v[0]);
  } else {
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const uint32_t v = r.v[k / 2];
      f[k] = type == S3R_BF16 ? (k & 1 ? bf16_hi(v) : bf16_lo(v)) : (k & 1 ? half_hi(v) : half_lo(v));
    }
  }
}
// all vectors of a thread in one branch; elements that are not there (`in`) are 0
template <int W, int N, typename In>
__device__ __forceinline__ void unpack_all(float (&f)[W * N], const Raw<W> (&r)[N], int type, In in) {
  if (type == S3R_F32) {
#pragma unroll
    for (int i = 0; i < N; ++i) unpack_as<W>(f + i * W, r[i], S3R_F32);
  } else if (type == S3R_BF16) {
#pragma unroll
    for (int i = 0; i < N; ++i) unpack_as<W>(f + i * W, r[i], S3R_BF16);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) unpack_as<W>(f + i * W, r[i], S3R_F16);
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (!in(i))
#pragma unroll
      for (int k = 0; k < W; ++k) f[i * W + k] = 0.f;
}
template <int W>
__device__ __forceinline__ void unpack(float (&f)[W], const Raw<W>& r, int type) {
  if (type == S3R_F32) unpack_as<W>(f, r, S3R_F32);
  else if (type == S3R_BF16) unpack_as<W>(f, r, S3R_BF16);
  else unpack_as<W>(f, r, S3R_F16);
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
__device__ __forceinline__ void store_raw(const Raw<W>& r, void* p, int type, int64_t i, bool in = true) {
  char* at = static_cast<char*>(p) + i * type_bytes(type);
  const int wide = in && type == S3R_F32, narrow = in && type != S3R_F32;
  if constexpr (W == 8) {
    asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.s32 a, %9, 0;\n\tsetp.ne.s32 b, %10, 0;\n\t"
                 "@a st.global.v4.b32 [%0], {%1, %2, %3, %4};\n\t@b st.global.v4.b32 [%0 + 16], {%5, %6, %7, %8};\n\t}"
                 ::"l"(at), "r"(r.v[0]), "r"(r.v[1]), "r"(r.v[2]), "r"(r.v[3]), "r"(r.v[4]), "r"(r.v[5]), "r"(r.v[6]), "r"(r.v[7]),
                 "r"(static_cast<int>(in)), "r"(wide) : "memory");
  } else if constexpr (W == 4) {
    asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.s32 a, %5, 0;\n\tsetp.ne.s32 b, %6, 0;\n\t"
                 "@a st.global.v2.b32 [%0], {%1, %2};\n\t@b st.global.v2.b32 [%0 + 8], {%3, %4};\n\t}"
                 ::"l"(at), "r"(r.v[0]), "r"(r.v[1]), "r"(r.v[2]), "r"(r.v[3]), "r"(static_cast<int>(in)), "r"(wide) : "memory");
  } else {
    asm volatile("{\n\t.reg .pred a, b;\n\t.reg .b16 h, z;\n\tsetp.ne.s32 a, %2, 0;\n\tsetp.ne.s32 b, %3, 0;\n\tmov.b32 {h, z}, %1;\n\t"
                 "@a st.global.b32 [%0], %1;\n\t@b st.global.b16 [%0], h;\n\t}"
                 ::"l"(at), "r"(r.v[0]), "r"(wide), "r"(narrow) : "memory");
  }
}
// rounds to the type (one branch), stores all vectors of a thread, and gives back what they hold now
template <int W, int N, typename At>
__device__ __forceinline__ void store_all(float (&f)[W * N], void* p, int type, At at, bool back = false) {
  Raw<W> o[N];
  auto one = [&](int i, int t) {
#pragma unroll
    for (int k = 0; k < W; ++k) {
      if (t == S3R_F32) o[i].v[k] = __float_as_uint(f[i * W + k]);
      else if (W == 1) o[i].v[0] = t == S3R_BF16 ? pack_bf16(f[i], 0.f) : pack_half(f[i], 0.f);
      else if (!(k & 1)) o[i].v[k / 2] = t == S3R_BF16 ? pack_bf16(f[i * W + k], f[i * W + (k + 1) % W]) : pack_half(f[i * W + k], f[i * W + (k + 1) % W]);
    }
    if (back) unpack_as<W>(f + i * W, o[i], t);
  };
  if (type == S3R_F32) {
#pragma unroll
    for (int i = 0; i < N; ++i) one(i, S3R_F32);
  } else if (type == S3R_BF16) {
#pragma unroll
    for (int i = 0; i < N; ++i) one(i, S3R_BF16);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) one(i, S3R_F16);
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t a = at(i);
      store_raw<W>(o[i], p, type, a, a >= 0);
    }
  } else if (type == S3R_F32) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (at(i) >= 0) static_cast<uint32_t*>(p)[at(i)] = o[i].v[0];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (at(i) >= 0) static_cast<uint16_t*>(p)[at(i)] = static_cast<uint16_t>(o[i].v[0]);
  }
}

__device__ __forceinline__ float load_one(const void* p, int type, int64_t i) {
  Raw<1> r;
  load_raw<1>(r, p, type, i);
  float f[1];
  unpack<1>(f, r, type);
  return f[0];
}
// f(an element's width): decided once in front of all loads, which then are on their way together; a load that decides for itself is waited for
// before the next, as load_one does (norms and rotation of 64 512 x 16 heads of 64: 139 us, this way 132; of one token 3.8 and 3.0)
template <typename F>
__device__ __forceinline__ void with_width(int type, F f) {
  if (type == S3R_F32) f(uint32_t());
  else f(uint16_t());
}
__device__ __forceinline__ float any_value(uint32_t w, int type) { return type == S3R_F32 ? __uint_as_float(w) : type == S3R_BF16 ? bf16_lo(w) : half_lo(w); }
template <int W>
__device__ __forceinline__ void load_vector(float (&f)[W], const void* p, int type, int64_t i) {
  Raw<W> r;
  load_raw<W>(r, p, type, i);
  unpack<W>(f, r, type);
}

// Rows on their way into shared memory (cp.async): each thread its own vectors, so that no barrier orders them.
constexpr int kRowsSmem = 220 * 1024;
template <int W>
__device__ __forceinline__ void stage_vector(uint32_t dst, const void* p, int type, int64_t i) {
  const char* src = static_cast<const char*>(p) + i * type_bytes(type);
  if constexpr (W == 8) {
    cp_async16(dst, src);
    if (type == S3R_F32) cp_async16(dst + 16, src + 16);
  } else {
    if (type == S3R_F32) cp_async16(dst, src);
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
  }
}
template <int W>
__device__ __forceinline__ void staged_raw(Raw<W>& r, const char* s, int type) {
  const uint32_t at = smem_u32(s);
  const int wide = type == S3R_F32;
  if constexpr (W == 8)
    asm volatile("{\n\t.reg .pred b;\n\tsetp.ne.s32 b, %9, 0;\n\t"
                 "ld.shared.v4.b32 {%0, %1, %2, %3}, [%8];\n\t@b ld.shared.v4.b32 {%4, %5, %6, %7}, [%8 + 16];\n\t}"
                 : "=r"(r.v[0]), "=r"(r.v[1]), "=r"(r.v[2]), "=r"(r.v[3]), "=r"(r.v[4]), "=r"(r.v[5]), "=r"(r.v[6]), "=r"(r.v[7]) : "r"(at), "r"(wide) : "memory");
  else
    asm volatile("{\n\t.reg .pred b;\n\tsetp.ne.s32 b, %5, 0;\n\t"
                 "ld.shared.v2.b32 {%0, %1}, [%4];\n\t@b ld.shared.v2.b32 {%2, %3}, [%4 + 8];\n\t}"
                 : "=r"(r.v[0]), "=r"(r.v[1]), "=r"(r.v[2]), "=r"(r.v[3]) : "r"(at), "r"(wide) : "memory");
}

// a vector's place in shared memory
template <int W>
__device__ __forceinline__ void zero_place(char* at, int bytes) {
#pragma unroll
  for (int k = 0; k < W; k += 2) {
    *reinterpret_cast<uint32_t*>(at + 2 * k) = 0;
    if (bytes == 4) *reinterpret_cast<uint32_t*>(at + 2 * W + 2 * k) = 0;
  }
}
__device__ __forceinline__ void cp_async_wait_for(int pending) {
  if (pending >= 3) cp_async_wait<3>();
  else if (pending == 2) cp_async_wait<2>();
  else if (pending == 1) cp_async_wait<1>();
  else cp_async_wait<0>();
}

// A sum that is not fused with the products in it: the assembler makes one instruction of a packed product and a packed sum, of a
// packed product and scalar sums it does not.
__device__ __forceinline__ float2 add_apart(float2 a, float2 b) { return make_float2(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y)); }

// the largest magnitude; NaN if one is
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float y;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
template <int W>
__device__ __forceinline__ float max_abs(float big, const float* v) {
#pragma unroll
  for (int k = 0; k + 1 < W; k += 2) big = max_abs(big, v[k], v[k + 1]);
  return W & 1 ? max_abs(big, v[W - 1], 0.f) : big;
}
// max that keeps NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// A quotient of 8 bits per element and one scale per row: what 127 is worth, and its inverse.  Rows whose largest magnitude is
// below 2^-119 become zeros (below 2^-121 the inverse, 127 / big, would be infinite); their scale is what it is.
struct RowScale {
  float scale, inverse;
};
__device__ __forceinline__ RowScale row_scale(float big) {
  return {__fdiv_rn(big, 127.f), big < 1.5046328e-36f ? 0.f : __fmul_rn(127.f, __frcp_rn(big))};      // as PyTorch takes 127 / big
}
// to nearest even, NaN to 0
__device__ __forceinline__ uint32_t to_s8(float v, float inverse) {
  int q;
  asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(q) : "f"(__fmul_rn(v, inverse)));
  return static_cast<uint32_t>(q) & 0xffu;
}
// four of them, the first in the lowest byte
__device__ __forceinline__ uint32_t to_s8x4(const float* v, float inverse) {
  const float2 lo = fmul2(make_float2(v[0], v[1]), make_float2(inverse, inverse)), hi = fmul2(make_float2(v[2], v[3]), make_float2(inverse, inverse));
  uint32_t w;
  asm("{\n\t.reg .s32 a, b, c, d;\n\tcvt.rni.s32.f32 a, %1;\n\tcvt.rni.s32.f32 b, %2;\n\tcvt.rni.s32.f32 c, %3;\n\tcvt.rni.s32.f32 d, %4;\n\t"
      "cvt.pack.sat.s8.s32.b32 c, d, c, 0;\n\tcvt.pack.sat.s8.s32.b32 %0, b, a, c;\n\t}"
      : "=r"(w) : "f"(lo.x), "f"(lo.y), "f"(hi.x), "f"(hi.y));
  return w;
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
// the largest of values that are not negative: their bits have the same order, NaN above all
template <int G>
__device__ __forceinline__ float row_max(float s, float* red, uint32_t& turn, int t, int bar) {
  s = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(s)));
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
