// AdamW over many tensors in one launch, with states in 32 or in 8 bits, and the norm of their gradients.
// Bound: HBM.  32-bit states 28 bytes per element (fp32 parameters: p, m, v read and written, g read), 8-bit states 16; the norm 4.
//
// 8-bit states: blocks of 256 codes share an exponent, so that a block is a warp's work: eight elements per lane, the largest
// magnitudes by shuffles.  The shared factor is a power of two: it changes only when a block's largest magnitude crosses one, so that
// the codes' grid stands still between steps.  Rounding a v that moves by 0.1 % a step then has a variance of step size x change
// (with any other factor every code would be rounded anew each step, with step size^2 / 6, 30 times as much, and to nearest it
// would hardly ever move).  All scalings are by powers of two and exact, but for values below a code's normal numbers (exponent field 0): these
// are fp32 subnormals once scaled, rounded to 2^-20 of a code's step before they are rounded to the code.  There is no other rounding of a state.
#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "rows.cuh"

namespace s3r {

// Tensors per launch: their table is an argument of the kernel, 23 KB for 320; a launch of a few tensors copies a shorter one.
constexpr int kAdamBlock = 256, kAdamThreads = 128, kAdamMax = 320, kAdamFew = 32;
constexpr int kAdamWarps = kAdamThreads / 32;
constexpr int kAdamPerCta = kAdamBlock * kAdamWarps;

struct AdamScalars {
  float factor;        // of the gradients
  float decay;         // 1 - lr * weight_decay
  float step_size;     // lr / (1 - beta1^t)
  float inv_root;      // 1 / sqrt(1 - beta2^t)
  uint32_t t;
  uint32_t skip;
};

struct AdamTensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  uint8_t *me, *ve;
  int64_t n;
  int64_t first;       // CTA
  uint32_t flags;      // types (2 bits each), vectors, 8-bit states, number << 8
};
struct AdamCommon {
  int n;
  float b1, c1, b2, c2, eps;
  int64_t seed;
  const AdamScalars* scalars;
};
// Which tensor the CTAs i << shift belong to: a search through all of 252 tensors was a twelfth of the time (0.9 M elements each: 645 us, this way 603).
template <int MAX>
struct Starts {
  uint16_t at[MAX + 1];
  int shift;
};
template <int MAX, typename T>
static void fill_starts(Starts<MAX>& s, const T* t, int n, int64_t ctas) {
  s.shift = 0;
  while ((ctas - 1) >> s.shift >= MAX) ++s.shift;
  const int last = static_cast<int>((ctas - 1) >> s.shift);
  for (int b = 0, i = 0; b <= last; ++b) {
    while (i + 1 < n && t[i + 1].first <= static_cast<int64_t>(b) << s.shift) ++i;
    s.at[b] = static_cast<uint16_t>(i);
  }
  s.at[last + 1] = static_cast<uint16_t>(n - 1);
}
template <int MAX>
struct AdamParams {
  AdamCommon c;
  Starts<MAX> starts;
  AdamTensor t[MAX];
};
constexpr uint32_t kAdamVector = 16, kAdamEight = 32;

template <typename T, int MAX>
__device__ __forceinline__ const T& tensor_of(const T (&t)[MAX], const Starts<MAX>& s, int64_t cta) {
  int lo = s.at[cta >> s.shift], hi = s.at[(cta >> s.shift) + 1];          // the last tensor whose first CTA is not behind this one
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t[mid].first <= cta) lo = mid;
    else hi = mid - 1;
  }
  return t[lo];
}

struct BeginParams {
  int64_t* step;
  const float* lr;
  double lr_host, log_b1, log_b2, weight_decay, max_norm;
  const float* norm;
  AdamScalars* out;
};

// what all elements share; one thread
__global__ void adamw_begin_kernel(const __grid_constant__ BeginParams p) {
  griddep_wait();
  griddep_launch();
  AdamScalars s = {};
  const float norm = p.norm ? *p.norm : 0.f;
  s.skip = !(fabsf(norm) <= 3.4028235e38f);
  const int64_t t = *p.step + 1;
  if (!s.skip) *p.step = t;
  s.factor = 1.f;
  if (p.norm && p.max_norm > 0) s.factor = fminf(__fdiv_rn(static_cast<float>(p.max_norm), __fadd_rn(norm, 1e-6f)), 1.f);
  const double lr = p.lr ? static_cast<double>(*p.lr) : p.lr_host;
  s.decay = static_cast<float>(1.0 - lr * p.weight_decay);
  // 1 - b^t = -expm1(t log b): exact to fp32 where b^t is close to 1
  s.step_size = static_cast<float>(lr) / -expm1f(static_cast<float>(t * p.log_b1));
  s.inv_root = 1.f / sqrtf(-expm1f(static_cast<float>(t * p.log_b2)));
  s.t = static_cast<uint32_t>(t);
  *p.out = s;
}

// Philox 2x32 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3), seven rounds
__device__ __forceinline__ uint2 philox(uint32_t a, uint32_t c, uint32_t key) {
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    const uint64_t m = static_cast<uint64_t>(a) * 0xD256D193u;
    a = static_cast<uint32_t>(m >> 32) ^ key ^ c;
    c = static_cast<uint32_t>(m);
    key += 0x9E3779B9u;
  }
  return make_uint2(a, c);
}

// The exponent of a block whose largest magnitude has these bits: 1.875 x 2^(e - 127) is the smallest such bound.  255: not finite, or
// beyond 2^100.  Below 2^-100 the exponent stays.
__device__ __forceinline__ uint32_t block_exponent(uint32_t bits) {
  const uint32_t e = bits >= 0x7f800000u ? 255u : (bits + 0xFFFFFu) >> 23;
  return e > 227u ? 255u : max(e, 27u);
}
__device__ __forceinline__ float power_of(uint32_t biased) { return __uint_as_float(biased << 23); }
// Codes are the top of the bits of |x| scaled so that the code's smallest exponent field is fp32's own; what is added below the last bit
// that is kept rounds them (0x7FFFF and that bit: to nearest even; a random number of as many bits: stochastically).  Two products, by
// powers of two: by the block's power of two, then by 2^-112 (m, 4 bits of exponent) or 2^-96 (v, 5 bits).
constexpr float kDownM = 1.92592994438723585e-34f, kDownV = 1.26217744835361889e-29f;
constexpr float kUpM = 5.19229685853482763e33f, kUpV = 7.92281625142643376e28f;
__device__ __forceinline__ float unit_of(uint32_t e) { return e == 255u ? __uint_as_float(0x7fffffffu) : power_of(e); }
__device__ __forceinline__ float2 both_of(float x) { return make_float2(x, x); }

// byte k of a word times 2^20; SIGN: its highest bit in all bits above
template <bool SIGN>
__device__ __forceinline__ uint32_t code_bits(uint32_t bytes, int k) {
  uint32_t w;
  asm("prmt.b32 %0, %1, 0, %2;" : "=r"(w) : "r"(bytes), "r"((SIGN ? 0x8044u + (k << 12) : 0x4044u) + (k << 8)));
  return w * 16u;
}
// the top bytes of four words
__device__ __forceinline__ uint32_t gather(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}
__device__ __forceinline__ void decode_m(float2 (&m)[4], uint2 codes, float unit) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = code_bits<true>(h ? codes.y : codes.x, k) & 0x87f00000u;      // sign, code << 20
    m[2 * h] = fmul2(fmul2(make_float2(__uint_as_float(w[0]), __uint_as_float(w[1])), both_of(kUpM)), both_of(unit));
    m[2 * h + 1] = fmul2(fmul2(make_float2(__uint_as_float(w[2]), __uint_as_float(w[3])), both_of(kUpM)), both_of(unit));
  }
}
__device__ __forceinline__ void decode_v(float2 (&v)[4], uint2 codes, float unit) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = code_bits<false>(h ? codes.y : codes.x, k);
    v[2 * h] = fmul2(fmul2(make_float2(__uint_as_float(w[0]), __uint_as_float(w[1])), both_of(kUpV)), both_of(unit));
    v[2 * h + 1] = fmul2(fmul2(make_float2(__uint_as_float(w[2]), __uint_as_float(w[3])), both_of(kUpV)), both_of(unit));
  }
}
template <bool SUBNORMAL>
__device__ __forceinline__ float sqrt_near(float x) {
  float y;
  if constexpr (SUBNORMAL) asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  else asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));            // 0 below 2^-126
  return y;
}
__device__ __forceinline__ float rcp_near(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Eight elements of a lane, as they come from memory.  W = 8: all of them exist and every array begins at a multiple of 16 bytes.
template <bool EIGHT>
struct Lane {
  Raw<8> g, w, m, v;         // with 8-bit states m.v[0..1] and v.v[0..1] are codes
  uint32_t me, ve;
};
template <int W>
__device__ __forceinline__ void load_lane(Raw<8>& r, const void* p, int type, int64_t at, int64_t n) {
  if constexpr (W == 8) {
    load_raw<8>(r, p, type, at);
  } else {
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = at + k < n ? load_one(p, type, at + k) : 0.f;
    pack<8>(r, f, type);
  }
}
template <int W>
__device__ __forceinline__ void store_lane(const float2 (&f)[4], void* p, int type, int64_t at, int64_t n) {
  float e[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) e[2 * k] = f[k].x, e[2 * k + 1] = f[k].y;
  if constexpr (W == 8) {
    Raw<8> r;
    pack<8>(r, e, type);
    store_raw<8>(r, p, type, at);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (at + k < n) {
        const float one[1] = {e[k]};
        Raw<1> r;
        pack<1>(r, one, type);
        store_raw<1>(r, p, type, at + k);
      }
  }
}
// Eight fp32 values of a lane, the array at a multiple of 16 bytes.  One store where they fill a sector of 32 bytes: in two, each of a warp's
// stores touches all its sectors (reading out 60 M elements: 108 us, this way 84).  The step, which reads more than it writes, gains nothing.
__device__ __forceinline__ void store_sector(const float2 (&f)[4], float* p) {
  if (reinterpret_cast<uintptr_t>(p) & 31) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
  } else {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "f"(f[0].x), "f"(f[0].y), "f"(f[1].x), "f"(f[1].y), "f"(f[2].x), "f"(f[2].y), "f"(f[3].x), "f"(f[3].y) : "memory");
  }
}
template <int W>
__device__ __forceinline__ uint2 load_codes(const uint8_t* p, int64_t at, int64_t n) {
  if constexpr (W == 8) return *reinterpret_cast<const uint2*>(p + at);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (at + k < n) w[k / 4] |= static_cast<uint32_t>(p[at + k]) << (8 * (k & 3));
  return make_uint2(w[0], w[1]);
}
template <int W>
__device__ __forceinline__ void store_codes(uint2 c, uint8_t* p, int64_t at, int64_t n) {
  if constexpr (W == 8) {
    *reinterpret_cast<uint2*>(p + at) = c;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (at + k < n) p[at + k] = static_cast<uint8_t>((k < 4 ? c.x : c.y) >> (8 * (k & 3)));
  }
}

template <int W, bool EIGHT>
__device__ __forceinline__ void load_block(Lane<EIGHT>& l, const AdamTensor& x, int64_t block, int lane) {
  const int64_t at = block * kAdamBlock + lane * 8;
  load_lane<W>(l.g, x.g, x.flags >> 2 & 3, at, x.n);
  load_lane<W>(l.w, x.p, x.flags & 3, at, x.n);
  if constexpr (EIGHT) {
    const uint2 mc = load_codes<W>(static_cast<const uint8_t*>(x.m), at, x.n), vc = load_codes<W>(static_cast<const uint8_t*>(x.v), at, x.n);
    l.m.v[0] = mc.x, l.m.v[1] = mc.y, l.v.v[0] = vc.x, l.v.v[1] = vc.y;
    l.me = x.me[block];
    l.ve = x.ve[block];
  } else {
    load_lane<W>(l.m, x.m, S3R_F32, at, x.n);
    load_lane<W>(l.v, x.v, S3R_F32, at, x.n);
  }
}

template <int W, bool EIGHT, bool SUBNORMAL>
__device__ __forceinline__ void step_block(const Lane<EIGHT>& l, const AdamCommon& p, const AdamTensor& x, const AdamScalars& s, int64_t block, int lane) {
  const int64_t at = block * kAdamBlock + lane * 8;
  const int p_type = x.flags & 3, g_type = x.flags >> 2 & 3;
  const bool nearest = p.seed < 0;
  float e[8];
  float2 w[4], m[4], v[4];
  unpack<8>(e, l.w, p_type);
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = make_float2(e[2 * k], e[2 * k + 1]);
  unpack<8>(e, l.g, g_type);
  if constexpr (EIGHT) {
    decode_m(m, make_uint2(l.m.v[0], l.m.v[1]), unit_of(l.me));
    decode_v(v, make_uint2(l.v.v[0], l.v.v[1]), unit_of(l.ve));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      m[k] = make_float2(__uint_as_float(l.m.v[2 * k]), __uint_as_float(l.m.v[2 * k + 1]));
      v[k] = make_float2(__uint_as_float(l.v.v[2 * k]), __uint_as_float(l.v.v[2 * k + 1]));
    }
  }
  // Every product and sum of the states is rounded by itself, as in separate operations: codes do not depend on which of them would
  // have been fused.  The parameter's own arithmetic is the approximate root and reciprocal (2^-23 of the step).
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 g = fmul2(make_float2(e[2 * k], e[2 * k + 1]), both_of(s.factor));
    m[k] = add_apart(fmul2(m[k], both_of(p.b1)), fmul2(g, both_of(p.c1)));
    v[k] = add_apart(fmul2(v[k], both_of(p.b2)), fmul2(fmul2(g, g), both_of(p.c2)));
    const float2 root = ffma2(make_float2(sqrt_near<SUBNORMAL>(v[k].x), sqrt_near<SUBNORMAL>(v[k].y)), both_of(s.inv_root), both_of(p.eps));
    const float2 step = fmul2(m[k], make_float2(rcp_near(root.x), rcp_near(root.y)));
    w[k] = ffma2(w[k], both_of(s.decay), fmul2(step, both_of(-s.step_size)));
  }
  uint32_t low[8];
  if (!nearest && (EIGHT || p_type == S3R_BF16)) {
    const uint32_t key = static_cast<uint32_t>(p.seed) + (x.flags >> 8) * 0x85EBCA6Bu;
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      const uint2 r = philox(static_cast<uint32_t>((at + k) >> 1), s.t, key);
      low[k] = r.x;
      low[k + 1] = r.y;
    }
    // All 16 bits that a bf16 parameter drops, so that an update of any size happens as often as it should; the lower 6 of them are the upper 6
    // of those that round v, on which a parameter's rounding hardly ever depends.  fp16's values below 2^-14 have fewer, so it is rounded to
    // nearest.
    if (p_type == S3R_BF16)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (fabsf(w[k].x) < 3.3e38f) w[k].x = __uint_as_float((__float_as_uint(w[k].x) + (low[2 * k] >> 16)) & 0xffff0000u);
        if (fabsf(w[k].y) < 3.3e38f) w[k].y = __uint_as_float((__float_as_uint(w[k].y) + (low[2 * k + 1] >> 16)) & 0xffff0000u);
      }
  }
  store_lane<W>(w, x.p, p_type, at, x.n);
  if constexpr (!EIGHT) {
    store_lane<W>(m, x.m, S3R_F32, at, x.n);
    store_lane<W>(v, x.v, S3R_F32, at, x.n);
  } else {
    // the largest magnitudes; NaN above all, as bits too
    float m_top = 0.f, v_top = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) m_top = max_abs(m_top, m[k].x, m[k].y), v_top = max_abs(v_top, v[k].x, v[k].y);
    const uint32_t me = block_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(m_top)));
    const uint32_t ve = block_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(v_top)));
    const float m_up = me == 255u ? 0.f : power_of(254u - me), v_up = ve == 255u ? 0.f : power_of(254u - ve);
    uint32_t mc[8], vc[8];
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      const float2 a = fmul2(fmul2(m[k / 2], both_of(m_up)), both_of(kDownM)), b = fmul2(fmul2(v[k / 2], both_of(v_up)), both_of(kDownV));
      mc[k] = __float_as_uint(a.x), mc[k + 1] = __float_as_uint(a.y);
      vc[k] = __float_as_uint(b.x), vc[k + 1] = __float_as_uint(b.y);
    }
    // To the top byte, rounded on the way (16 x + 16 r).  8 random bits of the 20 that a code of m drops, 14 of v's: v moves less in a step.
    // No code passes its largest one: the block's exponent is such that 1.875 times the power of two is reached exactly at most.
    uint32_t v_least = 0xffffffffu;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t sign = mc[k];
      if (nearest) {
        mc[k] = (mc[k] + 0x7FFFFu + (mc[k] >> 20 & 1u)) * 16u;
        vc[k] = (vc[k] + 0x7FFFFu + (vc[k] >> 20 & 1u)) * 16u;
      } else {
        mc[k] = mc[k] * 16u + __byte_perm(low[k], 0x8000u, 0x7054);                      // low[7:0] << 16, half of the last bit below
        vc[k] = (vc[k] * 4u + ((low[k] & 0x3FFF00u) | 0x80u)) * 4u;
      }
      mc[k] = (mc[k] & 0x7fffffffu) | (sign & 0x80000000u);
      v_least = min(v_least, vc[k]);
    }
    // a v that is not zero keeps a code that is not: a denominator never becomes eps alone by rounding
    if (v_least < 1u << 24) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (vc[k] < 1u << 24 && (k & 1 ? v[k / 2].y : v[k / 2].x) != 0.f) vc[k] = 1u << 24;
    }
    const uint2 m_codes = make_uint2(gather(mc[0], mc[1], mc[2], mc[3]), gather(mc[4], mc[5], mc[6], mc[7]));
    const uint2 v_codes = make_uint2(gather(vc[0], vc[1], vc[2], vc[3]), gather(vc[4], vc[5], vc[6], vc[7]));
    store_codes<W>(me == 255u ? make_uint2(0, 0) : m_codes, static_cast<uint8_t*>(x.m), at, x.n);
    store_codes<W>(ve == 255u ? make_uint2(0, 0) : v_codes, static_cast<uint8_t*>(x.v), at, x.n);
    if (lane == 0) {
      x.me[block] = static_cast<uint8_t>(me);
      x.ve[block] = static_cast<uint8_t>(ve);
    }
  }
}

// A warp has one block.  What hides the latency of its loads is other warps: with 56 registers 36 of them fit an SM (227 M elements in 252
// tensors, 8-bit states, 601 us = 6.0 TB/s, 172 bytes of spills and all; with 64 registers 629, with 48 a hundredth more than with 56), and a
// loop over several blocks, with or without the next one on its way in registers, lost more of them than it gained.  CTAs of 128 leave an SM in smaller
// parts than those of 256 (640 where those take 715).
template <bool EIGHT, bool SUBNORMAL>
__device__ __forceinline__ void run_block(const AdamCommon& p, const AdamTensor& x, int64_t block, int lane) {
  Lane<EIGHT> l;
  // whole blocks of tensors that begin at multiples of 16 bytes; what ends a tensor, and tensors that begin anywhere, element by element
  if ((x.flags & kAdamVector) && (block + 1) * kAdamBlock <= x.n) {
    load_block<8, EIGHT>(l, x, block, lane);
    const AdamScalars s = *p.scalars;
    if (!s.skip) step_block<8, EIGHT, SUBNORMAL>(l, p, x, s, block, lane);
  } else {
    load_block<1, EIGHT>(l, x, block, lane);
    const AdamScalars s = *p.scalars;
    if (!s.skip) step_block<1, EIGHT, SUBNORMAL>(l, p, x, s, block, lane);
  }
}

template <int MAX, bool SUBNORMAL>
__global__ void __launch_bounds__(kAdamThreads, 9) adamw_kernel(const __grid_constant__ AdamParams<MAX> p) {
  const AdamTensor& x = tensor_of(p.t, p.starts, blockIdx.x);
  const int64_t block = (blockIdx.x - x.first) * kAdamWarps + (threadIdx.x >> 5);
  griddep_wait();
  griddep_launch();
  if (block * kAdamBlock >= x.n) return;
  if (x.flags & kAdamEight) run_block<true, SUBNORMAL>(p.c, x, block, threadIdx.x & 31);
  else run_block<false, SUBNORMAL>(p.c, x, block, threadIdx.x & 31);
}

// ---- the norm of the gradients: squares in 64 bits, where every one of them is exact ------------------------------------
constexpr int kNormThreads = 256, kNormPerCta = 16384;

struct NormTensor {
  const void* g;
  int64_t n;
  int64_t first;
  uint32_t flags;
};
template <int MAX>
struct GradNormParams {
  double* partial;
  int n;
  Starts<MAX> starts;
  NormTensor t[MAX];
};

template <int MAX>
__global__ void __launch_bounds__(kNormThreads) grad_norm_kernel(const __grid_constant__ GradNormParams<MAX> p) {
  __shared__ double red[kNormThreads / 32];
  const NormTensor& x = tensor_of(p.t, p.starts, blockIdx.x);
  griddep_wait();
  griddep_launch();
  const int64_t from = (blockIdx.x - x.first) * kNormPerCta, to = min(x.n, from + kNormPerCta);
  const int type = x.flags & 3;
  double s[4] = {0., 0., 0., 0.};
  int64_t at = from + threadIdx.x * 8;
  if (x.flags & kAdamVector) {
#pragma unroll 2
    for (; at + 8 <= to; at += kNormThreads * 8) {
      float f[8];
      load_vector<8>(f, x.g, type, at);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const double d = f[k];
        s[k & 3] = fma(d, d, s[k & 3]);
      }
    }
  }
  for (; at < to; at += kNormThreads * 8)
    for (int64_t k = at; k < min(at + 8, to); ++k) {
      const double d = load_one(x.g, type, k);
      s[0] = fma(d, d, s[0]);
    }
  double sum = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kNormThreads / 32; ++w) sum += red[w];
    p.partial[blockIdx.x] = sum;
  }
}

__global__ void __launch_bounds__(1024) grad_norm_end_kernel(const double* partial, int64_t n, float* norm) {
  __shared__ double red[32];
  griddep_wait();
  griddep_launch();
  double s = 0.;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += partial[i];
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = red[threadIdx.x];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) *norm = static_cast<float>(sqrt(s));
  }
}

// ---- what 8-bit states stand for -----------------------------------------------------------------------------------------
struct StateTensor {
  const uint8_t *m, *v, *me, *ve;
  float *m_out, *v_out;
  int64_t n, first;
  uint32_t flags;
};
template <int MAX>
struct StateParams {
  int n;
  Starts<MAX> starts;
  StateTensor t[MAX];
};
template <int MAX>
__global__ void __launch_bounds__(kAdamThreads) adamw_state_kernel(const __grid_constant__ StateParams<MAX> p) {
  const StateTensor& x = tensor_of(p.t, p.starts, blockIdx.x);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t block = (blockIdx.x - x.first) * kAdamWarps + warp, at = block * kAdamBlock + lane * 8;
  griddep_wait();
  griddep_launch();
  if (at >= x.n) return;
  const bool whole = (x.flags & kAdamVector) && at + 8 <= x.n;
  const uint2 mc = whole ? load_codes<8>(x.m, at, x.n) : load_codes<1>(x.m, at, x.n), vc = whole ? load_codes<8>(x.v, at, x.n) : load_codes<1>(x.v, at, x.n);
  float2 m[4], v[4];
  decode_m(m, mc, unit_of(x.me[block]));
  decode_v(v, vc, unit_of(x.ve[block]));
  if (whole) {
    store_sector(m, x.m_out + at);
    store_sector(v, x.v_out + at);
  } else {
    store_lane<1>(m, x.m_out, S3R_F32, at, x.n);
    store_lane<1>(v, x.v_out, S3R_F32, at, x.n);
  }
}

static bool at_16(std::initializer_list<const void*> p) {
  uintptr_t all = 0;
  for (const void* q : p) all |= reinterpret_cast<uintptr_t>(q);
  return (all & 15) == 0;
}

}  // namespace s3r

using namespace s3r;

extern "C" size_t s3r_grad_norm_workspace_bytes(int n, const int64_t* counts) {
  size_t parts = 0;
  for (int i = 0; counts && i < n; ++i) parts += counts[i] > 0 ? (counts[i] + kNormPerCta - 1) / kNormPerCta : 0;
  return (parts + 1) * sizeof(double);
}

extern "C" int s3r_grad_norm(int n, const void* const* tensors, const int64_t* counts, const int* types, float* norm, void* workspace,
                             size_t workspace_bytes, void* stream) {
  S3R_REQUIRE(n >= 0, S3R_ERR_SHAPE, "s3r_grad_norm: %d tensors", n);
  S3R_REQUIRE(norm && workspace && (n == 0 || (tensors && counts && types)), S3R_ERR_NULL, "s3r_grad_norm: NULL pointer");
  S3R_REQUIRE(workspace_bytes >= s3r_grad_norm_workspace_bytes(n, counts) && reinterpret_cast<uintptr_t>(workspace) % 8 == 0, S3R_ERR_TOO_LARGE,
              "s3r_grad_norm: workspace of %zu bytes is smaller than the %zu needed", workspace_bytes, s3r_grad_norm_workspace_bytes(n, counts));
  for (int i = 0; i < n; ++i) {
    S3R_REQUIRE(counts[i] >= 0, S3R_ERR_SHAPE, "s3r_grad_norm: negative count");
    S3R_REQUIRE(counts[i] == 0 || tensors[i], S3R_ERR_NULL, "s3r_grad_norm: NULL pointer");
    S3R_REQUIRE(known_type(types[i]), S3R_ERR_UNSUPPORTED, "s3r_grad_norm: types are fp32, bf16 and fp16");
    S3R_REQUIRE(reinterpret_cast<uintptr_t>(tensors[i]) % type_bytes(types[i]) == 0, S3R_ERR_ALIGNMENT, "s3r_grad_norm: elements must be aligned");
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  static thread_local GradNormParams<kAdamMax> p;
  GradNormParams<kAdamFew> few;
  p.partial = static_cast<double*>(workspace);
  p.n = 0;
  int64_t ctas = 0, all = 0;
  for (int i = 0; i <= n; ++i) {
    if (p.n && (i == n || p.n == kAdamMax)) {
      int rc;
      if (p.n <= kAdamFew) {
        few.partial = p.partial;
        few.n = p.n;
        std::copy_n(p.t, p.n, few.t);
        fill_starts(few.starts, p.t, p.n, ctas);
        rc = launch(grad_norm_kernel<kAdamFew>, static_cast<unsigned>(ctas), kNormThreads, 0, st, few);
      } else {
        fill_starts(p.starts, p.t, p.n, ctas);
        rc = launch(grad_norm_kernel<kAdamMax>, static_cast<unsigned>(ctas), kNormThreads, 0, st, p);
      }
      if (rc) return rc;
      p.partial += ctas;
      all += ctas;
      p.n = 0;
      ctas = 0;
    }
    if (i == n || counts[i] == 0) continue;
    p.t[p.n++] = {tensors[i], counts[i], ctas, static_cast<uint32_t>(types[i]) | (at_16({tensors[i]}) ? kAdamVector : 0u)};
    ctas += (counts[i] + kNormPerCta - 1) / kNormPerCta;
    S3R_REQUIRE(ctas < (1ll << 31), S3R_ERR_TOO_LARGE, "s3r_grad_norm: grid too large");
  }
  return launch(grad_norm_end_kernel, 1u, 1024, 0, st, static_cast<const double*>(workspace), all, norm);
}

extern "C" int s3r_adamw_step(const s3r_adamw* args, void* stream) { return s3r_adamw_step_numbered(args, nullptr, stream); }

extern "C" int s3r_adamw_step_numbered(const s3r_adamw* args, const uint32_t* numbers, void* stream) {
  S3R_REQUIRE(args, S3R_ERR_NULL, "s3r_adamw_step: NULL pointer");
  const s3r_adamw& a = *args;
  S3R_REQUIRE(a.n >= 0, S3R_ERR_SHAPE, "s3r_adamw_step: %d tensors", a.n);
  S3R_REQUIRE(a.step && a.workspace && (a.n == 0 || (a.params && a.grads && a.m && a.v && a.counts && a.param_types && a.grad_types)), S3R_ERR_NULL,
              "s3r_adamw_step: NULL pointer");
  S3R_REQUIRE(a.beta1 >= 0 && a.beta1 < 1 && a.beta2 >= 0 && a.beta2 < 1 && a.eps >= 0, S3R_ERR_UNSUPPORTED, "s3r_adamw_step: betas are in [0, 1), eps is not negative");
  S3R_REQUIRE(a.eps == 0 || a.eps >= 0x1p-126, S3R_ERR_UNSUPPORTED, "s3r_adamw_step: eps is 0 or a normal number of fp32, got %g", a.eps);
  S3R_REQUIRE(reinterpret_cast<uintptr_t>(a.step) % 8 == 0 && reinterpret_cast<uintptr_t>(a.workspace) % 8 == 0, S3R_ERR_ALIGNMENT, "s3r_adamw_step: elements must be aligned");
  for (int i = 0; i < a.n; ++i) {
    S3R_REQUIRE(a.counts[i] >= 0, S3R_ERR_SHAPE, "s3r_adamw_step: negative count");
    if (a.counts[i] == 0) continue;
    S3R_REQUIRE(a.params[i] && a.grads[i] && a.m[i] && a.v[i], S3R_ERR_NULL, "s3r_adamw_step: NULL pointer");
    S3R_REQUIRE(known_type(a.param_types[i]) && known_type(a.grad_types[i]), S3R_ERR_UNSUPPORTED, "s3r_adamw_step: types are fp32, bf16 and fp16");
    const bool eight = a.m_exponents && a.m_exponents[i];
    S3R_REQUIRE(eight == (a.v_exponents && a.v_exponents[i]), S3R_ERR_NULL, "s3r_adamw_step: exponents of m and v come together");
    S3R_REQUIRE(reinterpret_cast<uintptr_t>(a.params[i]) % type_bytes(a.param_types[i]) == 0 && reinterpret_cast<uintptr_t>(a.grads[i]) % type_bytes(a.grad_types[i]) == 0 &&
                    (eight || (reinterpret_cast<uintptr_t>(a.m[i]) | reinterpret_cast<uintptr_t>(a.v[i])) % 4 == 0), S3R_ERR_ALIGNMENT, "s3r_adamw_step: elements must be aligned");
    S3R_REQUIRE(a.counts[i] < (1ll << 33), S3R_ERR_TOO_LARGE, "s3r_adamw_step: more than 2^33 elements in a tensor");
    S3R_REQUIRE((numbers ? numbers[i] : static_cast<uint32_t>(i)) < 1u << 24, S3R_ERR_TOO_LARGE, "s3r_adamw_step: tensors are numbered below 2^24");
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  AdamScalars* scalars = static_cast<AdamScalars*>(a.workspace);
  // log 0 = -inf: 1 - 0^t = 1
  const BeginParams b = {a.step, a.lr, a.lr_host, log(a.beta1), log(a.beta2), a.weight_decay, a.max_norm, a.norm, scalars};
  if (const int rc = launch(adamw_begin_kernel, 1u, 1, 0, st, b)) return rc;
  static thread_local AdamParams<kAdamMax> p;
  AdamParams<kAdamFew> few;
  p.c.b1 = static_cast<float>(a.beta1);
  p.c.c1 = static_cast<float>(1.0 - a.beta1);
  p.c.b2 = static_cast<float>(a.beta2);
  p.c.c2 = static_cast<float>(1.0 - a.beta2);
  p.c.eps = static_cast<float>(a.eps);
  p.c.seed = static_cast<uint32_t>(a.seed) + static_cast<uint32_t>(a.seed >> 32) * 0xC2B2AE35u;
  if (a.seed < 0) p.c.seed = -1;
  p.c.scalars = scalars;
  p.c.n = 0;
  // A v below 2^-126 has a root below 2^-63, times 1 / sqrt(1 - beta2) at most.  Where that is 2^-24 of eps and less it may be taken as 0 (the
  // cheaper root: the other one costs 8-bit states 1 to 3 %); with a smaller eps it is what the step is divided by.
  const bool subnormal = a.eps * sqrt(1.0 - a.beta2) < 0x1p-39;
  int64_t ctas = 0;
  for (int i = 0; i <= a.n; ++i) {
    if (p.c.n && (i == a.n || p.c.n == kAdamMax)) {
      int rc;
      if (p.c.n <= kAdamFew) {
        few.c = p.c;
        std::copy_n(p.t, p.c.n, few.t);
        fill_starts(few.starts, p.t, p.c.n, ctas);
        rc = launch(subnormal ? adamw_kernel<kAdamFew, true> : adamw_kernel<kAdamFew, false>, static_cast<unsigned>(ctas), kAdamThreads, 0, st, few);
      } else {
        fill_starts(p.starts, p.t, p.c.n, ctas);
        rc = launch(subnormal ? adamw_kernel<kAdamMax, true> : adamw_kernel<kAdamMax, false>, static_cast<unsigned>(ctas), kAdamThreads, 0, st, p);
      }
      if (rc) return rc;
      p.c.n = 0;
      ctas = 0;
    }
    if (i == a.n || a.counts[i] == 0) continue;
    uint8_t *me = a.m_exponents ? a.m_exponents[i] : nullptr, *ve = a.v_exponents ? a.v_exponents[i] : nullptr;
    const uint32_t flags = static_cast<uint32_t>(a.param_types[i]) | static_cast<uint32_t>(a.grad_types[i]) << 2 |
                           (at_16({a.params[i], a.grads[i], a.m[i], a.v[i]}) ? kAdamVector : 0u) | (me ? kAdamEight : 0u) | (numbers ? numbers[i] : static_cast<uint32_t>(i)) << 8;
    p.t[p.c.n++] = {a.params[i], a.grads[i], a.m[i], a.v[i], me, ve, a.counts[i], ctas, flags};
    ctas += (a.counts[i] + kAdamPerCta - 1) / kAdamPerCta;
    S3R_REQUIRE(ctas < (1ll << 31), S3R_ERR_TOO_LARGE, "s3r_adamw_step: grid too large");
  }
  return 0;
}

extern "C" int s3r_adamw_state(int n, const void* const* m, const void* const* v, const uint8_t* const* m_exponents,
                               const uint8_t* const* v_exponents, float* const* m_out, float* const* v_out, const int64_t* counts, void* stream) {
  S3R_REQUIRE(n >= 0, S3R_ERR_SHAPE, "s3r_adamw_state: %d tensors", n);
  S3R_REQUIRE(n == 0 || (m && v && m_exponents && v_exponents && m_out && v_out && counts), S3R_ERR_NULL, "s3r_adamw_state: NULL pointer");
  for (int i = 0; i < n; ++i) {
    S3R_REQUIRE(counts[i] >= 0 && counts[i] < (1ll << 33), S3R_ERR_SHAPE, "s3r_adamw_state: %lld elements", (long long)counts[i]);
    S3R_REQUIRE(counts[i] == 0 || (m[i] && v[i] && m_exponents[i] && v_exponents[i] && m_out[i] && v_out[i]), S3R_ERR_NULL, "s3r_adamw_state: NULL pointer");
    S3R_REQUIRE((reinterpret_cast<uintptr_t>(m_out[i]) | reinterpret_cast<uintptr_t>(v_out[i])) % 4 == 0, S3R_ERR_ALIGNMENT, "s3r_adamw_state: elements must be aligned");
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  static thread_local StateParams<kAdamMax> p;
  StateParams<kAdamFew> few;
  p.n = 0;
  int64_t ctas = 0;
  for (int i = 0; i <= n; ++i) {
    if (p.n && (i == n || p.n == kAdamMax)) {
      int rc;
      if (p.n <= kAdamFew) {
        few.n = p.n;
        std::copy_n(p.t, p.n, few.t);
        fill_starts(few.starts, p.t, p.n, ctas);
        rc = launch(adamw_state_kernel<kAdamFew>, static_cast<unsigned>(ctas), kAdamThreads, 0, st, few);
      } else {
        fill_starts(p.starts, p.t, p.n, ctas);
        rc = launch(adamw_state_kernel<kAdamMax>, static_cast<unsigned>(ctas), kAdamThreads, 0, st, p);
      }
      if (rc) return rc;
      p.n = 0;
      ctas = 0;
    }
    if (i == n || counts[i] == 0) continue;
    p.t[p.n++] = {static_cast<const uint8_t*>(m[i]), static_cast<const uint8_t*>(v[i]), m_exponents[i], v_exponents[i], m_out[i], v_out[i], counts[i], ctas,
                  at_16({m[i], v[i], m_out[i], v_out[i]}) ? kAdamVector : 0u};
    ctas += (counts[i] + kAdamPerCta - 1) / kAdamPerCta;
    S3R_REQUIRE(ctas < (1ll << 31), S3R_ERR_TOO_LARGE, "s3r_adamw_state: grid too large");
  }
  return 0;
}
