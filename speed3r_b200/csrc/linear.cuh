// Products of bf16 or fp16 tiles with what follows them in their epilogue: the kernel, and its launch.
#pragma once

#include <climits>
#include <cmath>

#include "pairs.cuh"

namespace s3r {

// ---------------------------------------------------------------------------------------------------------------------
// activations
// ---------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 fast_rcp2(float2 x) { return make_float2(fast_rcp(x.x), fast_rcp(x.y)); }
__device__ __forceinline__ float2 exp2_2(float2 x) { return make_float2(fast_exp2(x.x), fast_exp2(x.y)); }
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// u = act(z), and its slope.
// GELU: z Phi(z) with Phi from erfc as Abramowitz and Stegun give it (7.1.26: a polynomial of degree 5 in t = 1 / (1 + p |x|), times exp(-x^2),
// off by 1.5e-7 at most, so Phi by 7.5e-8): one exponential, which the slope's density shares, one reciprocal and eleven packed operations per
// pair.  A polynomial without either would need degree 12 for that and take as many.
// GELU by tanh: z sigmoid(2 sqrt(2 / pi) (z + 0.044715 z^3)), the same function.
template <int ACT, bool SLOPE>
__device__ __forceinline__ float2 activate(float2 z, float2& slope) {
  if constexpr (ACT == S3R_ACT_NONE) {
    if (SLOPE) slope = both(1.f);
    return z;
  } else if constexpr (ACT == S3R_ACT_GELU) {
    const float2 a = make_float2(fabsf(z.x), fabsf(z.y));
    const float2 t = fast_rcp2(ffma2(a, both(0.23164190f), both(1.f)));             // 0.3275911 / sqrt(2)
    const float2 e = exp2_2(fmul2(fmul2(z, z), both(-0.72134752f)));                // exp(-z^2 / 2)
    float2 h = both(-0.530702715f);                                                 // the halved coefficients, negative
    h = ffma2(h, t, both(0.726576014f));
    h = ffma2(h, t, both(-0.710706868f));
    h = ffma2(h, t, both(0.142248368f));
    h = ffma2(h, t, both(-0.127414796f));
    h = ffma2(fmul2(h, t), e, both(0.5f));                                          // 1/2 - Phi(-|z|)
    if (SLOPE) {
      const float2 above = make_float2(copysignf(h.x, z.x), copysignf(h.y, z.y));
      slope = fadd2(ffma2(fmul2(z, both(0.398942280f)), e, above), both(0.5f));
    }
    return ffma2(a, h, fmul2(z, both(0.5f)));
  } else {
    const float2 q = fmul2(z, z);
    const float2 arg = ACT == S3R_ACT_SILU ? fmul2(z, both(-1.44269504f)) : fmul2(z, ffma2(q, both(-0.102943240f), both(-2.30220819f)));
    const float2 p = fast_rcp2(fadd2(exp2_2(arg), both(1.f)));
    const float2 u = fmul2(z, p);
    if (SLOPE) {
      // p + u (1 - p) times the argument's own slope: 1, or 2 sqrt(2 / pi) (1 + 3 * 0.044715 z^2), last, for it may be huge where 1 - p is 0.  z^2
      // is infinite from |z| = 2^64 on, and 0 times that NaN: it stays at 2^100, from where on u (1 - p) has long been 0 on either side.
      const float2 rest = fadd2(both(1.f), make_float2(-p.x, -p.y)), finite = make_float2(fminf(q.x, 0x1p100f), fminf(q.y, 0x1p100f));
      slope = ACT == S3R_ACT_SILU ? ffma2(u, rest, p) : ffma2(fmul2(u, rest), ffma2(finite, both(0.214064488f), both(1.59576912f)), p);
    }
    return u;
  }
}
// f(the activation as a constant)
template <typename F>
inline __host__ __device__ int with_act(int act, F f) {
  if (act == S3R_ACT_NONE) return f(std::integral_constant<int, S3R_ACT_NONE>());
  if (act == S3R_ACT_GELU) return f(std::integral_constant<int, S3R_ACT_GELU>());
  if (act == S3R_ACT_GELU_TANH) return f(std::integral_constant<int, S3R_ACT_GELU_TANH>());
  return f(std::integral_constant<int, S3R_ACT_SILU>());
}

// An operand of a product: `rows` of the result's rows or columns, `k` steps of the contraction; pitch in elements.
struct LinOperand {
  const void* data;
  int64_t pitch;
  bool turned;
};
struct LinParams;
// Each kind of kernel in a file of its own, which are compiled side by side.
int linear_narrow(const LinOperand& a, const LinOperand& b, int64_t k, bool bf16, const LinParams& p, cudaStream_t st);          // 16-bit result, nothing added
int linear_wide(const LinOperand& a, const LinOperand& b, int64_t k, bool bf16, const LinParams& p, cudaStream_t st);            // fp32 result, nothing added
int linear_added(const LinOperand& a, const LinOperand& b, int64_t k, bool bf16, const LinParams& p, cudaStream_t st);           // with a residual
int linear_dz(const LinOperand& a, const LinOperand& b, int64_t k, bool bf16, const LinParams& p, cudaStream_t st);
int linear_partial(const LinOperand& a, const LinOperand& b, int64_t k, bool bf16, const LinParams& p, cudaStream_t st);         // parts of the contraction, fp32

// ---------------------------------------------------------------------------------------------------------------------
// product on tcgen05: persistent CTAs (pairs of them), the contraction in steps of 64 through a ring of TMA copies, the sums of two tiles in
// tensor memory so that one is written out while the next is summed.  One warp copies, one issues the products, eight take the sums, 32 rows
// and half of the columns each.
// Either operand lies with the contraction contiguous ([rows][k]: x, W of the forward, dz of dx) or turned ([k][rows]: W of dx, dz and x of dW);
// a turned one comes in boxes of 64 rows x 64 steps and is read through the other form of the matrix descriptor.
//
// Bound: the tensor cores, and at full size the power they take.  64 512 x 4096 x 1024 in bf16: the products alone 322 us (1680 TFLOP/s), with GELU
// 388 at first and 458 at the clock that power leaves.  What the epilogue takes must stay below the products' time: alone (K = 64) it is 103 us for a sum that
// is only rounded, 186 with SiLU, 234 with GELU, 376 with an fp32 residual, 391 for dz with GELU's slope and a sum over rows, of which the memory
// traffic is 80, 80, 80, 320 and 161 (dz: dy read, dz written).  dz is the one that issues most: 40 % of all cycles, the tensor cores busy in 65 %
// (forward with GELU 83 %).
// Roundings: the tensor cores cut every addition to an fp32 sum off towards zero, so that over K = 4096 terms z is 4.4e-6 too small (a library's fp32
// result of the same product, too), and d_scale with it.  dz is rounded to the operands' type, as its two products take it: half a step more in
// dx and dW; two halves of 16 bits would keep it, for twice both products.
// Tried, and slower: sixteen summing warps, which spill (166 -> 237, dz 375 -> 494); two pieces of output per warp where nothing is read beside the
// sums (166 -> 172); two sets of dz's sums in registers (373 -> 395).
// ---------------------------------------------------------------------------------------------------------------------
// Warps 0 and 1 feed, the last eight take the sums.  Two in between do nothing: without them every kind of epilogue took 4 to 10 % longer.
constexpr int kLinFirst = 4, kLinWarps = 8, kLinThreads = 32 * (kLinFirst + kLinWarps);
constexpr int kLinPiece = 4096;                                    // a warp's piece of the output: 32 rows of 128 bytes
constexpr int kLinStep = 64;                                       // elements of the contraction per stage: 128 bytes
constexpr int kNoOther = -1, kAnyAct = -1, kPartial = -2;

struct LinParams {
  const void *bias, *scale, *other;    // other: the residual | dy
  void* out;
  float *bias_sums, *scale_sums;       // [32-row blocks, N]: sums of dz and of dy * u
  int64_t M, rows, out_pitch;          // rows: kPartial's, of a
  int N, steps, m_tiles, n_tiles;
  int parts, row_tiles, part_steps;           // kPartial: tiles of a's rows, steps of a part; m_tiles is that of all parts, M their rows
  int bias_type, scale_type, other_type, out_type, act;
  uint32_t idesc, a_turned, b_turned, copy_out, other_vectors;         // other's rows: in vectors of 16 bytes (the residual), in pairs (dy)
  uint32_t other_copied;               // dy | the residual by TMA
  uint32_t* status;
};

// PIECES: per summing warp
template <int TN, int CTAS, int PIECES>
struct LinCfg {
  static constexpr int kABytes = 128 * 128, kBBytes = TN / CTAS * 128, kBytes = kABytes + kBBytes;
  static constexpr int kRing = 196608 - kLinWarps * PIECES * kLinPiece, kStages = kRing / kBytes > 6 ? 6 : kRing / kBytes;
  static constexpr int kOut = kStages * kBytes, kColumns = kOut + kLinWarps * PIECES * kLinPiece;
  static constexpr int kSpan = TN / 2 < 64 ? 64 : TN / 2;       // columns of an epilogue warp: whole pieces
  static constexpr int kSmem = kColumns + kLinWarps * kSpan * 8 + 1024;
};

struct LinCtl {
  uint64_t full[6], empty[6], acc_full[2], acc_empty[2], drained, pause, piece_full[kLinWarps][2];
  uint32_t tmem_base, abort_flag;
};

// How long a tile's sums are waited for: a step takes about 0.25 us, and a contraction may have 33 million of them.
__device__ __forceinline__ uint64_t tile_limit_ns(int steps) { return 1000000000ull + 1000ull * static_cast<uint32_t>(steps); }

// kind::f16 with fp32 sums; a_type, b_type: 0 fp16, 1 bf16
constexpr uint32_t umma_idesc_half(uint32_t M, uint32_t N, uint32_t bf16, uint32_t a_turned, uint32_t b_turned) {
  return (1u << 4) | (bf16 << 7) | (bf16 << 10) | (a_turned << 15) | (b_turned << 16) | ((N >> 3) << 17) | ((M >> 4) << 24);
}
// Four k-steps of 16.
#define S3R_LIN_K4(group)                                                    \
  asm volatile(                                                              \
      "{\n\t.reg .pred p, pt;\n\t.reg .b64 a, b;\n\t"                        \
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.u32 pt, 0, 0;\n\t"                   \
      "tcgen05.mma.cta_group::" group ".kind::f16 [%0], %1, %2, %3, p;\n\t"  \
      "add.s64 a, %1, %5;\n\tadd.s64 b, %2, %6;\n\t"                         \
      "tcgen05.mma.cta_group::" group ".kind::f16 [%0], a, b, %3, pt;\n\t"   \
      "add.s64 a, a, %5;\n\tadd.s64 b, b, %6;\n\t"                           \
      "tcgen05.mma.cta_group::" group ".kind::f16 [%0], a, b, %3, pt;\n\t"   \
      "add.s64 a, a, %5;\n\tadd.s64 b, b, %6;\n\t"                           \
      "tcgen05.mma.cta_group::" group ".kind::f16 [%0], a, b, %3, pt;\n\t}"  \
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accum), "l"(a_step), "l"(b_step) \
      : "memory")
template <int CTAS>
__device__ __forceinline__ void umma_half_k4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accum, uint64_t a_step, uint64_t b_step) {
  if constexpr (CTAS == 2) S3R_LIN_K4("2");
  else S3R_LIN_K4("1");
}

// ---- what is read beside the sums, as it lies in memory: 32 words of fp32, 16 of a 16-bit type ----------------------------
// 32 columns of a lane's row from element `at` on, of which n (any number) are there; `vectors`: rows begin at multiples of 16 bytes
template <int TYPE, int WORDS>
__device__ __forceinline__ void load_row(uint32_t (&o)[WORDS], const void* p, int64_t at, int n, bool vectors) {
  constexpr int kPer = TYPE == S3R_F32 ? 1 : 2;                    // elements of a word
  const char* from = static_cast<const char*>(p) + at * type_bytes(TYPE);
  if (n >= 32 && vectors) {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(from) + i / 4);
      o[i] = v.x, o[i + 1] = v.y, o[i + 2] = v.z, o[i + 3] = v.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < WORDS; ++i) {
    o[i] = 0;
    if (kPer == 1) {
      if (i < n) o[i] = __ldg(reinterpret_cast<const uint32_t*>(from) + i);
    } else {
      if (2 * i < n) o[i] = __ldg(reinterpret_cast<const uint16_t*>(from) + 2 * i);
      if (2 * i + 1 < n) o[i] |= static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(from) + 2 * i + 1)) << 16;
    }
  }
}
// Rows row, row + 8, row + 16, row + 24, of either of four times eight columns two from col on, row by row; `pairs`: rows begin at multiples of two
// elements
template <int TYPE, int WORDS>
__device__ __forceinline__ void load_square(uint32_t (&o)[WORDS], const void* p, int64_t row, int64_t M, int N, int col, int end, bool pairs) {
  constexpr int kPer = WORDS / 16;                                 // words of a pair
  const char* from = static_cast<const char*>(p) + (row * N + col) * type_bytes(TYPE);
  const int64_t pitch = 8ll * N * type_bytes(TYPE);
  if (pairs && row + 25 <= M && col + 26 <= end) {                 // all of them are there
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const char* at = from + i * pitch + 8 * j * type_bytes(TYPE);
        uint32_t* to = o + (i * 4 + j) * kPer;
        if constexpr (TYPE == S3R_F32) {
          const uint2 v = __ldg(reinterpret_cast<const uint2*>(at));
          to[0] = v.x, to[1] = v.y;
        } else {
          to[0] = __ldg(reinterpret_cast<const uint32_t*>(at));
        }
      }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const char* at = from + i * pitch + 8 * j * type_bytes(TYPE);
      uint32_t* to = o + (i * 4 + j) * kPer;
      const int n = row + 8 * i < M ? end - col - 8 * j : 0;
      to[0] = 0;
      if constexpr (TYPE == S3R_F32) {
        to[1] = 0;
        if (n > 0) to[0] = __ldg(reinterpret_cast<const uint32_t*>(at));
        if (n > 1) to[1] = __ldg(reinterpret_cast<const uint32_t*>(at) + 1);
      } else {
        if (n > 0) to[0] = __ldg(reinterpret_cast<const uint16_t*>(at));
        if (n > 1) to[0] |= static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(at) + 1)) << 16;
      }
    }
}
// elements k and k + 1 of 32 (k even, a constant)
template <int TYPE, int WORDS>
__device__ __forceinline__ float2 other_pair(const uint32_t (&o)[WORDS], int k) {
  if constexpr (TYPE == S3R_F32) return make_float2(__uint_as_float(o[k]), __uint_as_float(o[k + 1]));
  else if constexpr (TYPE == S3R_BF16) return make_float2(bf16_lo(o[k / 2]), bf16_hi(o[k / 2]));
  else if constexpr (TYPE == S3R_F16) return make_float2(half_lo(o[k / 2]), half_hi(o[k / 2]));
  else return make_float2(0.f, 0.f);
}
// 16 pairs as they are stored
template <bool WIDE, int WORDS>
__device__ __forceinline__ void pack_pairs(uint32_t (&x)[WORDS], const float2 (&y)[16], int type) {
  if constexpr (WIDE) {
#pragma unroll
    for (int k = 0; k < 16; ++k) x[2 * k] = __float_as_uint(y[k].x), x[2 * k + 1] = __float_as_uint(y[k].y);
  } else if (type == S3R_BF16) {
#pragma unroll
    for (int k = 0; k < 16; ++k) x[k] = pack_bf16(y[k].x, y[k].y);
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k) x[k] = pack_half(y[k].x, y[k].y);
  }
}

// every 32nd element from `col` on, as it lies in memory, 0 from element `end` on
template <int N>
__device__ __forceinline__ void load_factors(uint32_t (&f)[N], const void* p, int type, int end, int col) {
  with_width(type, [&](auto width) {
    const auto* from = static_cast<const decltype(width)*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = col + 32 * i < end ? __ldg(from + col + 32 * i) : 0;
  });
}

// four 8 x 8 matrices of 16-bit elements: lane l has elements 2 (l % 4) and the next of row l / 4, and gives the address of row l % 8 of matrix l / 8
__device__ __forceinline__ void stsm_x4(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r0), "r"(r1), "r"(r2), "r"(r3) : "memory");
}
__device__ __forceinline__ void bulk_wait_read_but_one() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }

// Sums over the eight lanes that share columns, of eight columns each: halves change hands, so that every lane ends with one column, number
// 8 (lane >> 3) + 2 (lane & 3) + (lane >> 2 & 1) of 32.
__device__ __forceinline__ float column_sum(const float2 (&d)[4], int lane) {
  const bool up = lane & 16, high = lane & 8, odd = lane & 4;
  float2 a[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float2 keep = up ? d[2 + k] : d[k], give = up ? d[k] : d[2 + k];
    a[k] = fadd2(keep, make_float2(__shfl_xor_sync(0xffffffffu, give.x, 16), __shfl_xor_sync(0xffffffffu, give.y, 16)));
  }
  const float2 keep = high ? a[1] : a[0], give = high ? a[0] : a[1];
  const float2 b = fadd2(keep, make_float2(__shfl_xor_sync(0xffffffffu, give.x, 8), __shfl_xor_sync(0xffffffffu, give.y, 8)));
  return (odd ? b.y : b.x) + __shfl_xor_sync(0xffffffffu, odd ? b.x : b.y, 4);
}

// ACT: the activation, kAnyAct: p.act, kPartial: none, and tile m of part s is number s * row_tiles + m.  OTHER: type of the residual | of dy, kNoOther: there is none.  WIDE: the result is fp32.
// DZ: 1 out = dz from dy, and its sums over rows, in place of the forward's result; 2 the same with a scale, and the sums for that
template <int TN, int CTAS, int ACT, int OTHER, bool WIDE, int DZ>
__global__ void __launch_bounds__(kLinThreads) linear_kernel(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb,
                                                             const __grid_constant__ CUtensorMap mo, const __grid_constant__ CUtensorMap md, const __grid_constant__ LinParams p) {
  using C = LinCfg<TN, CTAS, DZ || OTHER != kNoOther ? 2 : 1>;
  extern __shared__ char raw_smem[];
  __shared__ LinCtl ctl;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CTAS == 2 ? static_cast<int>(blockIdx.x & 1) : 0;          // a cluster is two consecutive CTAs
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&ctl.full[s], 1);
      mbar_init(&ctl.empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&ctl.acc_full[s], 1);
      mbar_init(&ctl.acc_empty[s], CTAS * kLinWarps);
    }
    if (OTHER != kNoOther)
      for (int s = 0; s < 2 * kLinWarps; ++s) mbar_init(&ctl.piece_full[s / 2][s % 2], 1);
    mbar_init(&ctl.drained, 1);
    mbar_init(&ctl.pause, 1);
    ctl.abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    if constexpr (CTAS == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem_base)), "r"(2 * TN) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tmem_alloc(&ctl.tmem_base, 2 * TN);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  sync_pair<CTAS>();
  tc_fence_after();
  griddep_wait();
  griddep_launch();
  const uint32_t tmem = ctl.tmem_base;
  volatile uint32_t* abort_flag = &ctl.abort_flag;
  const int tiles = p.m_tiles * p.n_tiles, steps = p.steps, first = blockIdx.x / CTAS, stride = gridDim.x / CTAS;
  // tile = m * n_tiles + n, walked without a division per tile
  struct Tile {
    int m, n;
  };
  const Tile begin = {first / p.n_tiles, first % p.n_tiles}, step_by = {stride / p.n_tiles, stride % p.n_tiles};
  auto advance = [&](Tile& t) {
    t.m += step_by.m;
    t.n += step_by.n;
    if (t.n >= p.n_tiles) t.n -= p.n_tiles, ++t.m;
  };
  const uint32_t base = smem_u32(smem);

  if (warp == 0) {
    int n = 0;                                                     // copies so far
    bool ok = true;
    const bool leader = elect_one_sync();
    Tile at = begin;
    for (int tile = first; tile < tiles && ok; tile += stride, advance(at)) {
      const int part = ACT == kPartial ? at.m / p.row_tiles : 0;
      const int m0 = ((at.m - part * p.row_tiles) * CTAS + rank) * 128, n0 = at.n * TN + rank * (TN / CTAS);
      const int k0 = part * p.part_steps, k1 = ACT == kPartial ? min(steps, k0 + p.part_steps) : steps;
      for (int k = k0; k < k1; ++k, ++n) {
        const int s = n % C::kStages;
        ok = mbar_wait_warp(&ctl.empty[s], (n / C::kStages & 1) ^ 1, abort_flag);
        if (!ok) break;
        if (leader) {
          const uint32_t bar = first_cta<CTAS>(&ctl.full[s]);      // both CTAs' copies complete the first one's barrier
          if (rank == 0) mbar_expect_tx(&ctl.full[s], CTAS * C::kBytes);
          const uint32_t a = base + s * C::kBytes, b = a + C::kABytes;
          if (!p.a_turned) {
            tma_load_2d<CTAS>(a, &ma, bar, k * kLinStep, m0);
          } else {
            tma_load_2d<CTAS>(a, &ma, bar, m0, k * kLinStep);
            tma_load_2d<CTAS>(a + 8192, &ma, bar, m0 + 64, k * kLinStep);
          }
          if (!p.b_turned) {
            tma_load_2d<CTAS>(b, &mb, bar, k * kLinStep, n0);
          } else {
            tma_load_2d<CTAS>(b, &mb, bar, n0, k * kLinStep);
            if constexpr (TN / CTAS == 128) tma_load_2d<CTAS>(b + 8192, &mb, bar, n0 + 64, k * kLinStep);
          }
        }
        __syncwarp();
      }
    }
    if (!ok) {                                                     // copies in flight land before the CTA's memory is given away
      volatile uint32_t dummy = 0;
      for (int i = n - C::kStages < 0 ? 0 : n - C::kStages; rank == 0 && i < n; ++i) {
        dummy = 0;
        mbar_wait(&ctl.full[i % C::kStages], i / C::kStages & 1, &dummy);
      }
      dummy = 0;
      mbar_wait_limit(&ctl.pause, 0, &dummy, 10000000ull);         // the second CTA does not see its own land: 10 ms
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const bool leader = elect_one_sync();
      // along a row 32 bytes per k-step; turned: 16 rows of 128 bytes, and the next 64 rows of the operand 8 KB further
      const uint64_t a_step = p.a_turned ? 128 : 2, b_step = p.b_turned ? 128 : 2;
      const uint32_t a_far = p.a_turned ? 8192 : 16, b_far = p.b_turned ? 8192 : 16;
      int n = 0, done = 0;
      bool ok = true;
      Tile at = begin;
      for (int tile = first; tile < tiles && ok; tile += stride, ++done, advance(at)) {
        const int buf = done & 1, k0 = ACT == kPartial ? at.m / p.row_tiles * p.part_steps : 0, count = ACT == kPartial ? min(steps - k0, p.part_steps) : steps;
        ok = mbar_wait_warp(&ctl.acc_empty[buf], (done >> 1 & 1) ^ 1, abort_flag);
        tc_fence_after();
        for (int k = 0; k < count && ok; ++k, ++n) {
          const int s = n % C::kStages;
          ok = mbar_wait_warp(&ctl.full[s], n / C::kStages & 1, abort_flag);
          if (!ok) break;
          tc_fence_after();
          if (leader) {
            umma_half_k4<CTAS>(tmem + buf * TN, umma_desc_sw128(base + s * C::kBytes, 1024, a_far),
                               umma_desc_sw128(base + s * C::kBytes + C::kABytes, 1024, b_far), p.idesc, k > 0, a_step, b_step);
            umma_commit(&ctl.empty[s], Ctas<CTAS>());
            if (k == count - 1) umma_commit(&ctl.acc_full[buf], Ctas<CTAS>());
          }
          __syncwarp();
        }
      }
      if (!ok) {
        if (leader) umma_commit(&ctl.drained, Ctas<CTAS>());
        __syncwarp();
        volatile uint32_t dummy = 0;
        mbar_wait(&ctl.drained, 0, &dummy);                        // let issued products drain before tensor memory is freed
      }
    }
  } else if (warp >= kLinFirst) {
    if constexpr (!DZ) {
      const int me = warp - kLinFirst, quarter = warp & 3, from = (me >> 2) * C::kSpan;      // lanes 32 * quarter .. of tensor memory; its first column
      float* factors = reinterpret_cast<float*>(smem + C::kColumns) + me * 2 * C::kSpan;     // scales and biases of its columns
      constexpr int per = WIDE ? 32 : 64;                            // columns of a piece
      constexpr int kMine = C::kSpan / 32, kPieces = OTHER == kNoOther ? 1 : 2;
      // A residual of the result's size comes by TMA into the piece that the sum leaves from, a piece ahead; rows that a lane reads from memory itself,
      // 16 bytes of 32 lines at a time, took 1092 us for 64 512 x 4096 x 1024 in fp32 where this way takes 575.  Other residuals are
      // read 32 columns ahead.
      constexpr bool kInPlace = OTHER != kNoOther && (OTHER == S3R_F32) == WIDE;
      const bool by_copy = kInPlace && p.other_copied;
      // What the next tile needs is asked for a tile ahead.
      uint32_t scales[kMine], biases[kMine];
      uint32_t o[OTHER == kNoOther ? 1 : OTHER == S3R_F32 ? 32 : 16];
      auto fetch = [&](int tile, Tile at) {
        if (p.scale) load_factors(scales, p.scale, p.scale_type, tile < tiles ? p.N : 0, at.n * TN + from + lane);
        if (p.bias) load_factors(biases, p.bias, p.bias_type, tile < tiles ? p.N : 0, at.n * TN + from + lane);
      };
      auto ahead = [&](int tile, Tile at, int g) {
        if constexpr (OTHER != kNoOther) {
          if (by_copy || tile >= tiles) return;
          const int64_t row = (static_cast<int64_t>(at.m) * CTAS + rank) * 128 + quarter * 32;
          const int col = at.n * TN + from + g * 32, end = min(p.N, at.n * TN + min(from + C::kSpan, TN));
          load_row<OTHER>(o, p.other, (row + lane) * p.N + col, row + lane < p.M ? end - col : 0, p.other_vectors);
        }
      };
      // its rows, a lane each, into L2: what is asked for 32 columns ahead would wait for memory longer than those columns take
      auto soon = [&](int tile, Tile at) {
        if constexpr (OTHER != kNoOther) {
          const int64_t row = (static_cast<int64_t>(at.m) * CTAS + rank) * 128 + quarter * 32 + lane;
          const int col = at.n * TN + from, n = min(p.N, at.n * TN + min(from + C::kSpan, TN)) - col;
          if (tile >= tiles || row >= p.M) return;
          const char* first_byte = static_cast<const char*>(p.other) + (row * p.N + col) * type_bytes(OTHER);
#pragma unroll
          for (int i = 0; i < C::kSpan * type_bytes(OTHER) / 128; ++i)
            if (i * (128 / type_bytes(OTHER)) < n) asm volatile("prefetch.global.L2 [%0];" ::"l"(first_byte + 128 * i));
        }
      };
      auto piece_at = [&](uint32_t q) { return smem + C::kOut + (me * kPieces + q % kPieces) * kLinPiece; };
      // The next piece to ask for; pieces without columns are left out everywhere.
      Tile at = begin, after = begin, asked = begin;
      int asked_tile = first, asked_piece = 0;
      uint32_t asks = 0, q = 0;
      auto ask_next = [&] {
        while (asked_tile < tiles) {
          const int c0 = from + asked_piece * per, n0 = asked.n * TN;
          const bool there = c0 < TN && n0 + c0 < p.N;
          if (there && lane == 0) {
            mbar_expect_tx(&ctl.piece_full[me][asks & 1], kLinPiece);
            tma_load_2d<1>(smem_u32(piece_at(asks)), &md, smem_u32(&ctl.piece_full[me][asks & 1]), n0 + c0, (asked.m * CTAS + rank) * 128 + quarter * 32);
          }
          asks += there;
          if (++asked_piece == C::kSpan / per) {
            asked_piece = 0;
            asked_tile += stride;
            advance(asked);
          }
          if (there) return;
        }
      };
      fetch(first, at);
      soon(first, at);
      if (by_copy) {
        ask_next();
        ask_next();
      }
      ahead(first, at, 0);
      int done = 0;
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += stride, at = after, ++done) {
        const int buf = done & 1;
        const int64_t m0 = (static_cast<int64_t>(at.m) * CTAS + rank) * 128 + quarter * 32;
        const int n0 = at.n * TN;
        const int width = min(min(from + C::kSpan, TN), p.N - n0);   // columns from .. width
        __syncwarp();                                                // the last tile's factors are read
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          factors[i * 32 + lane] = p.scale ? any_value(scales[i], p.scale_type) : 1.f;
          factors[C::kSpan + i * 32 + lane] = p.bias ? any_value(biases[i], p.bias_type) : 0.f;
        }
        __syncwarp();
        advance(after);
        fetch(tile + stride, after);
        soon(tile + stride, after);
        ok = mbar_wait_warp(&ctl.acc_full[buf], done >> 1 & 1, abort_flag, tile_limit_ns(steps));
        if (!ok) break;
        tc_fence_after();
        // 32 columns' sums; when they are there, or have been used, the next 32 are asked for; the last ones free the tile's columns
        const uint32_t sums = tmem + (static_cast<uint32_t>(quarter) << 21) + buf * TN + from;
        constexpr int kSets = OTHER == kNoOther ? 2 : 1;               // what is added takes the other set's place
        uint32_t two[kSets][32];
        auto take = [&](int g) {
          if (from >= TN) return;
          tmem_ld32(sums + g * 32, two[g % kSets]);
        };
        auto taken = [&](int g) {
          if (g + 1 < kMine) {
            take(g + 1);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_first_cta<CTAS>(&ctl.acc_empty[buf]);
          }
        };
        take(0);
#pragma unroll
        for (int g = 0; g < kMine; ++g) {
          uint32_t x[WIDE ? 32 : 16];                                // as it is stored
          const bool some = from + g * 32 < width;
          const int half_piece = WIDE ? 0 : g & 1;
          char* piece = piece_at(q);
          const float *s = factors + g * 32, *b = s + C::kSpan;
          uint32_t (&v)[32] = two[g % kSets];
          tmem_ld_wait_for(v);
          if (kSets == 2) taken(g);
          if constexpr (kInPlace) {
            if (by_copy && some) {
              if (!half_piece) {
                ok = mbar_wait_warp(&ctl.piece_full[me][q & 1], q >> 1 & 1, abort_flag);
                if (!ok) break;
              }
#pragma unroll
              for (int k = 0; k < (WIDE ? 8 : 4); ++k) {
                const uint4 w = lds128(smem_u32(piece + swz128(lane, half_piece * 4 + k)));
                o[4 * k] = w.x, o[4 * k + 1] = w.y, o[4 * k + 2] = w.z, o[4 * k + 3] = w.w;
              }
              if (!half_piece && asks - q < 2) {                     // the piece before has left its place: the one behind this one comes there
                if (lane == 0) bulk_wait_read();
                __syncwarp();
                ask_next();
              }
            }
          }
          {
            float2 y[16];
            auto columns = [&](auto act) {
#pragma unroll
              for (int k = 0; k < 32; k += 4) {
                const float4 add = *reinterpret_cast<const float4*>(b + k);
                float2 slope;
                y[k / 2] = activate<decltype(act)::value, false>(fadd2(make_float2(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), make_float2(add.x, add.y)), slope);
                y[k / 2 + 1] = activate<decltype(act)::value, false>(fadd2(make_float2(__uint_as_float(v[k + 2]), __uint_as_float(v[k + 3])), make_float2(add.z, add.w)), slope);
              }
              return 0;
            };
            if constexpr (ACT == kAnyAct) with_act(p.act, columns);
            else if constexpr (ACT == kPartial) columns(std::integral_constant<int, S3R_ACT_NONE>());
            else columns(std::integral_constant<int, ACT>());
            if (OTHER != kNoOther || p.scale) {
#pragma unroll
              for (int k = 0; k < 32; k += 4) {
                const float4 f = *reinterpret_cast<const float4*>(s + k);
                const float2 lo = make_float2(f.x, f.y), hi = make_float2(f.z, f.w);
                y[k / 2] = OTHER == kNoOther ? fmul2(y[k / 2], lo) : ffma2(y[k / 2], lo, other_pair<OTHER>(o, k));
                y[k / 2 + 1] = OTHER == kNoOther ? fmul2(y[k / 2 + 1], hi) : ffma2(y[k / 2 + 1], hi, other_pair<OTHER>(o, k + 2));
              }
            }
            pack_pairs<WIDE>(x, y, p.out_type);
          }
          if (kSets == 1) taken(g);
          if (g + 1 < kMine) ahead(tile, at, g + 1);
          else ahead(tile + stride, after, 0);
          if (some) {
            if (!half_piece && !by_copy) {
              if (lane == 0) kPieces == 2 ? bulk_wait_read_but_one() : bulk_wait_read();     // the store before has left this piece
              __syncwarp();
            }
            // rows of 128 bytes, their 16-byte chunks swizzled by the row
#pragma unroll
            for (int k = 0; k < (WIDE ? 8 : 4); ++k)
              *reinterpret_cast<uint4*>(piece + swz128(lane, half_piece * 4 + k)) = make_uint4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
            if (WIDE || half_piece || from + g * 32 + 32 >= width) {
              ++q;
              const int c0 = from + (g - half_piece) * 32;
              if (p.copy_out) {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                  if (m0 < p.M) tma_store_2d(&mo, smem_u32(piece), n0 + c0, static_cast<int>(m0));
                  bulk_commit();
                }
              } else {
                __syncwarp();
                constexpr int kSize = WIDE ? 4 : 2;
                store_lines<WIDE ? S3R_F32 : S3R_BF16>(static_cast<char*>(p.out) + (m0 * p.out_pitch + n0 + c0) * kSize, p.out_pitch * kSize, piece,
                                                       min(per, width - c0), static_cast<int>(min(static_cast<int64_t>(32), p.M - m0)), lane);
                __syncwarp();                                        // read before the next piece is written
              }
            }
          }
        }
      }
      if (!ok) {                                                     // copies in flight land before the CTA's memory is given away
        volatile uint32_t dummy;
        for (uint32_t k = asks > 2 ? asks - 2 : 0; k < asks; ++k) {
          dummy = 0;
          mbar_wait(&ctl.piece_full[me][k & 1], k >> 1 & 1, &dummy);
        }
      }
      if (lane == 0) bulk_wait_all();
      if (!ok && lane == 0) atomicOr(p.status, kStatusWaitTimeout);
    } else {
      const int me = warp - kLinFirst, quarter = warp & 3, from = (me >> 2) * C::kSpan;
      float* factors = reinterpret_cast<float*>(smem + C::kColumns) + me * 2 * C::kSpan;
      constexpr int kMine = C::kSpan / 32, kPerTile = C::kSpan / 64;
      const int r = lane >> 2, c = 2 * (lane & 3);                   // rows r, r + 8, r + 16, r + 24, of every eight columns two from c on
      // dy of 16 bits comes by TMA, 32 rows x 64 columns into one of two pieces, where dz takes its place and leaves by TMA as well; half a piece
      // ahead.  In the layout of tensor memory's 16 x 256 bits a lane's elements are those of 8 x 8 matrices.  Other dy is read from memory, fp32
      // 32 columns ahead.
      const bool by_copy = OTHER != S3R_F32 && p.other_copied;
      uint32_t scales[kMine], biases[kMine];
      uint32_t o[OTHER == S3R_F32 ? 32 : 16];
      auto fetch = [&](int tile, Tile at) {
        if (DZ == 2) load_factors(scales, p.scale, p.scale_type, tile < tiles ? p.N : 0, at.n * TN + from + lane);
        if (p.bias) load_factors(biases, p.bias, p.bias_type, tile < tiles ? p.N : 0, at.n * TN + from + lane);
      };
      auto ahead = [&](int tile, Tile at, int g) {
        if (OTHER != S3R_F32 || tile >= tiles) return;
        const int64_t row = (static_cast<int64_t>(at.m) * CTAS + rank) * 128 + quarter * 32;
        load_square<OTHER>(o, p.other, row + r, p.M, p.N, at.n * TN + from + g * 32 + c, min(p.N, at.n * TN + min(from + C::kSpan, TN)), p.other_vectors);
      };
      auto soon = [&](int tile, Tile at) {                           // its rows, a lane each, into L2
        const int64_t row = (static_cast<int64_t>(at.m) * CTAS + rank) * 128 + quarter * 32 + lane;
        const int col = at.n * TN + from, n = min(p.N, at.n * TN + min(from + C::kSpan, TN)) - col;
        if (tile >= tiles || row >= p.M) return;
        const char* first_byte = static_cast<const char*>(p.other) + (row * p.N + col) * type_bytes(OTHER);
#pragma unroll
        for (int i = 0; i < C::kSpan * type_bytes(OTHER) / 128; ++i)
          if (i * (128 / type_bytes(OTHER)) < n) asm volatile("prefetch.global.L2 [%0];" ::"l"(first_byte + 128 * i));
      };
      auto piece_at = [&](uint32_t q) { return smem + C::kOut + (me * 2 + (q & 1)) * kLinPiece; };
      // piece h of a tile, number q of this warp's: asked for; pieces without columns are left out everywhere
      auto has = [&](Tile at, int h) { return from + h * 64 < TN && at.n * TN + from + h * 64 < p.N; };
      auto ask = [&](Tile at, int h, uint32_t q) {
        if (lane == 0) {
          mbar_expect_tx(&ctl.piece_full[me][q & 1], kLinPiece);
          tma_load_2d<1>(smem_u32(piece_at(q)), &md, smem_u32(&ctl.piece_full[me][q & 1]), at.n * TN + from + h * 64, (at.m * CTAS + rank) * 128 + quarter * 32);
        }
      };
      Tile at = begin, after = begin, asked = begin;                 // asked, asked_tile, asked_piece: the next piece to ask for
      int asked_tile = first, asked_piece = 0;
      uint32_t asks = 0, q = 0;
      auto ask_next = [&] {
        while (asked_tile < tiles) {
          const bool there = has(asked, asked_piece);
          if (there) ask(asked, asked_piece, asks++);
          if (++asked_piece == kPerTile) {
            asked_piece = 0;
            asked_tile += stride;
            advance(asked);
          }
          if (there) return;
        }
      };
      fetch(first, at);
      soon(first, at);
      if (by_copy) {
        ask_next();
        ask_next();
      }
      ahead(first, at, 0);
      int done = 0;
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += stride, at = after, ++done) {
        const int buf = done & 1;
        const int64_t m0 = (static_cast<int64_t>(at.m) * CTAS + rank) * 128 + quarter * 32;
        const int n0 = at.n * TN;
        const int width = min(min(from + C::kSpan, TN), p.N - n0);   // columns from .. width
        __syncwarp();                                                // the last tile's factors are read
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          if (DZ == 2) factors[i * 32 + lane] = any_value(scales[i], p.scale_type);
          factors[C::kSpan + i * 32 + lane] = p.bias ? any_value(biases[i], p.bias_type) : 0.f;
        }
        __syncwarp();
        advance(after);
        fetch(tile + stride, after);
        soon(tile + stride, after);
        ok = mbar_wait_warp(&ctl.acc_full[buf], done >> 1 & 1, abort_flag, tile_limit_ns(steps));
        if (!ok) break;
        tc_fence_after();
        const uint32_t sums = tmem + (static_cast<uint32_t>(quarter) << 21) + buf * TN + from;
        uint32_t v[32];
        if (from < TN) tmem_ld_32x32(sums, v);
        const bool whole = m0 + 32 <= p.M;
#pragma unroll
        for (int g = 0; g < kMine; ++g) {
          const bool some = from + g * 32 < width;
          char* piece = piece_at(q);
          // matrices (i, j): rows 8 i .. of columns 8 j ..; lane l gives the address of row l % 8 of matrix l / 8
          auto matrix_row = [&](int j) { return smem_u32(piece + swz128(lane, (g & 1) * 4 + j)); };
          tmem_ld_wait_for(v);
          if (OTHER != S3R_F32 && some) {
            if (by_copy) {
              if (!(g & 1)) ok = mbar_wait_warp(&ctl.piece_full[me][q & 1], q >> 1 & 1, abort_flag);
              if (!ok) break;
#pragma unroll
              for (int j = 0; j < 4; ++j) ldsm_x4(o[j], o[4 + j], o[8 + j], o[12 + j], matrix_row(j));
            } else {
              load_square<OTHER>(o, p.other, m0 + r, p.M, p.N, n0 + from + g * 32 + c, n0 + width, p.other_vectors);
            }
          }
          float2 y[16], db[4], ds[4];
          const float *s = factors + g * 32, *b = s + C::kSpan;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = *reinterpret_cast<const float2*>(s + 8 * j + c), add = *reinterpret_cast<const float2*>(b + 8 * j + c);
            ds[j] = both(0.f);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int k = (i >> 1) * 16 + j * 4 + (i & 1) * 2;
              float2 slope;
              const float2 u = activate<ACT, true>(fadd2(make_float2(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), add), slope);
              const float2 dy = other_pair<OTHER>(o, (i * 4 + j) * 2);
              y[i * 4 + j] = fmul2(DZ == 2 ? fmul2(dy, f) : dy, slope);
              if (DZ == 2) ds[j] = ffma2(dy, whole || m0 + r + 8 * i < p.M ? u : both(0.f), ds[j]);
            }
          }
          if (!whole) {                                              // a row that is not there has dy = 0, but may have any z
#pragma unroll
            for (int k = 0; k < 16; ++k)
              if (m0 + r + 8 * (k >> 2) >= p.M) y[k] = both(0.f);
          }
          if (g + 1 < kMine) {
            if (from < TN) tmem_ld_32x32(sums + g * 32 + 32, v);
            ahead(tile, at, g + 1);
          } else {                                                   // this warp's sums are in registers
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_first_cta<CTAS>(&ctl.acc_empty[buf]);
            ahead(tile + stride, after, 0);
          }
          const int col = from + g * 32 + (lane & 24) + 2 * (lane & 3) + (lane >> 2 & 1);
          const int64_t to = (m0 >> 5) * p.N + n0 + col;
          const bool there = m0 < p.M && col < width;
          if (p.bias_sums) {
#pragma unroll
            for (int j = 0; j < 4; ++j) db[j] = fadd2(fadd2(y[j], y[4 + j]), fadd2(y[8 + j], y[12 + j]));
            const float sum = column_sum(db, lane);
            if (there) p.bias_sums[to] = sum;
          }
          if (DZ == 2 && p.scale_sums) {
            const float sum = column_sum(ds, lane);
            if (there) p.scale_sums[to] = sum;
          }
          if (!some) continue;
          if (p.out) {
            if (!(g & 1) && !by_copy) {
              if (lane == 0) bulk_wait_read_but_one();               // the store before the last has left this piece
              __syncwarp();
            }
            uint32_t x[16];
            pack_pairs<false>(x, y, p.out_type);
#pragma unroll
            for (int j = 0; j < 4; ++j) stsm_x4(matrix_row(j), x[j], x[4 + j], x[8 + j], x[12 + j]);
          }
          const bool last = (g & 1) || from + g * 32 + 32 >= width;
          if (by_copy && (!(g & 1)) && q > 0) {                      // the piece before has left its place: the one behind this one comes there
            if (lane == 0) bulk_wait_read();
            __syncwarp();
            ask_next();
          }
          if (!last) continue;
          if (p.out) {
            const int c0 = from + (g & ~1) * 32;
            if (p.copy_out) {
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                if (m0 < p.M) tma_store_2d(&mo, smem_u32(piece), n0 + c0, static_cast<int>(m0));
                bulk_commit();
              }
            } else {
              __syncwarp();
              store_lines<S3R_BF16>(static_cast<char*>(p.out) + (m0 * p.out_pitch + n0 + c0) * 2, p.out_pitch * 2, piece, min(64, width - c0),
                                    static_cast<int>(min(static_cast<int64_t>(32), p.M - m0)), lane);
            }
          }
          ++q;
        }
      }
      if (!ok) {                                                     // copies in flight land before the CTA's memory is given away
        volatile uint32_t dummy;
        for (uint32_t i = asks > 2 ? asks - 2 : 0; i < asks; ++i) {
          dummy = 0;
          mbar_wait(&ctl.piece_full[me][i & 1], i >> 1 & 1, &dummy);
        }
      }
      if (lane == 0) bulk_wait_all();
      if (!ok && lane == 0) atomicOr(p.status, kStatusWaitTimeout);
    }
  }
  tc_fence_before();
  __syncthreads();
  sync_pair<CTAS>();                                               // the other CTA's products and arrivals reach this one's memory
  if (warp == 1) tmem_free<CTAS>(tmem, 2 * TN);
}

static int operand_map(CUtensorMap* map, const LinOperand& o, int64_t rows, int64_t k, uint32_t box_rows, bool bf16) {
  const uint64_t dims[2] = {static_cast<uint64_t>(o.turned ? rows : k), static_cast<uint64_t>(o.turned ? k : rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(o.pitch) * 2};
  const uint32_t box[2] = {64, o.turned ? 64 : box_rows};
  return make_tensor_map(map, o.data, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
}

// rows of a part, which are whole tiles
inline int64_t part_rows(int64_t rows, int ctas) { return (rows + 128 * ctas - 1) / (128 * ctas) * (128 * ctas); }

template <int TN, int CTAS, int ACT, int OTHER, bool WIDE, int DZ>
static int launch_linear(const LinOperand& a, const LinOperand& b, int64_t k, bool bf16, LinParams p, cudaStream_t st) {
  using C = LinCfg<TN, CTAS, DZ || OTHER != kNoOther ? 2 : 1>;
  CUtensorMap ma, mb, mo, md;
  const int64_t rows = ACT == kPartial ? p.rows : p.M;
  if (const int rc = operand_map(&ma, a, rows, k, 128, bf16)) return rc;
  if (const int rc = operand_map(&mb, b, p.N, k, TN / CTAS, bf16)) return rc;
  mo = md = ma;
  if (ACT == kPartial) p.M = part_rows(rows, CTAS) * p.parts;
  constexpr int kSize = WIDE ? 4 : 2;
  p.copy_out = (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 && p.out_pitch * kSize % 16 == 0;
  if (p.copy_out && p.out) {
    const uint64_t dims[2] = {static_cast<uint64_t>(p.N), static_cast<uint64_t>(p.M)}, strides[1] = {static_cast<uint64_t>(p.out_pitch) * kSize};
    const uint32_t box[2] = {128 / kSize, 32};
    const CUtensorMapDataType type = WIDE ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : p.out_type == S3R_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if (const int rc = make_tensor_map(&mo, p.out, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, type)) return rc;
  }
  constexpr bool kCopied = DZ ? OTHER != S3R_F32 : OTHER != kNoOther && (OTHER == S3R_F32) == WIDE;
  p.other_copied = kCopied && (reinterpret_cast<uintptr_t>(p.other) & 15) == 0 && static_cast<int64_t>(p.N) * kSize % 16 == 0 && (p.copy_out || !p.out);
  if (p.other_copied) {
    const uint64_t dims[2] = {static_cast<uint64_t>(p.N), static_cast<uint64_t>(p.M)}, strides[1] = {static_cast<uint64_t>(p.N) * kSize};
    const uint32_t box[2] = {128 / kSize, 32};
    const CUtensorMapDataType type = OTHER == S3R_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : OTHER == S3R_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if (const int rc = make_tensor_map(&md, p.other, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, type)) return rc;
  }
  p.idesc = umma_idesc_half(128 * CTAS, TN, bf16, a.turned, b.turned);
  p.a_turned = a.turned;
  p.b_turned = b.turned;
  p.steps = static_cast<int>((k + kLinStep - 1) / kLinStep);
  p.m_tiles = static_cast<int>((rows + 128 * CTAS - 1) / (128 * CTAS));
  if (ACT == kPartial) {
    p.row_tiles = p.m_tiles;
    p.part_steps = (p.steps + p.parts - 1) / p.parts;
    p.m_tiles *= p.parts;
  }
  p.n_tiles = (p.N + TN - 1) / TN;
  const int64_t tiles = static_cast<int64_t>(p.m_tiles) * p.n_tiles, at_once = sm_count() / CTAS;
  S3R_REQUIRE(tiles < (1ll << 31) - 1024, S3R_ERR_TOO_LARGE, "s3r_linear: too many tiles");
  static std::atomic<uint64_t> ready{0};
  if (attributes_missing(ready)) {
    S3R_CUDA(cudaFuncSetAttribute(linear_kernel<TN, CTAS, ACT, OTHER, WIDE, DZ>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    attributes_set(ready);
  }
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(static_cast<unsigned>((tiles < at_once ? tiles : at_once) * CTAS));
  c.blockDim = dim3(kLinThreads);
  c.dynamicSmemBytes = C::kSmem;
  c.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CTAS;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  c.attrs = attr;
  c.numAttrs = CTAS == 2 ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&c, linear_kernel<TN, CTAS, ACT, OTHER, WIDE, DZ>, ma, mb, mo, md, p), "kernel launch");
}

// The tile and the number of parts of the contraction whose waves cost least.  A wave of narrower tiles takes less, but not in proportion (the same
// rows of a).  Parts - each a tile of its own, whose sums are joined by a second kernel - pay where there are few tiles and many steps (inputs in
// HBM): 64 x 1024 x 4096 in sixteen parts 13 us, in one 21; the weight gradient 1024 x 1024 of 12 288 tokens in four 36, in one 60.
struct LinPlan {
  int width, ctas, parts, step;
};
inline LinPlan linear_plan(int64_t M, int64_t N, int64_t K, bool parts) {
  const LinPlan tiles[] = {{256, 2, 1, 640}, {128, 2, 1, 460}, {128, 1, 1, 500}, {64, 1, 1, 440}};
  const int64_t steps = (K + kLinStep - 1) / kLinStep;
  LinPlan best = {};
  double least = HUGE_VAL;
  for (const LinPlan& t : tiles)
    for (int n = 1; n <= 16; n *= 2) {
      if ((t.ctas == 2 && M <= 128) || (n > 1 && (!parts || steps < 4 * n))) continue;
      const int64_t part = (steps + n - 1) / n, used = (steps + part - 1) / part;      // parts that have steps
      const int64_t all = (M + 128 * t.ctas - 1) / (128 * t.ctas) * ((N + t.width - 1) / t.width) * used, at_once = sm_count() / t.ctas;
      // cycles: of a step (a full GPU, L2 behind it), of a tile's start and end; of the second kernel and its traffic
      const double cost = static_cast<double>((all + at_once - 1) / at_once) * (part * t.step + 1500) + (n > 1 ? 6000 + static_cast<double>(used * M) * N / 275 : 0);
      if (cost < least) least = cost, best = {t.width, t.ctas, static_cast<int>(used), t.step};
    }
  return best;
}
template <int ACT, int OTHER, bool WIDE, int DZ>
static int run_linear(const LinOperand& a, const LinOperand& b, int64_t k, bool bf16, const LinParams& p, cudaStream_t st) {
  const LinPlan t = ACT == kPartial ? linear_plan(p.rows, p.N, k, true) : linear_plan(p.M, p.N, k, false);
  if (t.ctas == 2 && t.width == 256) return launch_linear<256, 2, ACT, OTHER, WIDE, DZ>(a, b, k, bf16, p, st);
  if (t.ctas == 2) return launch_linear<128, 2, ACT, OTHER, WIDE, DZ>(a, b, k, bf16, p, st);
  if (t.width == 128) return launch_linear<128, 1, ACT, OTHER, WIDE, DZ>(a, b, k, bf16, p, st);
  return launch_linear<64, 1, ACT, OTHER, WIDE, DZ>(a, b, k, bf16, p, st);
}

}  // namespace s3r
