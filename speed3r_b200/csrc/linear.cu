// Matrix products of bf16 or fp16 with what follows them in their epilogue, forward and backward.
//   forward   z = x W^T + bias,  u = act(z),  out = residual + u * scale: one rounding, to the result's type
//   backward  du = dy * scale,  dz = du * act'(z),  d_bias = sum of dz over rows,  d_scale = sum of dy * u over rows;  dx = dz W,  dW = dz^T x
// z is not kept: where it is needed (an activation's slope, the scale's gradient) the backward makes it again, and dz is the epilogue of that product.
// The forward then writes nothing but its result, and both sums over rows see z as it was, not rounded to 16 bits.
#include <climits>

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
// off by 1.5e-7 at most, so Phi by 7.5e-8): one exponential, which the slope's density shares, one reciprocal and seven packed operations per pair.
// erff takes about three times as many, and at K = 1024 a tile's products leave 32 issue slots per value.
// GELU by tanh: z sigmoid(2 sqrt(2 / pi) (z + 0.044715 z^3)), the same function.
template <bool SLOPE>
__device__ __forceinline__ float2 activate(float2 z, int act, float2& slope) {
  if (act == S3R_ACT_GELU) {
    const float2 a = make_float2(fabsf(z.x), fabsf(z.y));
    const float2 t = fast_rcp2(ffma2(a, both(0.23164190f), both(1.f)));             // 0.3275911 / sqrt(2)
    const float2 e = exp2_2(fmul2(fmul2(z, z), both(-0.72134752f)));                // exp(-z^2 / 2)
    float2 h = both(0.530702715f);                                                  // the halved coefficients
    h = ffma2(h, t, both(-0.726576014f));
    h = ffma2(h, t, both(0.710706868f));
    h = ffma2(h, t, both(-0.142248368f));
    h = ffma2(h, t, both(0.127414796f));
    h = fmul2(fmul2(h, t), e);                                                      // Phi(-|z|)
    const float2 below = make_float2(z.x < 0.f ? h.x : 1.f - h.x, z.y < 0.f ? h.y : 1.f - h.y);
    if (SLOPE) slope = ffma2(fmul2(z, both(0.398942280f)), e, below);
    return fmul2(z, below);
  }
  if (act == S3R_ACT_NONE) {
    if (SLOPE) slope = both(1.f);
    return z;
  }
  const float2 q = fmul2(z, z);
  const float2 arg = act == S3R_ACT_SILU ? fmul2(z, both(-1.44269504f)) : fmul2(z, ffma2(q, both(-0.102943240f), both(-2.30220819f)));
  const float2 p = fast_rcp2(fadd2(exp2_2(arg), both(1.f)));
  const float2 u = fmul2(z, p);
  if (SLOPE) {
    // the argument's own slope: 1, or 2 sqrt(2 / pi) (1 + 3 * 0.044715 z^2)
    const float2 inner = act == S3R_ACT_SILU ? both(1.f) : ffma2(q, both(0.214064488f), both(1.59576912f));
    slope = ffma2(fmul2(u, inner), fadd2(both(1.f), make_float2(-p.x, -p.y)), p);
  }
  return u;
}

// ---------------------------------------------------------------------------------------------------------------------
// product on tcgen05: persistent CTAs (pairs of them), the contraction in steps of 64 through a ring of TMA copies, the sums of two tiles in
// tensor memory so that one is written out while the next is summed.  One warp copies, one issues the products, eight take the sums: 32 rows
// and half of the columns each, four rows and eight columns of every 32 x 32 per lane.
// Either operand lies with the contraction contiguous ([rows][k]: x, W of the forward, dz of dx) or turned ([k][rows]: W of dx, dz and x of dW);
// a turned one comes in boxes of 64 rows x 64 steps and is read through the other form of the matrix descriptor.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kLinWarps = 8, kLinThreads = 64 + 32 * kLinWarps, kLinPiece = 4096;       // a warp's piece of the output: 32 rows of 128 bytes
constexpr int kLinStep = 64;                                                            // elements of the contraction per stage: 128 bytes

struct LinParams {
  const void *bias, *scale, *residual, *dy;
  void* out;
  float *bias_sums, *scale_sums;       // [32-row blocks, N]: sums of dz and of dy * u
  int64_t M, out_pitch;
  int N, steps, m_tiles, n_tiles;
  int bias_type, scale_type, residual_type, dy_type, out_type, act;
  uint32_t idesc, a_turned, b_turned, copy_out, residual_pairs;      // rows of the residual | of dy in pairs of elements
  uint32_t* status;
};

template <int TN, int CTAS>
struct LinCfg {
  static constexpr int kABytes = 128 * 128, kBBytes = TN / CTAS * 128, kBytes = kABytes + kBBytes;
  static constexpr int kStages = 163840 / kBytes > 6 ? 6 : 163840 / kBytes;
  static constexpr int kOut = kStages * kBytes, kColumns = kOut + kLinWarps * kLinPiece;
  static constexpr int kSpan = TN / 2 < 64 ? 64 : TN / 2;       // columns of an epilogue warp: whole pieces
  static constexpr int kSmem = kColumns + kLinWarps * kSpan * 16 + 1024;
};

struct LinCtl {
  uint64_t full[6], empty[6], acc_full[2], acc_empty[2], drained, pause;
  uint32_t tmem_base, abort_flag;
};

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

// Two neighbours of a row, of which `n` are there; `pairs`: they begin at a multiple of both.
__device__ __forceinline__ float2 load_pair(const void* p, int type, int64_t at, int n, bool pairs) {
  float2 v = make_float2(0.f, 0.f);
  if (type == S3R_F32) {
    const float* f = static_cast<const float*>(p) + at;
    if (pairs && n == 2) return __ldg(reinterpret_cast<const float2*>(f));
    if (n > 0) v.x = __ldg(f);
    if (n > 1) v.y = __ldg(f + 1);
    return v;
  }
  const uint16_t* h = static_cast<const uint16_t*>(p) + at;
  uint32_t w = 0;
  if (pairs && n == 2) {
    w = __ldg(reinterpret_cast<const uint32_t*>(h));
  } else {
    if (n > 0) w = __ldg(h);
    if (n > 1) w |= static_cast<uint32_t>(__ldg(h + 1)) << 16;
  }
  return type == S3R_BF16 ? make_float2(bf16_lo(w), bf16_hi(w)) : make_float2(half_lo(w), half_hi(w));
}

// WIDE: the result is fp32.  DZ: out = dz from dy, and sums over rows, in place of the forward's result
template <int TN, int CTAS, bool WIDE, bool DZ>
__global__ void __launch_bounds__(kLinThreads) linear_kernel(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb,
                                                             const __grid_constant__ CUtensorMap mo, const __grid_constant__ LinParams p) {
  using C = LinCfg<TN, CTAS>;
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
      const int m0 = (at.m * CTAS + rank) * 128, n0 = at.n * TN + rank * (TN / CTAS);
      for (int k = 0; k < steps; ++k, ++n) {
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
      for (int tile = first; tile < tiles && ok; tile += stride, ++done) {
        const int buf = done & 1;
        ok = mbar_wait_warp(&ctl.acc_empty[buf], (done >> 1 & 1) ^ 1, abort_flag);
        tc_fence_after();
        for (int k = 0; k < steps && ok; ++k, ++n) {
          const int s = n % C::kStages;
          ok = mbar_wait_warp(&ctl.full[s], n / C::kStages & 1, abort_flag);
          if (!ok) break;
          tc_fence_after();
          if (leader) {
            umma_half_k4<CTAS>(tmem + buf * TN, umma_desc_sw128(base + s * C::kBytes, 1024, a_far),
                               umma_desc_sw128(base + s * C::kBytes + C::kABytes, 1024, b_far), p.idesc, k > 0, a_step, b_step);
            umma_commit(&ctl.empty[s], Ctas<CTAS>());
            if (k == steps - 1) umma_commit(&ctl.acc_full[buf], Ctas<CTAS>());
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
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;          // lanes 32 * quarter .. of tensor memory; half of the columns
    char* piece = smem + C::kOut + (warp - 2) * kLinPiece;
    const uint32_t stage = smem_u32(piece);
    // scales and biases of its columns, of this tile and the next one
    float* factors = reinterpret_cast<float*>(smem + C::kColumns) + (warp - 2) * 4 * C::kSpan;
    constexpr int per = WIDE ? 32 : 64;                            // columns of a piece
    const int from = half * C::kSpan;
    constexpr int kMine = C::kSpan / 32;
    const int r = lane >> 2, c = 2 * (lane & 3);                   // rows r, r + 8, r + 16, r + 24, of every eight columns two from c on
    const void* other = DZ ? p.dy : p.residual;
    const int other_type = DZ ? p.dy_type : p.residual_type;
    auto fetch = [&](int tile, Tile at, float* to) {
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int col = at.n * TN + from + i * 32 + lane;
        const bool in = tile < tiles && col < p.N;
        to[i * 32 + lane] = in && p.scale ? load_one(p.scale, p.scale_type, col) : 1.f;
        to[C::kSpan + i * 32 + lane] = in && p.bias ? load_one(p.bias, p.bias_type, col) : 0.f;
      }
    };
    Tile at = begin, after = begin;
    fetch(first, at, factors);
    int done = 0;
    bool ok = true;
    for (int tile = first; tile < tiles && ok; tile += stride, at = after, ++done) {
      const int buf = done & 1;
      const int64_t m0 = (static_cast<int64_t>(at.m) * CTAS + rank) * 128 + quarter * 32;
      const int n0 = at.n * TN;
      const int width = min(min(from + C::kSpan, TN), p.N - n0);   // columns from .. width
      const float* columns = factors + buf * 2 * C::kSpan;
      __syncwarp();
      advance(after);
      fetch(tile + stride, after, factors + (buf ^ 1) * 2 * C::kSpan);
      ok = mbar_wait_warp(&ctl.acc_full[buf], done >> 1 & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      // 32 columns' sums; once they are taken the next 32 are asked for, under no condition, so that their registers have no other writer to
      // wait for, and are on their way while these are stored.
      const uint32_t sums = tmem + (static_cast<uint32_t>(quarter) << 21) + buf * TN + from;
      uint32_t v[32];
      if (from < TN) tmem_ld_32x32(sums, v);
#pragma unroll
      for (int g = 0; g < kMine; ++g) {
        float2 x[4][4], o[4][4];
        if (other) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int64_t row = m0 + r + 8 * i;
              const int col = from + g * 32 + 8 * j + c, n = row < p.M && col < width ? min(2, width - col) : 0;
              o[j][i] = load_pair(other, other_type, row * p.N + n0 + col, n, p.residual_pairs);
            }
        }
        tmem_ld_wait_for(v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 s = *reinterpret_cast<const float2*>(columns + g * 32 + 8 * j + c);
          const float2 b = *reinterpret_cast<const float2*>(columns + C::kSpan + g * 32 + 8 * j + c);
          float2 db = both(0.f), ds = both(0.f);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = (i >> 1) * 16 + j * 4 + (i & 1) * 2;
            const float2 z = fadd2(make_float2(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), b);
            float2 slope;
            const float2 u = activate<DZ>(z, p.act, slope);
            if constexpr (DZ) {
              x[j][i] = fmul2(fmul2(o[j][i], s), slope);
              if (m0 + r + 8 * i < p.M) {                          // a row that is not there has dy = 0, but may have any z
                db = fadd2(db, x[j][i]);
                ds = ffma2(o[j][i], u, ds);
              }
            } else {
              x[j][i] = other ? ffma2(u, s, o[j][i]) : fmul2(u, s);
            }
          }
          if constexpr (DZ) {
            if (p.bias_sums || p.scale_sums) {
#pragma unroll
              for (int step = 4; step < 32; step *= 2) {
                db = fadd2(db, make_float2(__shfl_xor_sync(0xffffffffu, db.x, step), __shfl_xor_sync(0xffffffffu, db.y, step)));
                ds = fadd2(ds, make_float2(__shfl_xor_sync(0xffffffffu, ds.x, step), __shfl_xor_sync(0xffffffffu, ds.y, step)));
              }
              const int col = from + g * 32 + 8 * j + c;
              const int64_t to = (m0 >> 5) * p.N + n0 + col;
              if (r == 0 && m0 < p.M && col < width) {
                if (p.bias_sums) p.bias_sums[to] = db.x;
                if (p.scale_sums) p.scale_sums[to] = ds.x;
                if (col + 1 < width) {
                  if (p.bias_sums) p.bias_sums[to + 1] = db.y;
                  if (p.scale_sums) p.scale_sums[to + 1] = ds.y;
                }
              }
            }
          }
        }
        if (g + 1 < kMine) {
          if (from < TN) tmem_ld_32x32(sums + g * 32 + 32, v);
        } else {                                                   // this warp's sums are in registers
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_first_cta<CTAS>(&ctl.acc_empty[buf]);
        }
        if (from + g * 32 < width && p.out) {
          const bool last = g + 1 == kMine || from + g * 32 + 32 >= width;
          if (per == 32 || !(g & 1)) {
            if (lane == 0) bulk_wait_read();                       // the store before has left this piece
            __syncwarp();
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            // row r + 8 i: 128 bytes, its 16-byte chunks swizzled by r
            char* to = piece + r * 128 + (WIDE ? (((2 * j + (c >> 2)) ^ r) << 4) + (c & 2) * 4 : ((((g & 1) * 4 + j) ^ r) << 4) + c * 2);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (WIDE) *reinterpret_cast<float2*>(to + i * 1024) = x[j][i];
              else *reinterpret_cast<uint32_t*>(to + i * 1024) = p.out_type == S3R_BF16 ? pack_bf16(x[j][i].x, x[j][i].y) : pack_half(x[j][i].x, x[j][i].y);
            }
          }
          if (per == 32 || (g & 1) || last) {
            const int c0 = from + (per == 32 ? g * 32 : g / 2 * 64);
            if (p.copy_out) {
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                if (m0 < p.M) tma_store_2d(&mo, stage, n0 + c0, static_cast<int>(m0));
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
      __syncwarp();                                                // its factors are read
    }
    if (lane == 0) bulk_wait_all();
    if (!ok && lane == 0) atomicOr(p.status, kStatusWaitTimeout);
  }
  tc_fence_before();
  __syncthreads();
  sync_pair<CTAS>();                                               // the other CTA's products and arrivals reach this one's memory
  if (warp == 1) tmem_free<CTAS>(tmem, 2 * TN);
}

// An operand: `rows` of the result's rows or columns, `k` steps of the contraction; pitch in elements.
struct LinOperand {
  const void* data;
  int64_t pitch;
  bool turned;
};
static int operand_map(CUtensorMap* map, const LinOperand& o, int64_t rows, int64_t k, uint32_t box_rows, bool bf16) {
  const uint64_t dims[2] = {static_cast<uint64_t>(o.turned ? rows : k), static_cast<uint64_t>(o.turned ? k : rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(o.pitch) * 2};
  const uint32_t box[2] = {64, o.turned ? 64 : box_rows};
  return make_tensor_map(map, o.data, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
}

template <int TN, int CTAS, bool WIDE, bool DZ>
static int launch_linear(const LinOperand& a, const LinOperand& b, int64_t k, bool bf16, LinParams p, cudaStream_t st) {
  using C = LinCfg<TN, CTAS>;
  CUtensorMap ma, mb, mo;
  if (const int rc = operand_map(&ma, a, p.M, k, 128, bf16)) return rc;
  if (const int rc = operand_map(&mb, b, p.N, k, TN / CTAS, bf16)) return rc;
  mo = ma;
  constexpr int kSize = WIDE ? 4 : 2;
  p.copy_out = (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 && p.out_pitch * kSize % 16 == 0;
  if (p.copy_out && p.out) {
    const uint64_t dims[2] = {static_cast<uint64_t>(p.N), static_cast<uint64_t>(p.M)}, strides[1] = {static_cast<uint64_t>(p.out_pitch) * kSize};
    const uint32_t box[2] = {128 / kSize, 32};
    const CUtensorMapDataType type = WIDE ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : p.out_type == S3R_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if (const int rc = make_tensor_map(&mo, p.out, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, type)) return rc;
  }
  p.idesc = umma_idesc_half(128 * CTAS, TN, bf16, a.turned, b.turned);
  p.a_turned = a.turned;
  p.b_turned = b.turned;
  p.steps = static_cast<int>((k + kLinStep - 1) / kLinStep);
  p.m_tiles = static_cast<int>((p.M + 128 * CTAS - 1) / (128 * CTAS));
  p.n_tiles = (p.N + TN - 1) / TN;
  const int64_t tiles = static_cast<int64_t>(p.m_tiles) * p.n_tiles, at_once = sm_count() / CTAS;
  S3R_REQUIRE(tiles < (1ll << 31) - 1024, S3R_ERR_TOO_LARGE, "s3r_linear: too many tiles");
  static std::atomic<uint64_t> ready{0};
  if (attributes_missing(ready)) {
    S3R_CUDA(cudaFuncSetAttribute(linear_kernel<TN, CTAS, WIDE, DZ>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
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
  return check_cuda(cudaLaunchKernelEx(&c, linear_kernel<TN, CTAS, WIDE, DZ>, ma, mb, mo, p), "kernel launch");
}

// The tile whose waves cost least: a wave of narrower tiles takes less, but not in proportion (the same rows of a).
template <bool WIDE, bool DZ>
static int run_linear(const LinOperand& a, const LinOperand& b, int64_t k, bool bf16, const LinParams& p, cudaStream_t st) {
  auto cost = [&](int tn, int ctas) {
    const int64_t tiles = (p.M + 128 * ctas - 1) / (128 * ctas) * ((p.N + tn - 1) / tn), at_once = sm_count() / ctas;
    return (tiles + at_once - 1) / at_once * (tn + (ctas == 2 ? 64 : 96));
  };
  const int64_t pair_256 = cost(256, 2), pair_128 = cost(128, 2), one_128 = cost(128, 1), one_64 = cost(64, 1);
  if (p.M > 128 && pair_256 <= pair_128 && pair_256 <= one_128 && pair_256 <= one_64) return launch_linear<256, 2, WIDE, DZ>(a, b, k, bf16, p, st);
  if (p.M > 128 && pair_128 <= one_128 && pair_128 <= one_64) return launch_linear<128, 2, WIDE, DZ>(a, b, k, bf16, p, st);
  if (one_128 <= one_64) return launch_linear<128, 1, WIDE, DZ>(a, b, k, bf16, p, st);
  return launch_linear<64, 1, WIDE, DZ>(a, b, k, bf16, p, st);
}

// ---------------------------------------------------------------------------------------------------------------------
// a few tokens: the weights are read once, at the rate of memory, and tensor cores would wait for tiles of them.  A warp has four output
// channels, a lane 16 bytes of each at a time; the tokens lie in shared memory.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kLinFew = 8, kLinFewBytes = 48 * 1024, kLinFewChannels = 4, kLinFewWarps = 8;

struct LinFewParams {
  const uint16_t *x, *w;
  const void *bias, *scale, *residual;
  void* out;
  int64_t x_pitch, w_pitch;
  int N, K, M, type, bias_type, scale_type, residual_type, out_type, act;
};

// eight elements from k on; what lies behind the row's end is 0 and not read
__device__ __forceinline__ uint4 load_8(const uint16_t* row, int k, int K) {
  if (k + 8 <= K) return __ldg(reinterpret_cast<const uint4*>(row + k));
  uint32_t w[4] = {0, 0, 0, 0};
  for (int i = 0; k + i < K; ++i) w[i >> 1] |= static_cast<uint32_t>(row[k + i]) << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <bool BF16>
__device__ __forceinline__ float2 pair_of(uint32_t w) {
  return BF16 ? make_float2(bf16_lo(w), bf16_hi(w)) : make_float2(half_lo(w), half_hi(w));
}

template <int M, bool BF16>
__global__ void __launch_bounds__(32 * kLinFewWarps) linear_few_kernel(const __grid_constant__ LinFewParams p) {
  extern __shared__ __align__(16) char smem[];
  griddep_wait();
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, chunks = (p.K + 7) / 8;
  uint4* x = reinterpret_cast<uint4*>(smem);                       // [M][chunks]
  const int n0 = (blockIdx.x * kLinFewWarps + warp) * kLinFewChannels;
  // the first weights are on their way while the tokens are fetched
  uint4 w[kLinFewChannels];
  auto fetch = [&](int c) {
#pragma unroll
    for (int i = 0; i < kLinFewChannels; ++i) w[i] = n0 + i < p.N && c < chunks ? load_8(p.w + (n0 + i) * p.w_pitch, c * 8, p.K) : make_uint4(0, 0, 0, 0);
  };
  fetch(lane);
#pragma unroll
  for (int m = 0; m < M; ++m)
    for (int c = threadIdx.x; c < chunks; c += 32 * kLinFewWarps) x[m * chunks + c] = m < p.M ? load_8(p.x + m * p.x_pitch, c * 8, p.K) : make_uint4(0, 0, 0, 0);
  __syncthreads();
  float2 sum[kLinFewChannels][M];
#pragma unroll
  for (int i = 0; i < kLinFewChannels; ++i)
#pragma unroll
    for (int m = 0; m < M; ++m) sum[i][m] = both(0.f);
  for (int c = lane; c < chunks; c += 32) {
    float2 now[kLinFewChannels][4];
#pragma unroll
    for (int i = 0; i < kLinFewChannels; ++i) {
      now[i][0] = pair_of<BF16>(w[i].x);
      now[i][1] = pair_of<BF16>(w[i].y);
      now[i][2] = pair_of<BF16>(w[i].z);
      now[i][3] = pair_of<BF16>(w[i].w);
    }
    fetch(c + 32);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const uint4 t = x[m * chunks + c];
      const float2 v[4] = {pair_of<BF16>(t.x), pair_of<BF16>(t.y), pair_of<BF16>(t.z), pair_of<BF16>(t.w)};
#pragma unroll
      for (int i = 0; i < kLinFewChannels; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[i][m] = ffma2(now[i][k], v[k], sum[i][m]);
    }
  }
#pragma unroll
  for (int i = 0; i < kLinFewChannels; ++i)
#pragma unroll
    for (int m = 0; m < M; ++m) {
      float total = sum[i][m].x + sum[i][m].y;
#pragma unroll
      for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      if (lane == i * M + m && m < p.M && n0 + i < p.N) {
        const int n = n0 + i;
        const int64_t at = static_cast<int64_t>(m) * p.N + n;
        if (p.bias) total += load_one(p.bias, p.bias_type, n);
        float2 slope;
        float v[1] = {activate<false>(both(total), p.act, slope).x};
        const float s = p.scale ? load_one(p.scale, p.scale_type, n) : 1.f;
        v[0] = p.residual ? __fmaf_rn(v[0], s, load_one(p.residual, p.residual_type, at)) : v[0] * s;
        Raw<1> o;
        pack<1>(o, v, p.out_type);
        store_raw<1>(o, p.out, p.out_type, at);
      }
    }
}

template <int M>
static int run_linear_few(const LinFewParams& p, cudaStream_t st) {
  static_assert(M * kLinFewChannels <= 32, "a lane per result");
  const int per = kLinFewWarps * kLinFewChannels;
  const unsigned grid = static_cast<unsigned>((p.N + per - 1) / per);
  const size_t smem = static_cast<size_t>(M) * ((p.K + 7) / 8) * 16;
  return p.type == S3R_BF16 ? launch(linear_few_kernel<M, true>, grid, 32 * kLinFewWarps, smem, st, p)
                            : launch(linear_few_kernel<M, false>, grid, 32 * kLinFewWarps, smem, st, p);
}

// ---------------------------------------------------------------------------------------------------------------------
// dz = dy * scale where no z is needed, with its sums over rows.  Bound: HBM.  A CTA has 64 rows and 256 columns, a thread eight columns of
// every eighth row.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kDzRows = 64, kDzColumns = 256;

struct DzParams {
  const void *dy, *scale;
  void* dz;
  float* sums;                    // [blocks of 64 rows, N], or NULL
  int64_t M, dz_pitch;
  int N, dy_type, scale_type, type;
};

template <int W>
__global__ void __launch_bounds__(256) linear_dz_kernel(const __grid_constant__ DzParams p) {
  constexpr int N = 8 / W;
  __shared__ float red[8][kDzColumns];
  griddep_wait();
  griddep_launch();
  const int t = threadIdx.x & 31, part = threadIdx.x >> 5, c0 = blockIdx.y * kDzColumns + t * 8;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kDzRows;
  float s[8], sum[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    s[k] = p.scale && c0 + k < p.N ? load_one(p.scale, p.scale_type, c0 + k) : 1.f;
    sum[k] = 0.f;
  }
  for (int i = part; i < kDzRows && r0 + i < p.M; i += 8) {
    const int64_t row = r0 + i;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int col = c0 + j * W;
      if (col >= p.N) break;
      float f[W];
      load_vector<W>(f, p.dy, p.dy_type, row * p.N + col);
#pragma unroll
      for (int k = 0; k < W; ++k) {
        f[k] *= s[j * W + k];
        sum[j * W + k] += f[k];
      }
      if (p.dz) {
        Raw<W> o;
        pack<W>(o, f, p.type);
        store_raw<W>(o, p.dz, p.type, row * p.dz_pitch + col);
      }
    }
  }
  if (!p.sums) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) red[part][t * 8 + k] = sum[k];
  __syncthreads();
  const int col = blockIdx.y * kDzColumns + threadIdx.x;
  float total = red[0][threadIdx.x];
#pragma unroll
  for (int i = 1; i < 8; ++i) total += red[i][threadIdx.x];
  if (col < p.N) p.sums[blockIdx.x * static_cast<int64_t>(p.N) + col] = total;
}

// Sums of blocks of rows, in a fixed order: a CTA has 32 columns, a warp every 32nd block.
struct SumParams {
  const float* sums[2];
  void* out[2];
  int types[2];
  int64_t blocks;
  int N;
};
__global__ void __launch_bounds__(1024) linear_sums_kernel(const __grid_constant__ SumParams p) {
  __shared__ float red[32][33];
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  const float* sums = blockIdx.y ? p.sums[1] : p.sums[0];
  void* out = blockIdx.y ? p.out[1] : p.out[0];
  const int type = blockIdx.y ? p.types[1] : p.types[0];
  float total = 0.f;
  if (col < p.N)
    for (int64_t i = warp; i < p.blocks; i += 32) total += __ldg(sums + i * p.N + col);
  red[warp][lane] = total;
  __syncthreads();
  if (warp == 0) {
    total = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) total += red[i][lane];
    if (col < p.N) {
      const float v[1] = {total};
      Raw<1> o;
      pack<1>(o, v, type);
      store_raw<1>(o, out, type, col);
    }
  }
}

static int run_sums(const SumParams& p, int n, cudaStream_t st) {
  return launch(linear_sums_kernel, dim3(static_cast<unsigned>((p.N + 31) / 32), static_cast<unsigned>(n)), 1024, 0, st, p);
}

static bool half_type(int type) { return type == S3R_BF16 || type == S3R_F16; }
static bool at_multiple(const void* p, int type) { return reinterpret_cast<uintptr_t>(p) % type_bytes(type) == 0; }
static bool copied_by_tma(const void* p, int64_t pitch) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && pitch % 8 == 0; }

static int check_linear(const s3r_linear* f, const char* what) {
  S3R_REQUIRE(f && f->x && f->weight, S3R_ERR_NULL, "%s: NULL pointer", what);
  S3R_REQUIRE(f->M > 0 && f->N > 0 && f->K > 0 && f->x_pitch >= f->K && f->w_pitch >= f->K, S3R_ERR_SHAPE, "%s: sizes must be positive, pitches no shorter than rows", what);
  S3R_REQUIRE(half_type(f->type), S3R_ERR_UNSUPPORTED, "%s: operands are bf16 or fp16", what);
  S3R_REQUIRE(known_type(f->out_type) && (!f->bias || known_type(f->bias_type)) && (!f->scale || known_type(f->scale_type)) &&
                  (!f->residual || known_type(f->residual_type)), S3R_ERR_UNSUPPORTED, "%s: types are fp32, bf16 and fp16", what);
  S3R_REQUIRE(f->act >= S3R_ACT_NONE && f->act <= S3R_ACT_SILU, S3R_ERR_UNSUPPORTED, "%s: activation %d", what, f->act);
  S3R_REQUIRE(f->M < (1ll << 31) - 512 && f->N < INT_MAX - 512 && f->K < INT_MAX - 512, S3R_ERR_TOO_LARGE, "%s: too many rows or columns", what);
  S3R_REQUIRE(copied_by_tma(f->x, f->x_pitch) && copied_by_tma(f->weight, f->w_pitch), S3R_ERR_ALIGNMENT, "%s: operands and their rows must begin at multiples of 16 bytes", what);
  S3R_REQUIRE((!f->bias || at_multiple(f->bias, f->bias_type)) && (!f->scale || at_multiple(f->scale, f->scale_type)) &&
                  (!f->residual || at_multiple(f->residual, f->residual_type)), S3R_ERR_ALIGNMENT, "%s: elements must be aligned", what);
  return 0;
}
static bool in_pairs(const void* p, int type, int N) { return N % 2 == 0 && reinterpret_cast<uintptr_t>(p) % (2 * type_bytes(type)) == 0; }

static LinParams linear_params(const s3r_linear* f) {
  LinParams p = {};
  p.M = f->M;
  p.N = f->N;
  p.bias = f->bias;
  p.scale = f->scale;
  p.bias_type = f->bias_type;
  p.scale_type = f->scale_type;
  p.act = f->act;
  p.status = device_status_ptr();
  return p;
}

}  // namespace s3r

using namespace s3r;

extern "C" int s3r_linear_fwd(const s3r_linear* f, void* stream) {
  if (const int rc = check_linear(f, "s3r_linear_fwd")) return rc;
  S3R_REQUIRE(f->out, S3R_ERR_NULL, "s3r_linear_fwd: NULL pointer");
  S3R_REQUIRE(at_multiple(f->out, f->out_type), S3R_ERR_ALIGNMENT, "s3r_linear_fwd: elements must be aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (f->M <= kLinFew && (f->M <= 2 ? f->M : f->M <= 4 ? 4 : 8) * ((static_cast<int64_t>(f->K) + 7) / 8 * 16) <= kLinFewBytes) {
    const LinFewParams p = {static_cast<const uint16_t*>(f->x), static_cast<const uint16_t*>(f->weight), f->bias, f->scale, f->residual, f->out, f->x_pitch, f->w_pitch,
                            f->N, f->K, static_cast<int>(f->M), f->type, f->bias_type, f->scale_type, f->residual_type, f->out_type, f->act};
    return f->M == 1 ? run_linear_few<1>(p, st) : f->M == 2 ? run_linear_few<2>(p, st) : f->M <= 4 ? run_linear_few<4>(p, st) : run_linear_few<8>(p, st);
  }
  LinParams p = linear_params(f);
  S3R_REQUIRE(p.status, S3R_ERR_DRIVER, "s3r_linear_fwd: no status word");
  p.residual = f->residual;
  p.residual_type = f->residual_type;
  p.residual_pairs = f->residual && in_pairs(f->residual, f->residual_type, f->N);
  p.out = f->out;
  p.out_pitch = f->N;
  p.out_type = f->out_type;
  const LinOperand a = {f->x, f->x_pitch, false}, b = {f->weight, f->w_pitch, false};
  const bool bf16 = f->type == S3R_BF16;
  return f->out_type == S3R_F32 ? run_linear<true, false>(a, b, f->K, bf16, p, st) : run_linear<false, false>(a, b, f->K, bf16, p, st);
}

static int64_t sum_blocks(int64_t M) { return (M + 31) / 32; }

extern "C" size_t s3r_linear_bwd_workspace_bytes(int64_t M, int N) {
  return M > 0 && N > 0 ? static_cast<size_t>(sum_blocks(M)) * N * sizeof(float) : 0;
}

extern "C" int s3r_linear_bwd(const s3r_linear* f, const s3r_linear_grad* g, void* stream) {
  if (const int rc = check_linear(f, "s3r_linear_bwd")) return rc;
  S3R_REQUIRE(g && g->dy, S3R_ERR_NULL, "s3r_linear_bwd: NULL pointer");
  S3R_REQUIRE(!g->dz || (g->dz_pitch >= f->N && copied_by_tma(g->dz, g->dz_pitch)), S3R_ERR_ALIGNMENT, "s3r_linear_bwd: rows of dz must begin at multiples of 16 bytes");
  S3R_REQUIRE(at_multiple(g->dy, f->out_type), S3R_ERR_ALIGNMENT, "s3r_linear_bwd: elements must be aligned");
  S3R_REQUIRE((!g->d_bias || f->bias) && (!g->d_scale || f->scale), S3R_ERR_NULL, "s3r_linear_bwd: a gradient of what is not there");
  const int sums = (g->d_bias != nullptr) + (g->d_scale != nullptr);
  const size_t each = s3r_linear_bwd_workspace_bytes(f->M, f->N);
  S3R_REQUIRE(!sums || (g->workspace && g->workspace_bytes >= each * sums && (reinterpret_cast<uintptr_t>(g->workspace) & 3) == 0), S3R_ERR_TOO_LARGE,
              "s3r_linear_bwd: workspace too small");
  if (!g->dz && !sums) return 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  float* bias_sums = g->d_bias ? static_cast<float*>(g->workspace) : nullptr;
  float* scale_sums = g->d_scale ? static_cast<float*>(g->workspace) + (g->d_bias ? each / 4 : 0) : nullptr;
  SumParams s = {};
  s.N = f->N;
  int rc;
  if (f->act == S3R_ACT_NONE && !g->d_scale) {
    const DzParams d = {g->dy, f->scale, g->dz, bias_sums, f->M, g->dz_pitch, f->N, f->out_type, f->scale_type, f->type};
    const int64_t blocks = (f->M + kDzRows - 1) / kDzRows;
    S3R_REQUIRE(f->N <= 65535 * kDzColumns, S3R_ERR_TOO_LARGE, "s3r_linear_bwd: %d columns", f->N);
    const void* ptr[] = {g->dy, g->dz};
    const int types[] = {f->out_type, f->type};
    const int w = row_vector(f->N, ptr, types, 2);
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((f->N + kDzColumns - 1) / kDzColumns));
    rc = w == 8 ? launch(linear_dz_kernel<8>, grid, 256, 0, st, d) : w == 4 ? launch(linear_dz_kernel<4>, grid, 256, 0, st, d) : launch(linear_dz_kernel<1>, grid, 256, 0, st, d);
    s.blocks = blocks;
  } else {
    LinParams p = linear_params(f);
    S3R_REQUIRE(p.status, S3R_ERR_DRIVER, "s3r_linear_bwd: no status word");
    p.dy = g->dy;
    p.dy_type = f->out_type;
    p.residual_pairs = in_pairs(g->dy, f->out_type, f->N);
    p.out = g->dz;
    p.out_pitch = g->dz ? g->dz_pitch : 8;
    p.out_type = f->type;
    p.bias_sums = bias_sums;
    p.scale_sums = scale_sums;
    rc = run_linear<false, true>({f->x, f->x_pitch, false}, {f->weight, f->w_pitch, false}, f->K, f->type == S3R_BF16, p, st);
    s.blocks = sum_blocks(f->M);
  }
  if (rc || !sums) return rc;
  int n = 0;
  if (g->d_bias) s.sums[n] = bias_sums, s.out[n] = g->d_bias, s.types[n] = f->bias_type, ++n;
  if (g->d_scale) s.sums[n] = scale_sums, s.out[n] = g->d_scale, s.types[n] = f->scale_type, ++n;
  return run_sums(s, n, st);
}

extern "C" int s3r_product(const void* a, int64_t a_pitch, int a_turned, const void* b, int64_t b_pitch, int b_turned, int type, void* out, int64_t M, int N,
                           int64_t K, void* stream) {
  S3R_REQUIRE(a && b && out, S3R_ERR_NULL, "s3r_product: NULL pointer");
  S3R_REQUIRE(M > 0 && N > 0 && K > 0 && a_pitch >= (a_turned ? M : K) && b_pitch >= (b_turned ? N : K), S3R_ERR_SHAPE,
              "s3r_product: sizes must be positive, pitches no shorter than rows");
  S3R_REQUIRE(half_type(type), S3R_ERR_UNSUPPORTED, "s3r_product: operands are bf16 or fp16");
  S3R_REQUIRE(M < (1ll << 31) - 512 && N < INT_MAX - 512 && K < (1ll << 31) - 512, S3R_ERR_TOO_LARGE, "s3r_product: too many rows or columns");
  S3R_REQUIRE(copied_by_tma(a, a_pitch) && copied_by_tma(b, b_pitch), S3R_ERR_ALIGNMENT, "s3r_product: operands and their rows must begin at multiples of 16 bytes");
  S3R_REQUIRE(at_multiple(out, type), S3R_ERR_ALIGNMENT, "s3r_product: elements must be aligned");
  LinParams p = {};
  p.M = M;
  p.N = N;
  p.out = out;
  p.out_pitch = N;
  p.out_type = type;
  p.status = device_status_ptr();
  S3R_REQUIRE(p.status, S3R_ERR_DRIVER, "s3r_product: no status word");
  return run_linear<false, false>({a, a_pitch, a_turned != 0}, {b, b_pitch, b_turned != 0}, K, type == S3R_BF16, p, static_cast<cudaStream_t>(stream));
}
