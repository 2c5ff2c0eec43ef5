// Products of 8-bit integers with a scale per token and per output channel, and the tokens they are made of.
//   quantise  scale[r] = max |x[r]| / 127, q = x / scale to nearest even.  Bound: HBM, a row is read once and kept in registers.
//   product   out[m, n] = (sum_k a[m, k] b[n, k]) a_scale[m] b_scale[n] + bias[n].  The sums are exact (32-bit integers), so that
//             no order of the k-steps changes a result.
#include "rows.cuh"

namespace s3r {

// ---------------------------------------------------------------------------------------------------------------------
// rows to 8 bits: G threads per row, E elements per thread in registers (E = 0: rows of any length, read twice)
// ---------------------------------------------------------------------------------------------------------------------
struct QuantParams {
  const void* x;
  int8_t* q;
  float* scale;
  int64_t x_pitch, q_pitch, rows;
  int type, channels;
};

template <int W>
__device__ __forceinline__ void store_s8(int8_t* q, const float (&f)[W], float inverse) {
  if constexpr (W == 1) {
    *q = static_cast<int8_t>(to_s8(f[0], inverse));
  } else {
    uint32_t w[W / 4];
#pragma unroll
    for (int k = 0; k < W; k += 4)
      w[k / 4] = to_s8(f[k], inverse) | to_s8(f[k + 1], inverse) << 8 | to_s8(f[k + 2], inverse) << 16 | to_s8(f[k + 3], inverse) << 24;
    if constexpr (W == 8) *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(q) = w[0];
  }
}

template <int W, int G, int E>
__global__ void __launch_bounds__(G < 128 ? 128 : G) quantize_kernel(const __grid_constant__ QuantParams p) {
  constexpr int kRows = G < 128 ? 128 / G : 1, N = E / W;
  __shared__ float red[G > 32 ? 8 * (G / 32) : 1];
  griddep_wait();
  griddep_launch();
  const int t = threadIdx.x % G, C = p.channels;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / G;
  if (row >= p.rows) return;
  const int64_t at = row * p.x_pitch;
  int8_t* q = p.q + row * p.q_pitch;
  uint32_t turn = 0;
  float big = 0.f;
  if constexpr (E > 0) {
    Raw<W> r[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((i * G + t) * W < C) load_raw<W>(r[i], p.x, p.type, at + (i * G + t) * W);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((i * G + t) * W < C) {
        float f[W];
        unpack<W>(f, r[i], p.type);
#pragma unroll
        for (int k = 0; k < W; ++k) big = max_nan(big, fabsf(f[k]));
      }
    big = row_max<G>(big, red, turn, t, 0);
    const RowScale s = row_scale(big);
    if (t == 0) p.scale[row] = s.scale;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((i * G + t) * W < C) {
        float f[W];
        unpack<W>(f, r[i], p.type);
        store_s8<W>(q + (i * G + t) * W, f, s.inverse);
      }
  } else {
    for (int c = t * W; c < C; c += G * W) {
      float f[W];
      load_vector<W>(f, p.x, p.type, at + c);
#pragma unroll
      for (int k = 0; k < W; ++k) big = max_nan(big, fabsf(f[k]));
    }
    big = row_max<G>(big, red, turn, t, 0);
    const RowScale s = row_scale(big);
    if (t == 0) p.scale[row] = s.scale;
    for (int c = t * W; c < C; c += G * W) {
      float f[W];
      load_vector<W>(f, p.x, p.type, at + c);
      store_s8<W>(q + c, f, s.inverse);
    }
  }
}

template <int W, int G, int E>
static int run_quantize(const QuantParams& p, cudaStream_t st) {
  constexpr int kRows = G < 128 ? 128 / G : 1;
  const int64_t grid = (p.rows + kRows - 1) / kRows;
  return launch(quantize_kernel<W, G, E>, static_cast<unsigned>(grid), G < 128 ? 128 : G, 0, st, p);
}
template <int W>
static int pick_quantize(const QuantParams& p, cudaStream_t st) {
  const int C = p.channels;
  if (C <= 256) return run_quantize<W, 32, 8>(p, st);
  if (C <= 1024 && p.rows <= 2 * sm_count()) return run_quantize<W, 128, 8>(p, st);
  if (C <= 1024) return run_quantize<W, 32, 32>(p, st);
  if (C <= 4096) return run_quantize<W, 128, 32>(p, st);
  if (C <= 16384) return run_quantize<W, 512, 32>(p, st);
  return run_quantize<W, 1024, 0>(p, st);
}

// ---------------------------------------------------------------------------------------------------------------------
// product on tcgen05: persistent CTAs; 128 x TN tiles, K in steps of 128 bytes through a ring of TMA copies, the sums of two
// tiles in tensor memory so that one is written out while the next is summed.  One warp copies, one issues the products, four
// take the sums, scale them and store through shared memory.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kI8Threads = 192, kI8Stage = 4096;       // a warp's piece of the output: 32 rows of 128 bytes

struct I8Params {
  const float *a_scale, *b_scale, *bias;
  void* out;
  int64_t M;
  int N, K, type;
  int m_tiles, n_tiles;
  uint32_t copy_out;             // rows of the output are a multiple of 16 bytes: TMA stores
  uint32_t* status;
};

template <int TN>
struct I8Cfg {
  static constexpr int kStages = TN == 256 ? 4 : 6;
  static constexpr int kABytes = 128 * 128, kBBytes = TN * 128, kBytes = kABytes + kBBytes;
  static constexpr int kOut = kStages * kBytes, kColumns = kOut + 4 * 2 * kI8Stage;
  static constexpr int kSmem = kColumns + 4 * 32 * 8 + 1024;
};

struct I8Ctl {
  uint64_t full[6], empty[6], acc_full[2], acc_empty[2], drained;
  uint32_t tmem_base, abort_flag;
};

// kind::i8, signed x signed -> int32
__host__ __device__ constexpr uint32_t umma_idesc_i8(uint32_t M, uint32_t N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | ((M >> 4) << 24);
}
// Four k-steps of 32 bytes.
__device__ __forceinline__ void umma_i8_k4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p, pt;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.u32 pt, 0, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
      "add.s64 a, %1, 2;\n\tadd.s64 b, %2, 2;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], a, b, %3, pt;\n\t"
      "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], a, b, %3, pt;\n\t"
      "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], a, b, %3, pt;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accum)
      : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst_smem, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst_smem), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src_smem, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];"
               ::"l"(map), "r"(src_smem), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

template <int TN>
__global__ void __launch_bounds__(kI8Threads) int8_linear_kernel(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb,
                                                                 const __grid_constant__ CUtensorMap mo, const __grid_constant__ I8Params p) {
  using C = I8Cfg<TN>;
  extern __shared__ char raw_smem[];
  __shared__ I8Ctl ctl;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&ctl.full[s], 1);
      mbar_init(&ctl.empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&ctl.acc_full[s], 1);
      mbar_init(&ctl.acc_empty[s], 4);
    }
    mbar_init(&ctl.drained, 1);
    ctl.abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(&ctl.tmem_base, 2 * TN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_wait();
  griddep_launch();
  const uint32_t tmem = ctl.tmem_base;
  volatile uint32_t* abort_flag = &ctl.abort_flag;
  const int tiles = p.m_tiles * p.n_tiles, steps = (p.K + 127) / 128;
  const uint32_t base = smem_u32(smem);

  if (warp == 0) {
    int n = 0;                                                     // copies so far
    bool ok = true;
    const bool leader = elect_one_sync();
    for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
      const int m0 = tile / p.n_tiles * 128, n0 = tile % p.n_tiles * TN;
      for (int k = 0; k < steps; ++k, ++n) {
        const int s = n % C::kStages;
        ok = mbar_wait_warp(&ctl.empty[s], (n / C::kStages & 1) ^ 1, abort_flag);
        if (!ok) break;
        if (leader) {
          mbar_expect_tx(&ctl.full[s], C::kBytes);
          tma_load_2d(base + s * C::kBytes, &ma, &ctl.full[s], k * 128, m0);
          tma_load_2d(base + s * C::kBytes + C::kABytes, &mb, &ctl.full[s], k * 128, n0);
        }
        __syncwarp();
      }
    }
    if (!ok) {                                                     // copies in flight land before the CTA's memory is given away
      for (int i = n - C::kStages < 0 ? 0 : n - C::kStages; i < n; ++i) {
        volatile uint32_t dummy = 0;
        mbar_wait(&ctl.full[i % C::kStages], i / C::kStages & 1, &dummy);
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = umma_idesc_i8(128, TN);
    const bool leader = elect_one_sync();
    int n = 0, done = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++done) {
      const int buf = done & 1;
      ok = mbar_wait_warp(&ctl.acc_empty[buf], (done >> 1 & 1) ^ 1, abort_flag);
      tc_fence_after();
      for (int k = 0; k < steps && ok; ++k, ++n) {
        const int s = n % C::kStages;
        ok = mbar_wait_warp(&ctl.full[s], n / C::kStages & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          umma_i8_k4(tmem + buf * TN, umma_desc_sw128(base + s * C::kBytes), umma_desc_sw128(base + s * C::kBytes + C::kABytes), idesc, k > 0);
          umma_commit(&ctl.empty[s]);
          if (k == steps - 1) umma_commit(&ctl.acc_full[buf]);
        }
        __syncwarp();
      }
    }
    if (!ok) {
      if (leader) umma_commit(&ctl.drained);
      __syncwarp();
      volatile uint32_t dummy = 0;
      mbar_wait(&ctl.drained, 0, &dummy);                          // let issued products drain before tensor memory is freed
    }
  } else {
    const int quarter = warp & 3;                                  // lanes 32 * quarter .. of tensor memory
    const uint32_t stage0 = base + C::kOut + quarter * 2 * kI8Stage;
    float2* columns = reinterpret_cast<float2*>(smem + C::kColumns) + quarter * 32;
    const int per = p.type == S3R_F32 ? 32 : 64;                   // columns of a piece
    int done = 0, piece = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++done) {
      const int buf = done & 1;
      const int64_t m0 = static_cast<int64_t>(tile / p.n_tiles) * 128 + quarter * 32;
      const int n0 = tile % p.n_tiles * TN;
      const float row_scale = m0 + lane < p.M ? __ldg(p.a_scale + m0 + lane) : 0.f;
      ok = mbar_wait_warp(&ctl.acc_full[buf], done >> 1 & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const int width = min(TN, p.N - n0);
      for (int c0 = 0; c0 < width; c0 += per, ++piece) {
        const uint32_t stage = stage0 + (piece & 1) * kI8Stage;
        if (lane == 0) bulk_wait_read<1>();                        // the store before the last has left this half
        __syncwarp();
        for (int half = 0; half < per; half += 32) {
          uint32_t v[32];
          tmem_ld32(tmem + (static_cast<uint32_t>(quarter) << 21) + buf * TN + c0 + half, v);
          const int col = n0 + c0 + half + lane;
          const bool in = col < p.N;
          columns[lane] = make_float2(in ? __ldg(p.b_scale + col) : 0.f, in && p.bias ? __ldg(p.bias + col) : 0.f);
          __syncwarp();
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float4 f = *reinterpret_cast<const float4*>(columns + i);
            const float x = __fmul_rn(__fmul_rn(__int2float_rn(static_cast<int>(v[i])), row_scale), f.x);
            const float y = __fmul_rn(__fmul_rn(__int2float_rn(static_cast<int>(v[i + 1])), row_scale), f.z);
            v[i] = __float_as_uint(p.bias ? __fadd_rn(x, f.y) : x);
            v[i + 1] = __float_as_uint(p.bias ? __fadd_rn(y, f.w) : y);
          }
          auto f = [&](int i) { return __uint_as_float(v[i]); };
          if (p.type == S3R_F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sts128(stage + swz128(lane, i), v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
          } else if (p.type == S3R_BF16) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              sts128(stage + swz128(lane, half / 8 + i), pack_bf16(f(8 * i), f(8 * i + 1)), pack_bf16(f(8 * i + 2), f(8 * i + 3)),
                     pack_bf16(f(8 * i + 4), f(8 * i + 5)), pack_bf16(f(8 * i + 6), f(8 * i + 7)));
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              sts128(stage + swz128(lane, half / 8 + i), pack_half(f(8 * i), f(8 * i + 1)), pack_half(f(8 * i + 2), f(8 * i + 3)),
                     pack_half(f(8 * i + 4), f(8 * i + 5)), pack_half(f(8 * i + 6), f(8 * i + 7)));
          }
          __syncwarp();                                            // all lanes have read the columns' factors
        }
        if (c0 + per >= width) {                                   // the tile's sums are in registers or stored
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctl.acc_empty[buf]);
        }
        if (p.copy_out) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (m0 < p.M) tma_store_2d(&mo, stage, n0 + c0, static_cast<int>(m0));
            bulk_commit();
          }
        } else {
          __syncwarp();
          const int left = min(per, width - c0);
          for (int r = 0; r < 32 && m0 + r < p.M; ++r) {
            const int64_t at = (m0 + r) * p.N + n0 + c0;
            for (int c = lane; c < left; c += 32) {
              const int byte = c * type_bytes(p.type);
              const char* from = smem + (stage - base) + swz128(r, byte >> 4) + (byte & 15);
              if (p.type == S3R_F32) static_cast<float*>(p.out)[at + c] = *reinterpret_cast<const float*>(from);
              else static_cast<uint16_t*>(p.out)[at + c] = *reinterpret_cast<const uint16_t*>(from);
            }
          }
        }
      }
    }
    if (lane == 0) bulk_wait_all();
    if (!ok && lane == 0) atomicOr(p.status, kStatusWaitTimeout);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 2 * TN);
}

template <int TN>
static int run_int8(const int8_t* a, int64_t a_pitch, const int8_t* b, int64_t b_pitch, I8Params p, cudaStream_t st) {
  using C = I8Cfg<TN>;
  CUtensorMap ma, mb, mo;
  {
    const uint64_t dims[2] = {static_cast<uint64_t>(p.K), static_cast<uint64_t>(p.M)}, strides[1] = {static_cast<uint64_t>(a_pitch)};
    const uint32_t box[2] = {128, 128};
    if (const int rc = make_tensor_map(&ma, a, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_DATA_TYPE_UINT8)) return rc;
  }
  {
    const uint64_t dims[2] = {static_cast<uint64_t>(p.K), static_cast<uint64_t>(p.N)}, strides[1] = {static_cast<uint64_t>(b_pitch)};
    const uint32_t box[2] = {128, TN};
    if (const int rc = make_tensor_map(&mb, b, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_DATA_TYPE_UINT8)) return rc;
  }
  mo = ma;
  if (p.copy_out) {
    const uint64_t dims[2] = {static_cast<uint64_t>(p.N), static_cast<uint64_t>(p.M)};
    const uint64_t strides[1] = {static_cast<uint64_t>(p.N) * type_bytes(p.type)};
    const uint32_t box[2] = {static_cast<uint32_t>(128 / type_bytes(p.type)), 32};
    const CUtensorMapDataType type = p.type == S3R_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : p.type == S3R_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if (const int rc = make_tensor_map(&mo, p.out, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, type)) return rc;
  }
  p.n_tiles = (p.N + TN - 1) / TN;
  const int64_t tiles = static_cast<int64_t>(p.m_tiles) * p.n_tiles;
  S3R_REQUIRE(tiles < (1ll << 31) - 1024, S3R_ERR_TOO_LARGE, "s3r_int8_linear: too many tiles");
  S3R_CUDA(cudaFuncSetAttribute(int8_linear_kernel<TN>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
  const unsigned grid = static_cast<unsigned>(tiles < sm_count() ? tiles : sm_count());
  return launch(int8_linear_kernel<TN>, grid, kI8Threads, C::kSmem, st, ma, mb, mo, p);
}

}  // namespace s3r

using namespace s3r;

extern "C" int s3r_quantize_rows(const void* x, int type, int64_t x_pitch, int8_t* q, int64_t q_pitch, float* scale, int64_t rows, int channels,
                                 void* stream) {
  S3R_REQUIRE(x && q && scale, S3R_ERR_NULL, "s3r_quantize_rows: NULL pointer");
  S3R_REQUIRE(rows > 0 && channels > 0 && x_pitch >= channels && q_pitch >= channels, S3R_ERR_SHAPE, "s3r_quantize_rows: sizes must be positive, pitches no shorter than rows");
  S3R_REQUIRE(known_type(type), S3R_ERR_UNSUPPORTED, "s3r_quantize_rows: types are fp32, bf16 and fp16");
  S3R_REQUIRE(rows < (1ll << 31), S3R_ERR_TOO_LARGE, "s3r_quantize_rows: too many rows");
  S3R_REQUIRE(reinterpret_cast<uintptr_t>(x) % type_bytes(type) == 0 && reinterpret_cast<uintptr_t>(scale) % 4 == 0, S3R_ERR_ALIGNMENT, "s3r_quantize_rows: elements must be aligned");
  const void* ptr[] = {x};
  int w = row_vector(channels, ptr, &type, 1);
  while (w > 1 && (x_pitch % w || (reinterpret_cast<uintptr_t>(q) | static_cast<uintptr_t>(q_pitch)) % w)) w = w == 8 ? 4 : 1;
  const QuantParams p = {x, q, scale, x_pitch, q_pitch, rows, type, channels};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return w == 8 ? pick_quantize<8>(p, st) : w == 4 ? pick_quantize<4>(p, st) : pick_quantize<1>(p, st);
}

extern "C" int s3r_int8_linear(const int8_t* a, int64_t a_pitch, const float* a_scale, const int8_t* b, int64_t b_pitch, const float* b_scale,
                               const float* bias, void* out, int type, int64_t M, int N, int K, void* stream) {
  S3R_REQUIRE(a && a_scale && b && b_scale && out, S3R_ERR_NULL, "s3r_int8_linear: NULL pointer");
  S3R_REQUIRE(M > 0 && N > 0 && K > 0 && a_pitch >= K && b_pitch >= K, S3R_ERR_SHAPE, "s3r_int8_linear: sizes must be positive, pitches no shorter than rows");
  S3R_REQUIRE(known_type(type), S3R_ERR_UNSUPPORTED, "s3r_int8_linear: types are fp32, bf16 and fp16");
  S3R_REQUIRE(K <= 65536, S3R_ERR_TOO_LARGE, "s3r_int8_linear: K = %d (at most 65536)", K);
  S3R_REQUIRE(M < (1ll << 31) - 256 && N < 0x7fffff00, S3R_ERR_TOO_LARGE, "s3r_int8_linear: too many rows");
  S3R_REQUIRE(((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0 && a_pitch % 16 == 0 && b_pitch % 16 == 0, S3R_ERR_ALIGNMENT,
              "s3r_int8_linear: operands and their pitches must be multiples of 16 bytes");
  S3R_REQUIRE(((reinterpret_cast<uintptr_t>(a_scale) | reinterpret_cast<uintptr_t>(b_scale) | reinterpret_cast<uintptr_t>(bias)) & 3) == 0 &&
                  reinterpret_cast<uintptr_t>(out) % type_bytes(type) == 0, S3R_ERR_ALIGNMENT, "s3r_int8_linear: elements must be aligned");
  I8Params p = {};
  p.a_scale = a_scale;
  p.b_scale = b_scale;
  p.bias = bias;
  p.out = out;
  p.M = M;
  p.N = N;
  p.K = K;
  p.type = type;
  p.m_tiles = static_cast<int>((M + 127) / 128);
  p.copy_out = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && static_cast<int64_t>(N) * type_bytes(type) % 16 == 0;
  p.status = device_status_ptr();
  S3R_REQUIRE(p.status, S3R_ERR_DRIVER, "s3r_int8_linear: no status word");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // the tile width whose waves cost least: a wave of narrower tiles takes less, but not in proportion (the same rows of a)
  auto cost = [&](int tn) {
    const int64_t tiles = static_cast<int64_t>(p.m_tiles) * ((N + tn - 1) / tn);
    return (tiles + sm_count() - 1) / sm_count() * (tn + 64);
  };
  if (cost(256) <= cost(128) && cost(256) <= cost(64)) return run_int8<256>(a, a_pitch, b, b_pitch, p, st);
  if (cost(128) <= cost(64)) return run_int8<128>(a, a_pitch, b, b_pitch, p, st);
  return run_int8<64>(a, a_pitch, b, b_pitch, p, st);
}
