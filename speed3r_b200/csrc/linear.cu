// Matrix products of bf16 or fp16 with what follows them in their epilogue, forward and backward.
//   forward   z = x W^T + bias,  u = act(z),  out = residual + u * scale: one rounding, to the result's type
//   backward  du = dy * scale,  dz = du * act'(z),  d_bias = sum of dz over rows,  d_scale = sum of dy * u over rows;  dx = dz W,  dW = dz^T x
// z is not kept: where it is needed (an activation's slope, the scale's gradient) the backward makes it again, and dz is the epilogue of that product.
// The forward then writes nothing but its result, and both sums over rows see z as it was, not rounded to 16 bits.
#include "linear.cuh"

namespace s3r {

// ---------------------------------------------------------------------------------------------------------------------
// a few tokens: the weights are read once, at the rate of memory, and tensor cores would wait for tiles of them.  A warp has two output channels
// (one where that still leaves an SM no more than a CTA), a lane 16 bytes at a time and eight of those in flight; the tokens lie in shared memory.
// Bound: the start of the kernel and its trips to memory, one for each 4 KB of a channel's weights.  One token x 4096 x 1024, one call behind the other in
// a graph, weights in HBM: 4.3 us, of which 1.3 are the weights' bytes; eight tokens x 1024 x 1024 6.0.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kLinFew = 8, kLinFewBytes = 48 * 1024, kLinFewWarps = 8;

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

// An element that is asked for long before it is used: a register for either width, so that nothing waits for the load in front of its use.
struct Early {
  uint32_t wide, narrow;
  Early() = default;
  __device__ __forceinline__ Early(const void* p, int type, int64_t i, bool in) {
    wide = p && in && type == S3R_F32 ? __ldg(static_cast<const uint32_t*>(p) + i) : 0;
    narrow = p && in && type != S3R_F32 ? __ldg(static_cast<const uint16_t*>(p) + i) : 0;
  }
  __device__ __forceinline__ float value(int type) const { return type == S3R_F32 ? __uint_as_float(wide) : type == S3R_BF16 ? bf16_lo(narrow) : half_lo(narrow); }
};

template <int M, bool BF16, int CHANNELS>
__global__ void __launch_bounds__(32 * kLinFewWarps) linear_few_kernel(const __grid_constant__ LinFewParams p) {
  constexpr int kAhead = 8 / CHANNELS;
  extern __shared__ __align__(16) char smem[];
  griddep_wait();
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, chunks = (p.K + 7) / 8;
  uint4* x = reinterpret_cast<uint4*>(smem);                       // [M][chunks]
  const int n0 = (blockIdx.x * kLinFewWarps + warp) * CHANNELS;
  // the first weights are on their way while the tokens are fetched
  uint4 w[kAhead][CHANNELS];
  auto fetch = [&](int c, int at) {
#pragma unroll
    for (int i = 0; i < CHANNELS; ++i) w[at][i] = n0 + i < p.N && c < chunks ? load_8(p.w + (n0 + i) * p.w_pitch, c * 8, p.K) : make_uint4(0, 0, 0, 0);
  };
#pragma unroll
  for (int k = 0; k < kAhead; ++k) fetch(lane + 32 * k, k);
#pragma unroll
  for (int m = 0; m < M; ++m)
    for (int c = threadIdx.x; c < chunks; c += 32 * kLinFewWarps) x[m * chunks + c] = m < p.M ? load_8(p.x + m * p.x_pitch, c * 8, p.K) : make_uint4(0, 0, 0, 0);
  __syncthreads();
  // what a lane needs for its one result comes beside the weights
  const int n = n0 + lane / M, row = lane % M;
  const bool mine = lane < CHANNELS * M && row < p.M && n < p.N;
  const int64_t at = static_cast<int64_t>(row) * p.N + n;
  const Early bias(p.bias, p.bias_type, n, mine), scale(p.scale, p.scale_type, n, mine), residual(p.residual, p.residual_type, at, mine);
  float2 sum[CHANNELS][M];
#pragma unroll
  for (int i = 0; i < CHANNELS; ++i)
#pragma unroll
    for (int m = 0; m < M; ++m) sum[i][m] = both(0.f);
  for (int c0 = lane; c0 < chunks; c0 += 32 * kAhead) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int c = c0 + 32 * k;
      float2 now[CHANNELS][4];
#pragma unroll
      for (int i = 0; i < CHANNELS; ++i) {
        now[i][0] = pair_of<BF16>(w[k][i].x);
        now[i][1] = pair_of<BF16>(w[k][i].y);
        now[i][2] = pair_of<BF16>(w[k][i].z);
        now[i][3] = pair_of<BF16>(w[k][i].w);
      }
      fetch(c + 32 * kAhead, k);
      if (c >= chunks) continue;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const uint4 t = x[m * chunks + c];
        const float2 v[4] = {pair_of<BF16>(t.x), pair_of<BF16>(t.y), pair_of<BF16>(t.z), pair_of<BF16>(t.w)};
#pragma unroll
        for (int i = 0; i < CHANNELS; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) sum[i][m] = ffma2(now[i][j], v[j], sum[i][m]);
      }
    }
  }
  float result = 0.f;
#pragma unroll
  for (int i = 0; i < CHANNELS; ++i)
#pragma unroll
    for (int m = 0; m < M; ++m) {
      float total = sum[i][m].x + sum[i][m].y;
#pragma unroll
      for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      if (lane == i * M + m) result = total;
    }
  if (!mine) return;
  if (p.bias) result += bias.value(p.bias_type);
  float v[1];
  with_act(p.act, [&](auto act) {
    float2 slope;
    v[0] = activate<decltype(act)::value, false>(both(result), slope).x;
    return 0;
  });
  const float s = p.scale ? scale.value(p.scale_type) : 1.f;
  v[0] = p.residual ? __fmaf_rn(v[0], s, residual.value(p.residual_type)) : v[0] * s;
  Raw<1> o;
  pack<1>(o, v, p.out_type);
  store_raw<1>(o, p.out, p.out_type, at);
}

template <int M, int CHANNELS>
static int run_few_channels(const LinFewParams& p, cudaStream_t st) {
  static_assert(M * CHANNELS <= 32, "a lane per result");
  const int per = kLinFewWarps * CHANNELS;
  const unsigned grid = static_cast<unsigned>((p.N + per - 1) / per);
  const size_t smem = static_cast<size_t>(M) * ((p.K + 7) / 8) * 16;
  return p.type == S3R_BF16 ? launch(linear_few_kernel<M, true, CHANNELS>, grid, 32 * kLinFewWarps, smem, st, p)
                            : launch(linear_few_kernel<M, false, CHANNELS>, grid, 32 * kLinFewWarps, smem, st, p);
}
// One channel of 1024, a token: 2.9 us, two 3.2; of 4096 5.9 and 9.2.  4096 channels fill the SMs either way.
template <int M>
static int run_linear_few(const LinFewParams& p, cudaStream_t st) {
  return p.N <= kLinFewWarps * sm_count() ? run_few_channels<M, 1>(p, st) : run_few_channels<M, 2>(p, st);
}

// ---------------------------------------------------------------------------------------------------------------------
// the sums of a contraction's parts, in their order, and what follows them: a thread has four columns of a row, and all parts' loads in flight.
// Bound: the latency of those loads, from L2, where the parts have just been written (64 x 1024 in sixteen parts: 4 MB).
// ---------------------------------------------------------------------------------------------------------------------
struct JoinParams {
  const float* sums;                    // [parts][part_rows][pitch]
  const void *bias, *scale, *residual;
  void* out;
  int64_t M, part_rows;
  int N, pitch, parts, quads;
  int bias_type, scale_type, residual_type, out_type, act, vectors;
};
__global__ void __launch_bounds__(256) linear_join_kernel(const __grid_constant__ JoinParams p) {
  griddep_wait();
  griddep_launch();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, row = i / p.quads;
  if (row >= p.M) return;
  const int col = static_cast<int>(i - row * p.quads) * 4;
  const float* from = p.sums + row * p.pitch + col;
  const int64_t part = p.part_rows * p.pitch;
  const int64_t at = row * p.N + col;
  Early bias[4], scale[4], residual[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    bias[k] = Early(p.bias, p.bias_type, col + k, col + k < p.N);
    scale[k] = Early(p.scale, p.scale_type, col + k, col + k < p.N);
    residual[k] = Early(p.residual, p.residual_type, at + k, col + k < p.N);
  }
  float4 v[16];
#pragma unroll
  for (int s = 0; s < 16; ++s)
    if (s < p.parts) v[s] = __ldg(reinterpret_cast<const float4*>(from + s * part));
  float f[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
  for (int s = 1; s < 16; ++s)
    if (s < p.parts) f[0] += v[s].x, f[1] += v[s].y, f[2] += v[s].z, f[3] += v[s].w;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (p.bias) f[k] += bias[k].value(p.bias_type);
  with_act(p.act, [&](auto act) {
    float2 slope;
    const float2 a = activate<decltype(act)::value, false>(make_float2(f[0], f[1]), slope), b = activate<decltype(act)::value, false>(make_float2(f[2], f[3]), slope);
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
    return 0;
  });
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float s = p.scale ? scale[k].value(p.scale_type) : 1.f;
    f[k] = p.residual ? __fmaf_rn(f[k], s, residual[k].value(p.residual_type)) : f[k] * s;
  }
  if (p.vectors) {
    Raw<4> o;
    pack<4>(o, f, p.out_type);
    store_raw<4>(o, p.out, p.out_type, at);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (col + k < p.N) {
        const float one[1] = {f[k]};
        Raw<1> o;
        pack<1>(o, one, p.out_type);
        store_raw<1>(o, p.out, p.out_type, at + k);
      }
  }
}

// Bytes of the parts' sums, 0 where there is one part
static size_t part_bytes(const LinPlan& t, int64_t M, int64_t N) {
  return t.parts > 1 ? static_cast<size_t>(part_rows(M, t.ctas)) * t.parts * ((N + 3) / 4 * 4) * sizeof(float) : 0;
}
// The product with its epilogue (p: everything but its result) in parts
static int run_parts(const LinPlan& t, const LinOperand& a, const LinOperand& b, int64_t k, bool bf16, const LinParams& p, void* workspace, cudaStream_t st) {
  LinParams part = {};
  part.rows = p.M;
  part.N = p.N;
  part.parts = t.parts;
  part.out = workspace;
  part.out_pitch = (p.N + 3) / 4 * 4;
  part.out_type = S3R_F32;
  part.status = p.status;
  if (const int rc = linear_partial(a, b, k, bf16, part, st)) return rc;
  JoinParams j = {};
  j.sums = static_cast<const float*>(workspace);
  j.bias = p.bias;
  j.scale = p.scale;
  j.residual = p.other;
  j.out = p.out;
  j.M = p.M;
  j.part_rows = part_rows(p.M, t.ctas);
  j.N = p.N;
  j.pitch = static_cast<int>(part.out_pitch);
  j.parts = t.parts;
  j.quads = (p.N + 3) / 4;
  j.bias_type = p.bias_type;
  j.scale_type = p.scale_type;
  j.residual_type = p.other_type;
  j.out_type = p.out_type;
  j.act = p.act;
  const void* ptr[] = {p.out};
  j.vectors = row_vector(p.N, ptr, &p.out_type, 1) >= 4;
  const int64_t blocks = (p.M * j.quads + 255) / 256;
  S3R_REQUIRE(blocks < (1ll << 31), S3R_ERR_TOO_LARGE, "s3r_linear: too many rows");
  return launch(linear_join_kernel, static_cast<unsigned>(blocks), 256, 0, st, j);
}

// ---------------------------------------------------------------------------------------------------------------------
// dz = dy * scale where no z is needed, with its sums over rows.  Bound: HBM, dy read and dz written once.  A CTA has 64 rows and 256 columns, a
// thread eight columns of every eighth row.
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
    for (int64_t i = warp; i < p.blocks; i += 32 * 8) {            // eight on their way at a time
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = i + 32 * k < p.blocks ? __ldg(sums + (i + 32 * k) * p.N + col) : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) total += v[k];
    }
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
// rows of N elements all begin at multiples of `bytes`
static bool in_vectors(const void* p, int type, int N, int bytes) { return static_cast<int64_t>(N) * type_bytes(type) % bytes == 0 && reinterpret_cast<uintptr_t>(p) % bytes == 0; }

static bool is_few(int64_t M, int64_t K) { return M <= kLinFew && (M <= 2 ? M : M <= 4 ? 4 : 8) * ((K + 7) / 8 * 16) <= kLinFewBytes; }
// A workspace is used where it is given and large enough: without one the contraction stays in one part.
static bool has_room(const void* workspace, size_t bytes, size_t need) { return workspace && bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0; }

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

extern "C" size_t s3r_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  return M > 0 && N > 0 && K > 0 && M < (1ll << 31) && N < (1ll << 31) && K < (1ll << 31) && !is_few(M, K) ? part_bytes(linear_plan(M, N, K, true), M, N) : 0;
}

extern "C" int s3r_linear_fwd(const s3r_linear* f, void* stream) {
  if (const int rc = check_linear(f, "s3r_linear_fwd")) return rc;
  S3R_REQUIRE(f->out, S3R_ERR_NULL, "s3r_linear_fwd: NULL pointer");
  S3R_REQUIRE(at_multiple(f->out, f->out_type), S3R_ERR_ALIGNMENT, "s3r_linear_fwd: elements must be aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (is_few(f->M, f->K)) {
    const LinFewParams p = {static_cast<const uint16_t*>(f->x), static_cast<const uint16_t*>(f->weight), f->bias, f->scale, f->residual, f->out, f->x_pitch, f->w_pitch,
                            f->N, f->K, static_cast<int>(f->M), f->type, f->bias_type, f->scale_type, f->residual_type, f->out_type, f->act};
    return f->M == 1 ? run_linear_few<1>(p, st) : f->M == 2 ? run_linear_few<2>(p, st) : f->M <= 4 ? run_linear_few<4>(p, st) : run_linear_few<8>(p, st);
  }
  LinParams p = linear_params(f);
  S3R_REQUIRE(p.status, S3R_ERR_DRIVER, "s3r_linear_fwd: no status word");
  p.other = f->residual;
  p.other_type = f->residual_type;
  p.other_vectors = f->residual && in_vectors(f->residual, f->residual_type, f->N, 16);
  p.out = f->out;
  p.out_pitch = f->N;
  p.out_type = f->out_type;
  const LinOperand a = {f->x, f->x_pitch, false}, b = {f->weight, f->w_pitch, false};
  const bool bf16 = f->type == S3R_BF16;
  const LinPlan t = linear_plan(f->M, f->N, f->K, true);
  if (t.parts > 1 && has_room(f->workspace, f->workspace_bytes, part_bytes(t, f->M, f->N))) return run_parts(t, a, b, f->K, bf16, p, f->workspace, st);
  return f->residual ? linear_added(a, b, f->K, bf16, p, st) : f->out_type == S3R_F32 ? linear_wide(a, b, f->K, bf16, p, st) : linear_narrow(a, b, f->K, bf16, p, st);
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
    p.other = g->dy;
    p.other_type = f->out_type;
    p.other_vectors = in_vectors(g->dy, f->out_type, f->N, 2 * type_bytes(f->out_type));
    p.out = g->dz;
    p.out_pitch = g->dz ? g->dz_pitch : 8;
    p.out_type = f->type;
    p.bias_sums = bias_sums;
    p.scale_sums = scale_sums;
    rc = linear_dz({f->x, f->x_pitch, false}, {f->weight, f->w_pitch, false}, f->K, f->type == S3R_BF16, p, st);
    s.blocks = sum_blocks(f->M);
  }
  if (rc || !sums) return rc;
  int n = 0;
  if (g->d_bias) s.sums[n] = bias_sums, s.out[n] = g->d_bias, s.types[n] = f->bias_type, ++n;
  if (g->d_scale) s.sums[n] = scale_sums, s.out[n] = g->d_scale, s.types[n] = f->scale_type, ++n;
  return run_sums(s, n, st);
}

extern "C" int s3r_product(const void* a, int64_t a_pitch, int a_turned, const void* b, int64_t b_pitch, int b_turned, int type, void* out, int64_t M, int N,
                           int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
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
  const LinOperand left = {a, a_pitch, a_turned != 0}, right = {b, b_pitch, b_turned != 0};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const LinPlan t = linear_plan(M, N, K, true);
  if (t.parts > 1 && has_room(workspace, workspace_bytes, part_bytes(t, M, N))) return run_parts(t, left, right, K, type == S3R_BF16, p, workspace, st);
  return linear_narrow(left, right, K, type == S3R_BF16, p, st);
}
