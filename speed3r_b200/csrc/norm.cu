// A block's residual, gate, LayerScale and norms in one pass each way:
//   u = y | post_norm(y);  r = x + (u * scale) * gate;  h = norm(r)
// and backward, with xh = norm before its affine part, n = channels, s = 1 / sqrt(..):
//   G = dr + s (dh w - mean(dh w) - xh mean(dh w xh))        (RMS: without the first mean)
//   dx = G;  du = G scale gate;  dy = du, or the same formula through the post norm
//   dw = sum_rows dh xh;  db = sum_rows dh;  dscale = sum G gate u;  dgate = sum G scale u;  post norm alike
// Bound: HBM, each tensor once each way (fp32 residual and bf16 branch: 12 bytes per element forward, 18 backward).
#include "rows.cuh"

namespace s3r {

constexpr int kNormMaxChannels = 8192;

struct NormParams {
  s3r_residual_norm a;
  int64_t rows;
  float inv_n;
  int stages;                  // rows on their way (norm_rows_kernel)
};

__device__ __forceinline__ float gate_of_row(const s3r_residual_norm& a, int64_t row) {
  if (a.gate_mode != S3R_GATE_ROW) return 1.f;
  const uint32_t tokens = static_cast<uint32_t>(a.tokens), b = static_cast<uint32_t>(row) / tokens;      // rows fit 31 bits
  return load_one(a.gate, a.gate_type, b * a.gate_stride_b + (static_cast<uint32_t>(row) - b * tokens) * a.gate_stride_t);
}

// ---------------------------------------------------------------------------------------------------------------------
// forward: G threads per row, E elements per thread in registers (vectors of W); the variance from the centred values
// ---------------------------------------------------------------------------------------------------------------------
template <int W, int G, int E>
__device__ __forceinline__ float2 row_statistics(const float (&v)[E], int kind, int channels, float inv_n, float eps, float* red, uint32_t& turn, int t,
                                                 int bar = 0) {
  float s[1] = {0.f};
  float mean = 0.f;
  if (kind == S3R_NORM_LAYER) {
#pragma unroll
    for (int k = 0; k < E; ++k) s[0] += v[k];            // places behind the row hold 0
    row_sum<G>(s, red, turn, t, bar);
    mean = s[0] * inv_n;
  }
  s[0] = 0.f;
#pragma unroll
  for (int i = 0; i < E / W; ++i)
    if ((i * G + t) * W < channels)
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const float d = v[i * W + k] - mean;
        s[0] = fmaf(d, d, s[0]);
      }
  row_sum<G>(s, red, turn, t, bar);
  return make_float2(mean, rsqrtf(fmaf(s[0], inv_n, eps)));
}

// A thread's places of `channels` elements from element `from` on, asked for.  Single elements (rows of odd width) in one branch on the
// type: their addresses are then one register and constants, where predicates took one each.
template <int W, int G, int N>
__device__ __forceinline__ void request_all(Raw<W> (&r)[N], const void* p, int type, int64_t from, int channels, int t, bool there = true) {
  if constexpr (W > 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) load_raw<W>(r[i], p, type, from + (i * G + t) * W, there && p && (i * G + t) * W < channels);
  } else if (there && p) {
    if (type == S3R_F32) {
      const uint32_t* q = static_cast<const uint32_t*>(p) + from + t;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i * G + t < channels) r[i].v[0] = __ldg(q + i * G);
    } else {
      const uint16_t* q = static_cast<const uint16_t*>(p) + from + t;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i * G + t < channels) r[i].v[0] = __ldg(q + i * G);
    }
  }
}
// [channels] parameters of a thread's places
template <int W, int G, int N>
__device__ __forceinline__ void load_params(float (&f)[W * N], const void* p, int type, int64_t from, int channels, int t) {
  Raw<W> r[N];
  request_all<W, G, N>(r, p, type, from, channels, t);
  unpack_all<W, N>(f, r, type, [](int) { return true; });
}

template <int W, int N>
__device__ __forceinline__ void apply_norm(float (&v)[W * N], float2 st, const void* weight, const Raw<W> (&w)[N], const void* bias, const Raw<W> (&b)[N],
                                           int type) {
  float p[W * N];
  const auto all = [](int) { return true; };
#pragma unroll
  for (int k = 0; k < W * N; ++k) v[k] = (v[k] - st.x) * st.y;
  if (weight) {
    unpack_all<W, N>(p, w, type, all);
#pragma unroll
    for (int k = 0; k < W * N; ++k) v[k] *= p[k];
  }
  if (bias) {
    unpack_all<W, N>(p, b, type, all);
#pragma unroll
    for (int k = 0; k < W * N; ++k) v[k] += p[k];
  }
}

// the row as 8-bit tokens
template <int W, int G, int E>
__device__ __forceinline__ void store_int8(const float (&v)[E], const s3r_residual_norm& a, int64_t row, float* red, uint32_t& turn, int t, int bar) {
  float big = 0.f;
#pragma unroll
  for (int i = 0; i < E / W; ++i)
    if ((i * G + t) * W < a.channels) big = max_abs<W>(big, v + i * W);
  big = row_max<G>(big, red, turn, t, bar);
  const RowScale s = row_scale(big);
  if (t == 0) a.q_scale[row] = s.scale;
#pragma unroll
  for (int i = 0; i < E / W; ++i) {
    if ((i * G + t) * W < a.channels) {
      int8_t* q = a.q + row * a.q_pitch + (i * G + t) * W;
      if constexpr (W == 1) {
        *q = static_cast<int8_t>(to_s8(v[i], s.inverse));
      } else {
#pragma unroll
        for (int k = 0; k < W; k += 4) *reinterpret_cast<uint32_t*>(q + k) = to_s8x4(v + i * W + k, s.inverse);
      }
    }
  }
}

// threads of a CTA that has groups of G, each a row
__host__ __device__ constexpr int cta_threads(int G) { return G < 96 ? 128 : G; }
template <int W, int G, int E>
__global__ void __launch_bounds__(cta_threads(G)) norm_fwd_kernel(const __grid_constant__ NormParams p) {
  constexpr int kRows = cta_threads(G) / G, N = E / W;
  __shared__ float red_all[kRows][G > 32 ? 8 * (G / 32) : 1];
  griddep_wait();
  griddep_launch();
  const s3r_residual_norm& a = p.a;
  const int t = threadIdx.x % G, C = a.channels, group = threadIdx.x / G, bar = group + 1;
  float* red = red_all[group];
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + group;
  if (row >= p.rows) return;                              // whole rows leave, each with a barrier of its own
  const int64_t at = row * C;
  uint32_t turn = 0;
  auto in = [&](int i) { return (i * G + t) * W < C; };
  auto place = [&](int i) { return in(i) ? at + (i * G + t) * W : int64_t{-1}; };
  Raw<W> xr[N], yr[N], sr[N], gr[N], wr[N], br[N];
  request_all<W, G, N>(xr, a.x, a.x_type, at, C, t);
  request_all<W, G, N>(yr, a.y, a.y_type, at, C, t);
  request_all<W, G, N>(sr, a.scale, a.param_type, 0, C, t);
  float v[E], f[E];
  if (a.y) {
    unpack_all<W, N>(v, yr, a.y_type, in);
    if (a.post) {
      const float2 st = row_statistics<W, G, E>(v, a.kind, C, p.inv_n, a.post_eps, red, turn, t, bar);
      if (a.stats && t == 0) a.stats[2 * p.rows + row] = st.x, a.stats[3 * p.rows + row] = st.y;
      request_all<W, G, N>(wr, a.post_weight, a.param_type, 0, C, t);
      request_all<W, G, N>(br, a.post_bias, a.param_type, 0, C, t);
      apply_norm<W, N>(v, st, a.post_weight, wr, a.post_bias, br, a.param_type);
    }
    if (a.scale) {
      unpack_all<W, N>(f, sr, a.param_type, [](int) { return true; });
#pragma unroll
      for (int k = 0; k < E; ++k) v[k] = __fmul_rn(v[k], f[k]);
    }
    if (a.gate_mode == S3R_GATE_CHANNEL) {
      request_all<W, G, N>(gr, a.gate, a.gate_type, static_cast<uint32_t>(row) / static_cast<uint32_t>(a.tokens) * a.gate_stride_b, C, t);
      unpack_all<W, N>(f, gr, a.gate_type, [](int) { return true; });
#pragma unroll
      for (int k = 0; k < E; ++k) v[k] = __fmul_rn(v[k], f[k]);
    } else if (a.gate_mode == S3R_GATE_ROW) {
      const float gate = gate_of_row(a, row);
#pragma unroll
      for (int k = 0; k < E; ++k) v[k] = __fmul_rn(v[k], gate);
    }
    unpack_all<W, N>(f, xr, a.x_type, in);
#pragma unroll
    for (int k = 0; k < E; ++k) v[k] = __fadd_rn(f[k], v[k]);
    // the norm is that of the stored sum, as it is for whoever reads it later, the backward among them
    store_all<W, N>(v, a.r, a.x_type, place, true);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (!in(i))
#pragma unroll
        for (int k = 0; k < W; ++k) v[i * W + k] = 0.f;
  } else {
    unpack_all<W, N>(v, xr, a.x_type, in);
    if (a.r) store_all<W, N>(v, a.r, a.x_type, place);
  }
  if (!a.h && !a.q) return;
  const float2 st = row_statistics<W, G, E>(v, a.kind, C, p.inv_n, a.eps, red, turn, t, bar);
  if (a.stats && t == 0) a.stats[row] = st.x, a.stats[p.rows + row] = st.y;
  request_all<W, G, N>(wr, a.weight, a.param_type, 0, C, t);
  request_all<W, G, N>(br, a.bias, a.param_type, 0, C, t);
  apply_norm<W, N>(v, st, a.weight, wr, a.bias, br, a.param_type);
  if (a.h) {
    store_all<W, N>(v, a.h, a.h_type, place);
    return;
  }
  store_int8<W, G, E>(v, a, row, red, turn, t, bar);
}

// CTAs per SM.  An fp32 sum: 512 threads and 128 registers (64 512 x 1024 122 us; 768 threads of 80 registers 149, 512 such 156).  16 bits:
// 768 threads, a row's bytes are fewer and its arithmetic the same (94 us, with 512 101).
__host__ __device__ constexpr int rows_resident(int G, bool full, bool wide) {
  return G > 256 ? 1 : G == 192 && (full || wide) ? 3 : (full || wide || G < 96 ? 512 : 768) / cta_threads(G);
}
// The same for many rows: CTAs stay, take every gridDim-th row, keep the parameters in registers and have the next rows on their way into
// shared memory (cp.async, each thread its own bytes, so that no barrier orders them).  With a CTA per row a row cost 2 ns whatever its
// bytes, the time it takes to start, wait for three loads one behind the other and end.
template <int W, int G, int E, bool FULL, bool WIDE>
__global__ void __launch_bounds__(cta_threads(G), rows_resident(G, FULL, WIDE)) norm_rows_kernel(const __grid_constant__ NormParams p) {
  constexpr int kThreads = cta_threads(G), kRows = kThreads / G, N = E / W, P = E / 2;
  extern __shared__ __align__(16) char smem[];
  __shared__ float red_all[kRows][G > 32 ? 8 * (G / 32) : 1];
  griddep_wait();
  griddep_launch();
  const s3r_residual_norm& a = p.a;
  const int t = threadIdx.x % G, group = threadIdx.x / G, C = a.channels, rows = static_cast<int>(p.rows);
  const int step = static_cast<int>(gridDim.x) * kRows, first = static_cast<int>(blockIdx.x) * kRows + group, bar = group + 1;
  float* red = red_all[group];
  uint32_t turn = 0;
  auto in = [&](int i) { return (i * G + t) * W < C; };
  const int xb = type_bytes(a.x_type), yb = type_bytes(a.y_type);
  const uint32_t at_y = G * E * xb, stage_bytes = at_y + G * E * yb;
  char* ring = smem + static_cast<size_t>(group) * p.stages * stage_bytes;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (!in(i))
      for (int s = 0; s < p.stages; ++s) {
        zero_place<W>(ring + s * stage_bytes + (i * G + t) * W * xb, xb);
        zero_place<W>(ring + s * stage_bytes + at_y + (i * G + t) * W * yb, yb);
      }
  auto request = [&](int row, int stage) {
    if (row < rows) {
      const uint32_t to = smem_u32(ring) + stage * stage_bytes;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = (i * G + t) * W;
        const int64_t at = static_cast<int64_t>(row) * C + c;
        if (c < C) {
          stage_vector<W>(to + c * xb, a.x, a.x_type, at);
          if (a.y) stage_vector<W>(to + at_y + c * yb, a.y, a.y_type, at);
        }
      }
    }
    cp_async_commit();
  };
  float2 w[P], b[P], scale[P], pw[FULL ? P : 1], pb[FULL ? P : 1];
  auto param = [&](float2* to, const void* from, int type, int64_t at, float other) {
    float v[E];
    if (from) load_params<W, G, N>(v, from, type, at, C, t);
#pragma unroll
    for (int k = 0; k < P; ++k) to[k] = !in(2 * k / W) ? make_float2(0.f, 0.f) : from ? make_float2(v[2 * k], v[2 * k + 1]) : make_float2(other, other);
  };
  for (int s = 0; s + 1 < p.stages; ++s) request(first + s * step, s);
  param(w, a.weight, a.param_type, 0, 1.f);
  param(b, a.bias, a.param_type, 0, 0.f);
  param(scale, a.scale, a.param_type, 0, 1.f);
  if constexpr (FULL) {
    param(pw, a.post_weight, a.param_type, 0, 1.f);
    param(pb, a.post_bias, a.param_type, 0, 0.f);
  }
  auto both = [](float x) { return make_float2(x, x); };
  // (mean, 1 / sqrt(..)); values behind the end of the row are 0
  auto statistics = [&](const float2 (&v)[P], float eps) {
    float sum[1] = {0.f};
    float2 s = both(0.f);
    float mean = 0.f;
    if (a.kind == S3R_NORM_LAYER) {
#pragma unroll
      for (int k = 0; k < P; ++k) s = fadd2(s, v[k]);
      sum[0] = s.x + s.y;
      row_sum<G>(sum, red, turn, t, bar);
      mean = sum[0] * p.inv_n;
      s = both(0.f);
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (in(i))
#pragma unroll
        for (int k = 0; k < W / 2; ++k) {
          const float2 d = fadd2(v[i * (W / 2) + k], both(-mean));
          s = ffma2(d, d, s);
        }
    sum[0] = s.x + s.y;
    row_sum<G>(sum, red, turn, t, bar);
    return make_float2(mean, rsqrtf(fmaf(sum[0], p.inv_n, eps)));
  };
  int stage = 0;
  for (int row = first; row < rows; row += step) {
    request(row + (p.stages - 1) * step, stage + p.stages - 1 >= p.stages ? stage - 1 : p.stages - 1);
    const float gate = gate_of_row(a, row);
    cp_async_wait_for(p.stages - 1);
    const char* here = ring + stage * stage_bytes;
    stage = stage + 1 == p.stages ? 0 : stage + 1;
    auto place = [&](int i) { return in(i) ? static_cast<int64_t>(row) * C + (i * G + t) * W : int64_t{-1}; };
    auto fetch = [&](float2 (&v)[P], uint32_t at, int type) {
      Raw<W> r[N];
      float e[E];
#pragma unroll
      for (int i = 0; i < N; ++i) staged_raw<W>(r[i], here + at + (i * G + t) * W * type_bytes(type), type);
      unpack_all<W, N>(e, r, type, [](int) { return true; });
#pragma unroll
      for (int k = 0; k < P; ++k) v[k] = make_float2(e[2 * k], e[2 * k + 1]);
    };
    auto put = [&](float2 (&v)[P], void* to, int type, bool back) {
      float e[E];
#pragma unroll
      for (int k = 0; k < P; ++k) e[2 * k] = v[k].x, e[2 * k + 1] = v[k].y;
      store_all<W, N>(e, to, type, place, back);
      if (back)
#pragma unroll
        for (int k = 0; k < P; ++k) v[k] = make_float2(e[2 * k], e[2 * k + 1]);
    };
    float2 v[P], f[P];
    if (a.y) {
      fetch(v, at_y, a.y_type);
      if constexpr (FULL) {
        if (a.post) {
          const float2 st = statistics(v, a.post_eps);
          if (a.stats && t == 0) a.stats[2 * p.rows + row] = st.x, a.stats[3 * p.rows + row] = st.y;
#pragma unroll
          for (int k = 0; k < P; ++k) v[k] = ffma2(fmul2(fadd2(v[k], both(-st.x)), both(st.y)), pw[k], pb[k]);
        }
      }
      // products and sum are rounded one by one, as in separate operations (norm_fwd_kernel's r, bit for bit)
      if (a.scale)
#pragma unroll
        for (int k = 0; k < P; ++k) v[k] = fmul2(v[k], scale[k]);
      if (a.gate_mode == S3R_GATE_ROW) {
#pragma unroll
        for (int k = 0; k < P; ++k) v[k] = fmul2(v[k], both(gate));
      }
      if constexpr (FULL) {
        if (a.gate_mode == S3R_GATE_CHANNEL) {
          param(f, a.gate, a.gate_type, static_cast<uint32_t>(row) / static_cast<uint32_t>(a.tokens) * a.gate_stride_b, 1.f);
#pragma unroll
          for (int k = 0; k < P; ++k) v[k] = fmul2(v[k], f[k]);
        }
      }
      fetch(f, 0, a.x_type);
#pragma unroll
      for (int k = 0; k < P; ++k) v[k] = add_apart(f[k], v[k]);
      put(v, a.r, a.x_type, true);
    } else {
      fetch(v, 0, a.x_type);
      if (a.r) put(v, a.r, a.x_type, false);
    }
    if (!a.h && !a.q) continue;
    const float2 st = statistics(v, a.eps);
    if (a.stats && t == 0) a.stats[row] = st.x, a.stats[p.rows + row] = st.y;
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = ffma2(fmul2(fadd2(v[k], both(-st.x)), both(st.y)), w[k], b[k]);
    if (a.h) {
      put(v, a.h, a.h_type, false);
    } else {
      float e[E];
#pragma unroll
      for (int k = 0; k < P; ++k) e[2 * k] = v[k].x, e[2 * k + 1] = v[k].y;
      store_int8<W, G, E>(e, a, row, red, turn, t, bar);
    }
  }
  cp_async_wait<0>();
}

// ---------------------------------------------------------------------------------------------------------------------
// backward: a CTA owns consecutive rows of one batch entry (of all rows where no gate is summed per batch entry), a thread the
// same columns of all of them, whose sums over rows it keeps in registers.  Rows are on their way into shared memory several
// ahead (cp.async, each thread its own bytes, so that no barrier orders them).
// ---------------------------------------------------------------------------------------------------------------------
enum { kSumWeight, kSumBias, kSumScale, kSumPostWeight, kSumPostBias, kSumGate, kSums };

struct NormBwdParams {
  s3r_residual_norm f;
  s3r_residual_norm_grad g;
  int64_t rows, span;          // rows of a batch entry (all rows)
  int slices;                  // per batch entry
  int stages;
  uint32_t stage_bytes;
  uint32_t at_y, at_dr, at_dh; // of a stage, behind r
  float inv_n;
  int sums;                    // that are wanted, and the place of each among them
  int place[kSums];
  float* partial;              // [batch entries x slices, sums, channels]
};

// CTAs per SM: 128 registers per thread, in a FULL backward 168.  The grid has as many as are resident: with a second, shorter round of CTAs
// 12 288 x 1024, fp32, post norm took 75 us instead of 58, and the sums over CTAs had a third more to read.
__host__ __device__ constexpr int bwd_resident(int G, bool full) {
  return G > 256 ? 1 : (full ? 384 : 512) / cta_threads(G);
}
// FULL: a post norm or a gate per channel too; without them their sums and factors take no registers
template <int W, int G, int E, bool FULL>
__global__ void __launch_bounds__(cta_threads(G), bwd_resident(G, FULL)) norm_bwd_kernel(const __grid_constant__ NormBwdParams p) {
  constexpr int kRows = cta_threads(G) / G, N = E / W, P = E / 2, F = FULL ? P : 1;
  extern __shared__ __align__(16) char smem[];
  __shared__ float red[kRows][G > 32 ? 8 * (G / 32) : 1];
  griddep_wait();
  griddep_launch();
  const s3r_residual_norm& f = p.f;
  const s3r_residual_norm_grad& g = p.g;
  const int t = threadIdx.x % G, group = threadIdx.x / G, C = f.channels;
  const int entry = blockIdx.x / p.slices, slice = blockIdx.x % p.slices;
  const int first = static_cast<int>(entry * p.span + p.span * slice / p.slices), last = static_cast<int>(entry * p.span + p.span * (slice + 1) / p.slices);
  const bool layer = f.kind == S3R_NORM_LAYER, branch = f.y != nullptr, norm = g.dh != nullptr, wants_gate = g.d_gate_row != nullptr;
  const bool reads_y = branch && (f.post || g.d_scale || g.d_gate_row || g.d_gate_channel);
  char* ring = smem + static_cast<size_t>(group) * p.stages * p.stage_bytes;
  uint32_t turn = 0;
  auto in = [&](int i) { return (i * G + t) * W < C; };

  float2 w[P], scale[P], gate_c[F], pw[F], pb[F];
  float2 d_w[P], d_b[P], d_s[P], d_g[F], d_pw[F], d_pb[F];
  auto param = [&](float2* to, const void* from, int type, int64_t at, float other) {
    float v[E];
    if (from) {
      load_params<W, G, N>(v, from, type, at, C, t);
    } else {
#pragma unroll
      for (int k = 0; k < E; ++k) v[k] = other;
    }
#pragma unroll
    for (int k = 0; k < P; ++k) to[k] = in(2 * k / W) ? make_float2(v[2 * k], W == 1 && !in(2 * k + 1) ? 0.f : v[2 * k + 1]) : make_float2(0.f, 0.f);
  };
  param(w, f.weight, f.param_type, 0, 1.f);
  param(scale, f.scale, f.param_type, 0, 1.f);
  if constexpr (FULL) {
    param(gate_c, f.gate_mode == S3R_GATE_CHANNEL ? f.gate : nullptr, f.gate_type, entry * f.gate_stride_b, 1.f);
    param(pw, f.post_weight, f.param_type, 0, 1.f);
    param(pb, f.post_bias, f.param_type, 0, 0.f);
  }
  const float2 nil = make_float2(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < P; ++k) {
    d_w[k] = d_b[k] = d_s[k] = nil;
    if constexpr (FULL) d_g[k] = d_pw[k] = d_pb[k] = nil;
  }

  // Places behind the end of a row: zeros that no copy overwrites, so that nothing has to be masked out further down (their
  // factors are 0 as well).
  const int xb = type_bytes(f.x_type), yb = type_bytes(f.y_type), hb = type_bytes(f.h_type);
  if constexpr (W > 1)
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (!in(i))
        for (int s = 0; s < p.stages; ++s) {
          char* to = ring + s * p.stage_bytes;
          const int c = (i * G + t) * W;
          zero_place<W>(to + c * xb, xb);
          zero_place<W>(to + p.at_y + c * yb, yb);
          zero_place<W>(to + p.at_dr + c * xb, xb);
          zero_place<W>(to + p.at_dh + c * hb, hb);
        }

  auto request = [&](int row, int stage) {
    if constexpr (W > 1) {
      if (row < last) {
        const uint32_t to = smem_u32(ring) + stage * p.stage_bytes;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int c = (i * G + t) * W;
          const int64_t at = static_cast<int64_t>(row) * C + c;
          if (c < C) {
            if (norm) stage_vector<W>(to + c * xb, f.r, f.x_type, at);
            if (reads_y) stage_vector<W>(to + p.at_y + c * yb, f.y, f.y_type, at);
            if (g.dr) stage_vector<W>(to + p.at_dr + c * xb, g.dr, f.x_type, at);
            if (norm) stage_vector<W>(to + p.at_dh + c * hb, g.dh, f.h_type, at);
          }
        }
      }
      cp_async_commit();
    }
  };
  // rows of odd width: one element at a time, a row ahead in registers
  constexpr int M = W == 1 ? N : 1;
  Raw<1> odd[4][M];
  auto request_odd = [&](int row) {
    if constexpr (W == 1) {
      const int64_t at = static_cast<int64_t>(row) * C;
      const bool there = row < last;
      request_all<1, G, N>(odd[0], f.r, f.x_type, at, C, t, there && norm);
      request_all<1, G, N>(odd[1], f.y, f.y_type, at, C, t, there && reads_y);
      request_all<1, G, N>(odd[2], g.dr, f.x_type, at, C, t, there);
      request_all<1, G, N>(odd[3], g.dh, f.h_type, at, C, t, there);
    }
  };
  // a thread's values of the present row, in pairs
  auto fetch = [&](float2 (&v)[P], const char* staged_at, int which, int type) {
    float e[E];
    if constexpr (W > 1) {
      Raw<W> r[N];
#pragma unroll
      for (int i = 0; i < N; ++i) staged_raw<W>(r[i], staged_at + (i * G + t) * W * type_bytes(type), type);
      unpack_all<W, N>(e, r, type, [](int) { return true; });
    } else {
      unpack_all<W, N>(e, odd[which], type, in);
    }
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = make_float2(e[2 * k], e[2 * k + 1]);
  };
  auto put = [&](float2 (&v)[P], void* to, int type, int row) {
    float e[E];
#pragma unroll
    for (int k = 0; k < P; ++k) e[2 * k] = v[k].x, e[2 * k + 1] = v[k].y;
    store_all<W, N>(e, to, type, [&](int i) { return in(i) ? static_cast<int64_t>(row) * C + (i * G + t) * W : int64_t{-1}; });
  };
  auto both = [](float x) { return make_float2(x, x); };
  // a row's mean, 1 / sqrt(..), those of the post norm, and its gate, a row ahead
  float ahead[5];
  auto scalars = [&](int row) {
    const int r = row < last ? row : last - 1;
    ahead[0] = norm ? __ldg(f.stats + r) : 0.f;
    ahead[1] = norm ? __ldg(f.stats + p.rows + r) : 0.f;
    ahead[2] = FULL && f.post ? __ldg(f.stats + 2 * p.rows + r) : 0.f;
    ahead[3] = FULL && f.post ? __ldg(f.stats + 3 * p.rows + r) : 0.f;
    ahead[4] = gate_of_row(f, r);
  };

  int stage = 0;
  for (int s = 0; s + 1 < p.stages; ++s) request(first + group + s * kRows, s);
  if (first + group < last) {
    scalars(first + group);
    request_odd(first + group);
  }
  for (int row = first + group; row < last; row += kRows) {
    request(row + (p.stages - 1) * kRows, stage + p.stages - 1 >= p.stages ? stage - 1 : p.stages - 1);
    const float mean = ahead[0], inv = ahead[1], p_mean = ahead[2], p_inv = ahead[3], gate = ahead[4];
    scalars(row + kRows);
    if constexpr (W > 1) cp_async_wait_for(p.stages - 1);
    const char* here = ring + stage * p.stage_bytes;
    stage = stage + 1 == p.stages ? 0 : stage + 1;

    float2 xh[P], d[P];
    if (norm) {
      float2 dh[P], s0 = nil, s1 = nil;
      fetch(xh, here, 0, f.x_type);
      fetch(dh, here + p.at_dh, 3, f.h_type);
#pragma unroll
      for (int k = 0; k < P; ++k) {
        xh[k] = fmul2(fadd2(xh[k], both(-mean)), both(inv));
        d_w[k] = ffma2(dh[k], xh[k], d_w[k]);
        d_b[k] = fadd2(dh[k], d_b[k]);
        d[k] = fmul2(dh[k], w[k]);
        s0 = fadd2(s0, d[k]);
        s1 = ffma2(d[k], xh[k], s1);
      }
      float sums[2] = {s0.x + s0.y, s1.x + s1.y};
      row_sum<G>(sums, red[group], turn, t, group + 1);
      const float along = sums[1] * p.inv_n, flat = layer ? sums[0] * p.inv_n : 0.f;
#pragma unroll
      for (int k = 0; k < P; ++k) d[k] = fmul2(ffma2(xh[k], both(-along), fadd2(d[k], both(-flat))), both(inv));
      if (g.dr) {
        fetch(dh, here + p.at_dr, 2, f.x_type);
#pragma unroll
        for (int k = 0; k < P; ++k) d[k] = fadd2(d[k], dh[k]);
      }
    } else {
      fetch(d, here + p.at_dr, 2, f.x_type);
    }
    put(d, g.dx, f.x_type, row);
    if (!branch) {
      request_odd(row + kRows);
      continue;
    }
    // Where the branch is not read its place is not staged either: whatever is there is multiplied into sums that nobody wants.
    float2 u[P], gate_sum = nil, s0 = nil, s1 = nil;
    if (reads_y) {
      fetch(u, here + p.at_y, 1, f.y_type);
    } else {
#pragma unroll
      for (int k = 0; k < P; ++k) u[k] = nil;
    }
    request_odd(row + kRows);
    if constexpr (FULL) {
      if (f.post)
#pragma unroll
        for (int k = 0; k < P; ++k) {
          xh[k] = fmul2(fadd2(u[k], both(-p_mean)), both(p_inv));
          u[k] = ffma2(xh[k], pw[k], pb[k]);
        }
    }
    if (FULL || wants_gate)
#pragma unroll
      for (int k = 0; k < P; ++k) {
        const float2 of_gate = fmul2(fmul2(d[k], scale[k]), u[k]);
        gate_sum = fadd2(gate_sum, of_gate);
        if constexpr (FULL) d_g[k] = fadd2(d_g[k], of_gate);
      }
#pragma unroll
    for (int k = 0; k < P; ++k) {
      d[k] = fmul2(d[k], both(gate));
      if constexpr (FULL) d[k] = fmul2(d[k], gate_c[k]);
      d_s[k] = ffma2(d[k], u[k], d_s[k]);
      d[k] = fmul2(d[k], scale[k]);
    }
    if constexpr (FULL) {
      if (f.post)
#pragma unroll
        for (int k = 0; k < P; ++k) {
          d_pw[k] = ffma2(d[k], xh[k], d_pw[k]);
          d_pb[k] = fadd2(d[k], d_pb[k]);
          d[k] = fmul2(d[k], pw[k]);
          s0 = fadd2(s0, d[k]);
          s1 = ffma2(d[k], xh[k], s1);
        }
    }
    if ((FULL && f.post) || wants_gate) {
      float sums[3] = {s0.x + s0.y, s1.x + s1.y, gate_sum.x + gate_sum.y};
      row_sum<G>(sums, red[group], turn, t, group + 1);
      if (wants_gate && t == 0) g.d_gate_row[row] = sums[2];
      if constexpr (FULL) {
        if (f.post) {
          const float along = sums[1] * p.inv_n, flat = layer ? sums[0] * p.inv_n : 0.f;
#pragma unroll
          for (int k = 0; k < P; ++k) d[k] = fmul2(ffma2(xh[k], both(-along), fadd2(d[k], both(-flat))), both(p_inv));
        }
      }
    }
    if (g.dy) put(d, g.dy, f.y_type, row);
  }

  // this CTA's sums over rows; groups of one CTA are added in order
  float* out = p.partial + static_cast<int64_t>(blockIdx.x) * p.sums * C;
  auto leave = [&](const float2* sums, int which, bool wanted) {
    if (!wanted) return;
    if constexpr (kRows > 1) {
      __syncthreads();                                  // the ring, or the sums before these
      float2* shared = reinterpret_cast<float2*>(smem);
#pragma unroll
      for (int k = 0; k < P; ++k) shared[(group * P + k) * G + t] = sums[k];
      __syncthreads();
      if (group) return;
    }
    float e[E];
#pragma unroll
    for (int k = 0; k < P; ++k) {
      float2 s = sums[k];
      if constexpr (kRows > 1) {
        const float2* shared = reinterpret_cast<const float2*>(smem);
#pragma unroll
        for (int o = 1; o < kRows; ++o) s = fadd2(s, shared[(o * P + k) * G + t]);
      }
      e[2 * k] = s.x, e[2 * k + 1] = s.y;
    }
    // workspaces begin anywhere: one element at a time
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (in(i))
#pragma unroll
        for (int k = 0; k < W; ++k) out[p.place[which] * C + (i * G + t) * W + k] = e[i * W + k];
  };
  if constexpr (W > 1) cp_async_wait<0>();
  leave(d_w, kSumWeight, g.d_weight != nullptr);
  leave(d_b, kSumBias, g.d_bias != nullptr);
  leave(d_s, kSumScale, g.d_scale != nullptr);
  if constexpr (FULL) {
    leave(d_pw, kSumPostWeight, g.d_post_weight != nullptr);
    leave(d_pb, kSumPostBias, g.d_post_bias != nullptr);
    leave(d_g, kSumGate, g.d_gate_channel != nullptr);
  }
}

struct NormSumsParams {
  const float* partial;
  void* out[kSums + 1];
  int n, channels, slices, entries;    // entries: batch entries of the gate (its slices are summed apart)
  int sums, place[kSums + 1];          // of a slice; the gate's place stands last
  int type, gate_type;
};

// sums of the CTAs' sums: 32 columns per CTA, its 32 warps take turns at the slices
__global__ void __launch_bounds__(1024) norm_sums_kernel(const __grid_constant__ NormSumsParams p) {
  __shared__ float red[32][33];
  griddep_wait();
  griddep_launch();
  const int columns = (p.channels + 31) / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t job = blockIdx.x / columns;
  const int c = static_cast<int>(blockIdx.x % columns) * 32 + lane;
  const bool gate = job >= p.n;
  const int place = p.place[gate ? p.n : job];
  const int64_t entry = gate ? job - p.n : 0;
  const int64_t first = gate ? entry * p.slices : 0, last = gate ? first + p.slices : static_cast<int64_t>(p.entries) * p.slices;
  float s = 0.f;
  if (c < p.channels)
#pragma unroll 8
    for (int64_t i = first + warp; i < last; i += 32) s += __ldg(p.partial + (i * p.sums + place) * p.channels + c);
  red[warp][lane] = s;
  __syncthreads();
  // a warp sums a column (lane: a warp's part), in a tree: the same order every time
  float f[1] = {red[lane][warp]};
#pragma unroll
  for (int o = 16; o; o >>= 1) f[0] += __shfl_xor_sync(0xffffffffu, f[0], o);
  const int column = static_cast<int>(blockIdx.x % columns) * 32 + warp;
  if (lane == 0 && column < p.channels) {
    Raw<1> o;
    pack<1>(o, f, gate ? p.gate_type : p.type);
    store_raw<1>(o, p.out[gate ? p.n : job], gate ? p.gate_type : p.type, gate ? entry * p.channels + column : column);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------------
static int check_args(const s3r_residual_norm& a, const char* what) {
  S3R_REQUIRE(a.batch > 0 && a.tokens > 0 && a.channels > 0, S3R_ERR_SHAPE, "%s: sizes must be positive", what);
  S3R_REQUIRE(a.channels <= kNormMaxChannels, S3R_ERR_TOO_LARGE, "%s: %d channels (at most %d)", what, a.channels, kNormMaxChannels);
  S3R_REQUIRE(a.batch < (1ll << 31) && a.tokens < (1ll << 31) && a.batch * a.tokens < (1ll << 31) - (1 << 20), S3R_ERR_TOO_LARGE, "%s: too many rows", what);
  S3R_REQUIRE(a.kind == S3R_NORM_LAYER || a.kind == S3R_NORM_RMS, S3R_ERR_UNSUPPORTED, "%s: kind %d", what, a.kind);
  S3R_REQUIRE(known_type(a.x_type) && known_type(a.y_type) && known_type(a.h_type) && known_type(a.param_type) && known_type(a.gate_type),
              S3R_ERR_UNSUPPORTED, "%s: types are fp32, bf16 and fp16", what);
  S3R_REQUIRE(a.gate_mode >= S3R_GATE_NONE && a.gate_mode <= S3R_GATE_CHANNEL, S3R_ERR_UNSUPPORTED, "%s: gate mode %d", what, a.gate_mode);
  S3R_REQUIRE((a.gate_mode == S3R_GATE_NONE) == (a.gate == nullptr), S3R_ERR_NULL, "%s: a gate and its mode come together", what);
  S3R_REQUIRE(a.y || (!a.post && !a.scale && !a.gate), S3R_ERR_NULL, "%s: scale, gate and post norm need a branch", what);
  const void* ptr[] = {a.x, a.y, a.r, a.h, a.weight, a.bias, a.scale, a.post_weight, a.post_bias, a.gate};
  const int type[] = {a.x_type, a.y_type, a.x_type, a.h_type, a.param_type, a.param_type, a.param_type, a.param_type, a.param_type, a.gate_type};
  for (int i = 0; i < 10; ++i)
    S3R_REQUIRE(reinterpret_cast<uintptr_t>(ptr[i]) % type_bytes(type[i]) == 0, S3R_ERR_ALIGNMENT, "%s: elements must be aligned", what);
  return 0;
}

static int gate_vector(const s3r_residual_norm& a) {
  if (a.gate_mode != S3R_GATE_CHANNEL) return 8;
  const int64_t step = a.gate_stride_b;
  return step % 8 == 0 ? 8 : step % 4 == 0 ? 4 : 1;
}

template <int W, int G, int E, bool FULL, bool WIDE>
static int run_rows(NormParams p, cudaStream_t st) {
  constexpr int kThreads = cta_threads(G), kRows = kThreads / G, kResident = rows_resident(G, FULL, WIDE);
  const int stage = G * E * (type_bytes(p.a.x_type) + type_bytes(p.a.y_type)), room = kRowsSmem / kResident / kRows / stage;
  p.stages = room < 4 ? room : 4;
  const int64_t want = (p.rows + kRows - 1) / kRows, most = static_cast<int64_t>(sm_count()) * kResident;
  static std::atomic<uint64_t> ready{0};
  if (attributes_missing(ready)) {
    S3R_CUDA(cudaFuncSetAttribute(norm_rows_kernel<W, G, E, FULL, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem));
    attributes_set(ready);
  }
  return launch(norm_rows_kernel<W, G, E, FULL, WIDE>, static_cast<unsigned>(want < most ? want : most), kThreads,
                static_cast<size_t>(kRows) * p.stages * stage, st, p);
}
template <int W, int G, int E>
static int run_fwd(const NormParams& p, cudaStream_t st) {
  constexpr int kRows = cta_threads(G) / G, kThreads = cta_threads(G);
  // where every CTA that fits has four rows and more
  if constexpr (W > 1 && E == 8)
    if (p.rows >= 4 * kRows * sm_count() * rows_resident(G, false, false)) {
      if (p.a.post || p.a.gate_mode == S3R_GATE_CHANNEL) return run_rows<W, G, E, true, true>(p, st);
      return p.a.x_type == S3R_F32 ? run_rows<W, G, E, false, true>(p, st) : run_rows<W, G, E, false, false>(p, st);
    }
  return launch(norm_fwd_kernel<W, G, E>, static_cast<unsigned>((p.rows + kRows - 1) / kRows), kThreads, 0, st, p);
}
template <int W>
static int pick_fwd(const NormParams& p, cudaStream_t st) {
  const int C = p.a.channels;
  // Eight values per thread: with 32 (a warp per row, no exchange between warps) 64 512 x 1024 took 134 us instead of 130, 12 288 33
  // instead of 29.5.  As few threads as have them: rows of 512 by 128 threads 90 us (58 593 of them, fp32), by 64 60; 768 by 128 67, by 96 63;
  // 1536 by 256 74, by 192 63.
  if (C <= 256) return run_fwd<W, 32, 8>(p, st);
  if (C <= 512) return run_fwd<W, 64, 8>(p, st);
  if (C <= 768) return run_fwd<W, 96, 8>(p, st);
  if (C <= 1024) return run_fwd<W, 128, 8>(p, st);
  if (C <= 1536) return run_fwd<W, 192, 8>(p, st);
  if (C <= 2048) return run_fwd<W, 256, 8>(p, st);
  if (C <= 4096) return run_fwd<W, 512, 8>(p, st);
  return run_fwd<W, 512, 16>(p, st);
}

// As few warps as have a row, but for fp32 rows of whole warps, where three and six warps leave too few threads on an SM: 768 channels fp32 by
// 128 threads 101 us (39 062 rows), by 96 115, bf16 85 and 79; 1536 fp32 by 256 103, by 192 109, bf16 90 and 82; 700 fp32 124 and 110.
static void bwd_shape(int channels, bool whole, int* G, int* E) {
  *G = channels <= 256 ? 32 : channels <= 512 ? 64 : channels <= 768 && !whole ? 96 : channels <= 1024 ? 128 : channels <= 1536 && !whole ? 192 : channels <= 2048 ? 256 : 512;
  *E = channels <= 4096 ? 8 : 16;
}
// slices per batch entry (of `entries`): CTAs that are resident together and no more (3 x 1041 rows of 1540, a gate per channel: 150 of them on
// 148 SMs took 61 us, 147 take 35), each with two rows per group or more where there are as many
static int bwd_slices(int64_t entries, int64_t span, int G, bool full) {
  const int threads = cta_threads(G), groups = threads / G;
  const int64_t resident = static_cast<int64_t>(sm_count()) * bwd_resident(G, full);
  const int64_t want = resident / entries, most = (span + 4 * groups - 1) / (4 * groups);
  const int64_t n = want < most ? want : most;
  return static_cast<int>(n < 1 ? 1 : n);
}

template <int W, int G, int E, bool FULL>
static int run_bwd(const NormBwdParams& p, unsigned ctas, cudaStream_t st) {
  constexpr int kThreads = cta_threads(G), kGroups = kThreads / G;
  static_assert(kGroups * E * G * 4 <= kRowsSmem, "sums of the groups");
  static std::atomic<uint64_t> ready{0};
  if (attributes_missing(ready)) {
    S3R_CUDA(cudaFuncSetAttribute(norm_bwd_kernel<W, G, E, FULL>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem));
    attributes_set(ready);
  }
  size_t smem = W > 1 ? static_cast<size_t>(kGroups) * p.stages * p.stage_bytes : 0;
  if constexpr (kGroups > 1) {
    constexpr size_t kSumBytes = static_cast<size_t>(kGroups) * E * G * 4;
    if (smem < kSumBytes) smem = kSumBytes;
  }
  return launch(norm_bwd_kernel<W, G, E, FULL>, ctas, kThreads, smem, st, p);
}
template <int W, bool FULL>
static int pick_bwd(const NormBwdParams& p, int G, int E, unsigned ctas, cudaStream_t st) {
  if (G == 32) return run_bwd<W, 32, 8, FULL>(p, ctas, st);
  if (G == 64) return run_bwd<W, 64, 8, FULL>(p, ctas, st);
  if (G == 96) return run_bwd<W, 96, 8, FULL>(p, ctas, st);
  if (G == 128) return run_bwd<W, 128, 8, FULL>(p, ctas, st);
  if (G == 192) return run_bwd<W, 192, 8, FULL>(p, ctas, st);
  if (G == 256) return run_bwd<W, 256, 8, FULL>(p, ctas, st);
  if (E == 8) return run_bwd<W, 512, 8, FULL>(p, ctas, st);
  return run_bwd<W, 512, 16, FULL>(p, ctas, st);
}

}  // namespace s3r

using namespace s3r;

extern "C" int s3r_residual_norm_fwd(const s3r_residual_norm* args, void* stream) {
  S3R_REQUIRE(args && args->x, S3R_ERR_NULL, "s3r_residual_norm_fwd: NULL pointer");
  const s3r_residual_norm& a = *args;
  if (const int rc = check_args(a, "s3r_residual_norm_fwd")) return rc;
  S3R_REQUIRE(!a.y || a.r, S3R_ERR_NULL, "s3r_residual_norm_fwd: no place for the sum");
  S3R_REQUIRE(a.r || a.h || a.q, S3R_ERR_NULL, "s3r_residual_norm_fwd: nothing to compute");
  S3R_REQUIRE(!(a.h && a.q), S3R_ERR_UNSUPPORTED, "s3r_residual_norm_fwd: the norm's result in its own type or in 8 bits");
  S3R_REQUIRE(!a.q || (a.q_scale && a.q_pitch >= a.channels), S3R_ERR_SHAPE, "s3r_residual_norm_fwd: 8-bit rows need scales and a pitch");
  const void* ptr[] = {a.x, a.y, a.r, a.h, a.weight, a.bias, a.scale, a.post_weight, a.post_bias, a.gate_mode == S3R_GATE_CHANNEL ? a.gate : nullptr};
  const int type[] = {a.x_type, a.y_type, a.x_type, a.h_type, a.param_type, a.param_type, a.param_type, a.param_type, a.param_type, a.gate_type};
  int w = row_vector(a.channels, ptr, type, 10);
  if (w > gate_vector(a)) w = gate_vector(a);
  if (a.q && (reinterpret_cast<uintptr_t>(a.q) | a.q_pitch) % 4) w = 1;
  const NormParams p = {a, a.batch * a.tokens, 1.f / static_cast<float>(a.channels), 0};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return w == 8 ? pick_fwd<8>(p, st) : w == 4 ? pick_fwd<4>(p, st) : pick_fwd<1>(p, st);
}

extern "C" size_t s3r_residual_norm_bwd_workspace_bytes(int64_t batch, int64_t tokens, int channels, int gate_mode) {
  if (batch <= 0 || tokens <= 0 || channels <= 0 || channels > kNormMaxChannels || batch > (1ll << 31) / tokens) return 0;
  const int64_t entries = gate_mode == S3R_GATE_CHANNEL ? batch : 1, span = gate_mode == S3R_GATE_CHANNEL ? tokens : batch * tokens;
  int slices = 0;                                        // whatever x's type, with and without a post norm
  for (const bool whole : {false, true}) {
    int G, E;
    bwd_shape(channels, whole, &G, &E);
    slices = std::max(slices, bwd_slices(entries, span, G, false));          // not fewer than those of a full one
  }
  return static_cast<size_t>(entries) * slices * kSums * channels * sizeof(float);
}

extern "C" int s3r_residual_norm_bwd(const s3r_residual_norm* f_, const s3r_residual_norm_grad* g_, void* stream) {
  S3R_REQUIRE(f_ && g_, S3R_ERR_NULL, "s3r_residual_norm_bwd: NULL pointer");
  const s3r_residual_norm& f = *f_;
  const s3r_residual_norm_grad& g = *g_;
  if (const int rc = check_args(f, "s3r_residual_norm_bwd")) return rc;
  S3R_REQUIRE(g.dx && (g.dr || g.dh), S3R_ERR_NULL, "s3r_residual_norm_bwd: NULL pointer");
  S3R_REQUIRE(!g.dh || (f.r && f.stats), S3R_ERR_NULL, "s3r_residual_norm_bwd: the forward's sum and statistics are missing");
  S3R_REQUIRE(!f.post || f.stats, S3R_ERR_NULL, "s3r_residual_norm_bwd: the forward's statistics are missing");
  S3R_REQUIRE(f.y || (!g.dy && !g.d_scale && !g.d_gate_row && !g.d_gate_channel && !g.d_post_weight && !g.d_post_bias), S3R_ERR_NULL,
              "s3r_residual_norm_bwd: gradients of a branch that is not there");
  S3R_REQUIRE(g.dh || (!g.d_weight && !g.d_bias), S3R_ERR_NULL, "s3r_residual_norm_bwd: gradients of a norm without its output's");
  S3R_REQUIRE(f.post || (!g.d_post_weight && !g.d_post_bias), S3R_ERR_NULL, "s3r_residual_norm_bwd: gradients of a post norm that is not there");
  S3R_REQUIRE((!g.d_gate_row || f.gate_mode == S3R_GATE_ROW) && (!g.d_gate_channel || f.gate_mode == S3R_GATE_CHANNEL), S3R_ERR_UNSUPPORTED,
              "s3r_residual_norm_bwd: the gate's gradient in another form than the gate");
  const void* ptr[] = {f.r, f.y, g.dr, g.dh, g.dx, g.dy, f.weight, f.scale, f.post_weight, f.post_bias, f.gate_mode == S3R_GATE_CHANNEL ? f.gate : nullptr};
  const int type[] = {f.x_type, f.y_type, f.x_type, f.h_type, f.x_type, f.y_type, f.param_type, f.param_type, f.param_type, f.param_type, f.gate_type};
  for (int i = 0; i < 6; ++i)
    S3R_REQUIRE(reinterpret_cast<uintptr_t>(ptr[i]) % type_bytes(type[i]) == 0, S3R_ERR_ALIGNMENT, "s3r_residual_norm_bwd: elements must be aligned");
  int w = row_vector(f.channels, ptr, type, 11);
  if (w > gate_vector(f)) w = gate_vector(f);

  NormBwdParams p = {};
  p.f = f;
  p.g = g;
  p.rows = f.batch * f.tokens;
  const bool per_entry = f.gate_mode == S3R_GATE_CHANNEL;
  const int64_t entries = per_entry ? f.batch : 1;
  p.span = per_entry ? f.tokens : p.rows;
  int G, E;
  bwd_shape(f.channels, f.x_type == S3R_F32 && f.channels % 256 == 0, &G, &E);
  const bool full = f.post || per_entry;
  p.slices = bwd_slices(entries, p.span, G, full);
  void* const out[kSums] = {g.d_weight, g.d_bias, g.d_scale, g.d_post_weight, g.d_post_bias, g.d_gate_channel};
  for (int i = 0; i < kSums; ++i) p.place[i] = out[i] ? p.sums++ : 0;
  const bool sums = p.sums > 0;
  const size_t need = s3r_residual_norm_bwd_workspace_bytes(f.batch, f.tokens, f.channels, f.gate_mode) / kSums * p.sums;
  S3R_REQUIRE(!sums || (g.workspace && g.workspace_bytes >= need && reinterpret_cast<uintptr_t>(g.workspace) % 4 == 0), S3R_ERR_TOO_LARGE,
              "s3r_residual_norm_bwd: workspace of %zu bytes is smaller than the %zu needed", g.workspace ? g.workspace_bytes : 0, need);
  p.partial = static_cast<float*>(g.workspace);
  p.inv_n = 1.f / static_cast<float>(f.channels);
  const uint32_t row = static_cast<uint32_t>(G) * E;            // every thread has places, behind the end of a row too
  p.at_y = row * type_bytes(f.x_type);
  p.at_dr = p.at_y + row * type_bytes(f.y_type);
  p.at_dh = p.at_dr + row * type_bytes(f.x_type);
  p.stage_bytes = p.at_dh + row * type_bytes(f.h_type);
  const int threads = cta_threads(G), resident = bwd_resident(G, full);
  const uint32_t room = kRowsSmem / resident / (threads / G);
  p.stages = static_cast<int>(room / p.stage_bytes < 4 ? room / p.stage_bytes : 4);
  S3R_REQUIRE(p.stages >= 1, S3R_ERR_TOO_LARGE, "s3r_residual_norm_bwd: rows do not fit shared memory");

  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned ctas = static_cast<unsigned>(entries * p.slices);
  int rc;
  if (w == 8) rc = full ? pick_bwd<8, true>(p, G, E, ctas, st) : pick_bwd<8, false>(p, G, E, ctas, st);
  else if (w == 4) rc = full ? pick_bwd<4, true>(p, G, E, ctas, st) : pick_bwd<4, false>(p, G, E, ctas, st);
  else rc = full ? pick_bwd<1, true>(p, G, E, ctas, st) : pick_bwd<1, false>(p, G, E, ctas, st);
  if (rc || !sums) return rc;

  NormSumsParams s = {};
  s.partial = p.partial;
  s.channels = f.channels;
  s.slices = p.slices;
  s.entries = static_cast<int>(entries);
  s.type = f.param_type;
  s.gate_type = f.gate_type;
  s.sums = p.sums;
  for (int i = 0; i < kSumGate; ++i)
    if (out[i]) s.place[s.n] = p.place[i], s.out[s.n++] = out[i];
  s.place[s.n] = p.place[kSumGate];
  s.out[s.n] = g.d_gate_channel;
  const int64_t jobs = s.n + (g.d_gate_channel ? entries : 0), blocks = jobs * ((f.channels + 31) / 32);
  S3R_REQUIRE(blocks < (1ll << 31), S3R_ERR_TOO_LARGE, "s3r_residual_norm_bwd: grid too large");
  return launch(norm_sums_kernel, static_cast<unsigned>(blocks), 1024, 0, st, s);
}
