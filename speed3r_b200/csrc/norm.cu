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
__device__ __forceinline__ float2 row_statistics(const float (&v)[E], int kind, int channels, float inv_n, float eps, float* red, uint32_t& turn, int t) {
  float s[1] = {0.f};
  float mean = 0.f;
  if (kind == S3R_NORM_LAYER) {
#pragma unroll
    for (int k = 0; k < E; ++k) s[0] += v[k];            // places behind the row hold 0
    row_sum<G>(s, red, turn, t, 0);
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
  row_sum<G>(s, red, turn, t, 0);
  return make_float2(mean, rsqrtf(fmaf(s[0], inv_n, eps)));
}

template <int W, int G, int E>
__device__ __forceinline__ void apply_norm(float (&v)[E], float2 st, const void* weight, const void* bias, int type, int channels, int t) {
#pragma unroll
  for (int i = 0; i < E / W; ++i) {
    const int c = (i * G + t) * W;
    if (c < channels) {
      float w[W], b[W];
      if (weight) load_vector<W>(w, weight, type, c);
      if (bias) load_vector<W>(b, bias, type, c);
#pragma unroll
      for (int k = 0; k < W; ++k) {
        float x = (v[i * W + k] - st.x) * st.y;
        if (weight) x *= w[k];
        if (bias) x += b[k];
        v[i * W + k] = x;
      }
    }
  }
}

template <int W, int G, int E>
__global__ void __launch_bounds__(G < 128 ? 128 : G) norm_fwd_kernel(const __grid_constant__ NormParams p) {
  constexpr int kRows = G < 128 ? 128 / G : 1, N = E / W;
  __shared__ float red[G > 32 ? 8 * (G / 32) : 1];
  griddep_wait();
  griddep_launch();
  const s3r_residual_norm& a = p.a;
  const int t = threadIdx.x % G, C = a.channels;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / G;
  if (row >= p.rows) return;                              // whole rows leave (rows of several warps have a CTA each)
  const int64_t at = row * C;
  uint32_t turn = 0;
  Raw<W> xr[N], yr[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (i * G + t) * W;
    if (c < C) {
      load_raw<W>(xr[i], a.x, a.x_type, at + c);
      if (a.y) load_raw<W>(yr[i], a.y, a.y_type, at + c);
    }
  }
  float v[E];
  if (a.y) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float f[W];
      unpack<W>(f, yr[i], a.y_type);
#pragma unroll
      for (int k = 0; k < W; ++k) v[i * W + k] = (i * G + t) * W < C ? f[k] : 0.f;
    }
    if (a.post) {
      const float2 st = row_statistics<W, G, E>(v, a.kind, C, p.inv_n, a.post_eps, red, turn, t);
      if (a.stats && t == 0) a.stats[2 * p.rows + row] = st.x, a.stats[3 * p.rows + row] = st.y;
      apply_norm<W, G, E>(v, st, a.post_weight, a.post_bias, a.param_type, C, t);
    }
    const float gate = gate_of_row(a, row);
    const int64_t gate_at = a.gate_mode == S3R_GATE_CHANNEL ? row / a.tokens * a.gate_stride_b : 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * G + t) * W;
      if (c < C) {
        float f[W];
        if (a.scale) {
          load_vector<W>(f, a.scale, a.param_type, c);
#pragma unroll
          for (int k = 0; k < W; ++k) v[i * W + k] = __fmul_rn(v[i * W + k], f[k]);
        }
        if (a.gate_mode == S3R_GATE_CHANNEL) {
          load_vector<W>(f, a.gate, a.gate_type, gate_at + c);
#pragma unroll
          for (int k = 0; k < W; ++k) v[i * W + k] = __fmul_rn(v[i * W + k], f[k]);
        } else if (a.gate_mode == S3R_GATE_ROW) {
#pragma unroll
          for (int k = 0; k < W; ++k) v[i * W + k] = __fmul_rn(v[i * W + k], gate);
        }
        unpack<W>(f, xr[i], a.x_type);
#pragma unroll
        for (int k = 0; k < W; ++k) f[k] = __fadd_rn(f[k], v[i * W + k]);
        // the norm is that of the stored sum, as it is for whoever reads it later, the backward among them
        Raw<W> o;
        pack<W>(o, f, a.x_type);
        store_raw<W>(o, a.r, a.x_type, at + c);
        unpack<W>(f, o, a.x_type);
#pragma unroll
        for (int k = 0; k < W; ++k) v[i * W + k] = f[k];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * G + t) * W;
      float f[W];
      unpack<W>(f, xr[i], a.x_type);
#pragma unroll
      for (int k = 0; k < W; ++k) v[i * W + k] = c < C ? f[k] : 0.f;
      if (a.r && c < C) store_raw<W>(xr[i], a.r, a.x_type, at + c);
    }
  }
  if (!a.h && !a.q) return;
  const float2 st = row_statistics<W, G, E>(v, a.kind, C, p.inv_n, a.eps, red, turn, t);
  if (a.stats && t == 0) a.stats[row] = st.x, a.stats[p.rows + row] = st.y;
  apply_norm<W, G, E>(v, st, a.weight, a.bias, a.param_type, C, t);
  if (a.h) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * G + t) * W;
      if (c < C) {
        float f[W];
#pragma unroll
        for (int k = 0; k < W; ++k) f[k] = v[i * W + k];
        Raw<W> o;
        pack<W>(o, f, a.h_type);
        store_raw<W>(o, a.h, a.h_type, at + c);
      }
    }
    return;
  }
  float big = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if ((i * G + t) * W < C)
#pragma unroll
      for (int k = 0; k < W; ++k) big = max_nan(big, fabsf(v[i * W + k]));
  big = row_max<G>(big, red, turn, t, 0);
  const RowScale s = row_scale(big);
  if (t == 0) a.q_scale[row] = s.scale;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (i * G + t) * W;
    if (c < C) {
      int8_t* q = a.q + row * a.q_pitch + c;
      if constexpr (W == 1) {
        *q = static_cast<int8_t>(to_s8(v[i], s.inverse));
      } else {
#pragma unroll
        for (int k = 0; k < W; k += 4)
          *reinterpret_cast<uint32_t*>(q + k) = to_s8(v[i * W + k], s.inverse) | to_s8(v[i * W + k + 1], s.inverse) << 8 |
                                                to_s8(v[i * W + k + 2], s.inverse) << 16 | to_s8(v[i * W + k + 3], s.inverse) << 24;
      }
    }
  }
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
  float* partial;              // [batch entries x slices, kSums, channels], the sums that are wanted
};

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
__device__ __forceinline__ void staged(float (&f)[W], const char* s, int type) {
  Raw<W> r;
  const uint32_t* q = reinterpret_cast<const uint32_t*>(s);
  if (type == S3R_F32) {
#pragma unroll
    for (int k = 0; k < W; k += 4) {
      const uint4 u = *reinterpret_cast<const uint4*>(q + k);
      r.v[k] = u.x, r.v[k + 1] = u.y, r.v[k + 2] = u.z, r.v[k + 3] = u.w;
    }
  } else if constexpr (W == 8) {
    const uint4 u = *reinterpret_cast<const uint4*>(q);
    r.v[0] = u.x, r.v[1] = u.y, r.v[2] = u.z, r.v[3] = u.w;
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(q);
    r.v[0] = u.x, r.v[1] = u.y;
  }
  unpack<W>(f, r, type);
}

__device__ __forceinline__ void cp_async_wait_for(int pending) {
  if (pending >= 3) cp_async_wait<3>();
  else if (pending == 2) cp_async_wait<2>();
  else if (pending == 1) cp_async_wait<1>();
  else cp_async_wait<0>();
}

constexpr int kNormSmem = 220 * 1024;

// FULL: a post norm or a gate per channel too; without them their sums and factors take no registers
template <int W, int G, int E, bool FULL>
__global__ void __launch_bounds__(G < 128 ? 128 : G) norm_bwd_kernel(const __grid_constant__ NormBwdParams p) {
  constexpr int kRows = G < 128 ? 128 / G : 1, N = E / W;
  extern __shared__ __align__(16) char smem[];
  __shared__ float red[kRows][G > 32 ? 8 * (G / 32) : 1];
  griddep_wait();
  griddep_launch();
  const s3r_residual_norm& f = p.f;
  const s3r_residual_norm_grad& g = p.g;
  const int t = threadIdx.x % G, group = threadIdx.x / G, C = f.channels;
  const int entry = blockIdx.x / p.slices, slice = blockIdx.x % p.slices;
  const int64_t first = entry * p.span + p.span * slice / p.slices, last = entry * p.span + p.span * (slice + 1) / p.slices;
  const bool layer = f.kind == S3R_NORM_LAYER, branch = f.y != nullptr;
  const bool norm = g.dh != nullptr;
  char* ring = smem + static_cast<size_t>(group) * p.stages * p.stage_bytes;
  uint32_t turn = 0;

  float w[E], scale[E], gate_c[FULL ? E : 1], pw[FULL ? E : 1], pb[FULL ? E : 1];
  float d_w[E], d_b[E], d_s[E], d_g[FULL ? E : 1], d_pw[FULL ? E : 1], d_pb[FULL ? E : 1];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (i * G + t) * W;
    float one[W], zero[W];
#pragma unroll
    for (int k = 0; k < W; ++k) one[k] = 1.f, zero[k] = 0.f;
    auto fetch = [&](float* to, const void* from, int type, int64_t at, const float* other) {
      float v[W];
      if (from && c < C) load_vector<W>(v, from, type, at + c);
#pragma unroll
      for (int k = 0; k < W; ++k) to[i * W + k] = from && c < C ? v[k] : other[k];
    };
    fetch(w, f.weight, f.param_type, 0, one);
    fetch(scale, f.scale, f.param_type, 0, one);
    if constexpr (FULL) {
      fetch(gate_c, f.gate_mode == S3R_GATE_CHANNEL ? f.gate : nullptr, f.gate_type, entry * f.gate_stride_b, one);
      fetch(pw, f.post_weight, f.param_type, 0, one);
      fetch(pb, f.post_bias, f.param_type, 0, zero);
    }
  }
#pragma unroll
  for (int k = 0; k < E; ++k) {
    d_w[k] = d_b[k] = d_s[k] = 0.f;
    if constexpr (FULL) d_g[k] = d_pw[k] = d_pb[k] = 0.f;
  }

  const bool reads_r = norm, reads_y = branch && (f.post || g.d_scale || g.d_gate_row || g.d_gate_channel);
  auto request = [&](int64_t row, int stage) {
    if constexpr (W > 1) {
      if (row < last) {
        const uint32_t to = smem_u32(ring) + stage * p.stage_bytes;
        const int64_t at = row * C;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int c = (i * G + t) * W;
          if (c < C) {
            if (reads_r) stage_vector<W>(to + c * type_bytes(f.x_type), f.r, f.x_type, at + c);
            if (reads_y) stage_vector<W>(to + p.at_y + c * type_bytes(f.y_type), f.y, f.y_type, at + c);
            if (g.dr) stage_vector<W>(to + p.at_dr + c * type_bytes(f.x_type), g.dr, f.x_type, at + c);
            if (g.dh) stage_vector<W>(to + p.at_dh + c * type_bytes(f.h_type), g.dh, f.h_type, at + c);
          }
        }
      }
      cp_async_commit();
    }
  };
  // a vector of the present row: where it was staged, or from memory (rows of odd width)
  auto fetch = [&](float (&v)[W], const char* stage, uint32_t at, const void* from, int type, int64_t row, int c) {
    if constexpr (W > 1) staged<W>(v, stage + at + c * type_bytes(type), type);
    else load_vector<W>(v, from, type, row * C + c);
  };

  int stage = 0;
  for (int s = 0; s + 1 < p.stages; ++s) request(first + group + static_cast<int64_t>(s) * kRows, s);
  for (int64_t row = first + group; row < last; row += kRows) {
    request(row + static_cast<int64_t>(p.stages - 1) * kRows, stage + p.stages - 1 >= p.stages ? stage - 1 : p.stages - 1);
    float mean = 0.f, inv = 0.f, p_mean = 0.f, p_inv = 0.f;
    if (norm) mean = __ldg(f.stats + row), inv = __ldg(f.stats + p.rows + row);
    if (FULL && f.post) p_mean = __ldg(f.stats + 2 * p.rows + row), p_inv = __ldg(f.stats + 3 * p.rows + row);
    const float gate = gate_of_row(f, row);
    if constexpr (W > 1) cp_async_wait_for(p.stages - 1);
    const char* here = ring + stage * p.stage_bytes;
    stage = stage + 1 == p.stages ? 0 : stage + 1;

    float xh[E], d[E], s[3] = {0.f, 0.f, 0.f};
    if (norm) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = (i * G + t) * W;
        float a[W], b[W];
        if (c < C) {
          fetch(a, here, 0, f.r, f.x_type, row, c);
          fetch(b, here, p.at_dh, g.dh, f.h_type, row, c);
        }
#pragma unroll
        for (int k = 0; k < W; ++k) {
          const int e = i * W + k;
          xh[e] = c < C ? (a[k] - mean) * inv : 0.f;
          const float dh = c < C ? b[k] : 0.f;
          d_w[e] = fmaf(dh, xh[e], d_w[e]);
          d_b[e] += dh;
          d[e] = dh * w[e];
          s[0] += d[e];
          s[1] = fmaf(d[e], xh[e], s[1]);
        }
      }
      float both[2] = {s[0], s[1]};
      row_sum<G>(both, red[group], turn, t, group + 1);
      const float along = both[1] * p.inv_n, flat = layer ? both[0] * p.inv_n : 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) d[e] = inv * (d[e] - flat - xh[e] * along);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) d[e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * G + t) * W;
      if (c < C) {
        float a[W];
        if (g.dr) {
          fetch(a, here, p.at_dr, g.dr, f.x_type, row, c);
#pragma unroll
          for (int k = 0; k < W; ++k) d[i * W + k] += a[k];
        }
#pragma unroll
        for (int k = 0; k < W; ++k) a[k] = d[i * W + k];
        Raw<W> o;
        pack<W>(o, a, f.x_type);
        store_raw<W>(o, g.dx, f.x_type, row * C + c);
      } else {
#pragma unroll
        for (int k = 0; k < W; ++k) d[i * W + k] = 0.f;
      }
    }
    if (!branch) continue;
    float gate_sum = 0.f;
    s[0] = s[1] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (i * G + t) * W;
      float y[W];
#pragma unroll
      for (int k = 0; k < W; ++k) y[k] = 0.f;
      if (reads_y && c < C) fetch(y, here, p.at_y, f.y, f.y_type, row, c);
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const int e = i * W + k;
        float u = y[k];
        if constexpr (FULL) {
          if (f.post) {
            xh[e] = c < C ? (y[k] - p_mean) * p_inv : 0.f;
            u = fmaf(xh[e], pw[e], pb[e]);
          }
        }
        const float of_scale = FULL ? d[e] * gate * gate_c[e] : d[e] * gate;
        d_s[e] = fmaf(of_scale, u, d_s[e]);
        const float of_gate = d[e] * scale[e] * u;
        gate_sum += of_gate;
        if constexpr (FULL) d_g[e] += of_gate;
        const float du = of_scale * scale[e];
        if constexpr (FULL) {
          if (f.post) {
            d_pw[e] = fmaf(du, xh[e], d_pw[e]);
            d_pb[e] += du;
            d[e] = du * pw[e];
            s[0] += d[e];
            s[1] = fmaf(d[e], xh[e], s[1]);
          } else {
            d[e] = du;
          }
        } else {
          d[e] = du;
        }
      }
    }
    const bool through = FULL && f.post;
    if (through || g.d_gate_row) {
      s[2] = gate_sum;
      row_sum<G>(s, red[group], turn, t, group + 1);
      if (g.d_gate_row && t == 0) g.d_gate_row[row] = s[2];
      if (through) {
        const float along = s[1] * p.inv_n, flat = layer ? s[0] * p.inv_n : 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) d[e] = p_inv * (d[e] - flat - xh[e] * along);
      }
    }
    if (g.dy) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = (i * G + t) * W;
        if (c < C) {
          float a[W];
#pragma unroll
          for (int k = 0; k < W; ++k) a[k] = d[i * W + k];
          Raw<W> o;
          pack<W>(o, a, f.y_type);
          store_raw<W>(o, g.dy, f.y_type, row * C + c);
        }
      }
    }
  }

  // this CTA's sums over rows; groups of one CTA are added in order
  float* out = p.partial + static_cast<int64_t>(blockIdx.x) * kSums * C;
  auto leave = [&](const float* sums, int which, bool wanted) {
    if (!wanted) return;
    if constexpr (kRows > 1) {
      __syncthreads();                                  // the ring, or the sums before these
      float* shared = reinterpret_cast<float*>(smem);
#pragma unroll
      for (int e = 0; e < E; ++e) shared[(group * E + e) * G + t] = sums[e];
      __syncthreads();
      if (group) return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const int e = i * W + k, c = (i * G + t) * W + k;
        float s = sums[e];
        if constexpr (kRows > 1) {
          const float* shared = reinterpret_cast<const float*>(smem);
#pragma unroll
          for (int o = 1; o < kRows; ++o) s += shared[(o * E + e) * G + t];
        }
        if (c < C) out[static_cast<int64_t>(which) * C + c] = s;
      }
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
  int which[kSums + 1];
  int type, gate_type;
};

// sums of the CTAs' sums: 32 columns per CTA, its 8 warps take turns at the slices
__global__ void __launch_bounds__(256) norm_sums_kernel(const __grid_constant__ NormSumsParams p) {
  __shared__ float red[8][32];
  griddep_wait();
  griddep_launch();
  const int columns = (p.channels + 31) / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t job = blockIdx.x / columns;
  const int c = static_cast<int>(blockIdx.x % columns) * 32 + lane;
  const bool gate = job >= p.n;
  const int which = gate ? kSumGate : p.which[job];
  const int64_t entry = gate ? job - p.n : 0;
  const int64_t first = gate ? entry * p.slices : 0, last = gate ? first + p.slices : static_cast<int64_t>(p.entries) * p.slices;
  float s = 0.f;
  if (c < p.channels)
#pragma unroll 4
    for (int64_t i = first + warp; i < last; i += 8) s += __ldg(p.partial + (i * kSums + which) * p.channels + c);
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < p.channels) {
#pragma unroll
    for (int w = 1; w < 8; ++w) s += red[w][lane];
    const float f[1] = {s};
    Raw<1> o;
    pack<1>(o, f, gate ? p.gate_type : p.type);
    store_raw<1>(o, p.out[gate ? p.n : job], gate ? p.gate_type : p.type, gate ? entry * p.channels + c : c);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------------
static int check_args(const s3r_residual_norm& a, const char* what) {
  S3R_REQUIRE(a.batch > 0 && a.tokens > 0 && a.channels > 0, S3R_ERR_SHAPE, "%s: sizes must be positive", what);
  S3R_REQUIRE(a.channels <= kNormMaxChannels, S3R_ERR_TOO_LARGE, "%s: %d channels (at most %d)", what, a.channels, kNormMaxChannels);
  S3R_REQUIRE(a.batch < (1ll << 31) && a.tokens < (1ll << 31) && a.batch * a.tokens < (1ll << 31), S3R_ERR_TOO_LARGE, "%s: too many rows", what);
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

template <int W, int G, int E>
static int run_fwd(const NormParams& p, cudaStream_t st) {
  constexpr int kRows = G < 128 ? 128 / G : 1;
  return launch(norm_fwd_kernel<W, G, E>, static_cast<unsigned>((p.rows + kRows - 1) / kRows), G < 128 ? 128 : G, 0, st, p);
}
template <int W>
static int pick_fwd(const NormParams& p, cudaStream_t st) {
  const int C = p.a.channels;
  if (C <= 256) return run_fwd<W, 32, 8>(p, st);
  if (C <= 1024 && p.rows <= 2 * sm_count()) return run_fwd<W, 128, 8>(p, st);
  if (C <= 512) return run_fwd<W, 32, 16>(p, st);
  if (C <= 1024) return run_fwd<W, 32, 32>(p, st);
  if (C <= 2048) return run_fwd<W, 128, 16>(p, st);
  if (C <= 4096) return run_fwd<W, 128, 32>(p, st);
  return run_fwd<W, 256, 32>(p, st);
}

struct BwdShape {
  int threads_per_row, per_thread, ctas, stages;
  uint32_t stage_bytes;
};
static void bwd_shape(int channels, int* G, int* E) {
  *G = channels <= 256 ? 32 : channels <= 512 ? 64 : channels <= 1024 ? 128 : channels <= 2048 ? 256 : 512;
  *E = channels <= 4096 ? 8 : 16;
}
// slices per batch entry (of `entries`): CTAs that are resident together, each with four rows per group at least
static int bwd_slices(int64_t entries, int64_t span, int G) {
  const int threads = G < 128 ? 128 : G, groups = threads / G;
  const int64_t resident = static_cast<int64_t>(sm_count()) * (512 / threads > 0 ? 512 / threads : 1);
  const int64_t want = (resident + entries - 1) / entries, most = (span + 4 * groups - 1) / (4 * groups);
  const int64_t n = want < most ? want : most;
  return static_cast<int>(n < 1 ? 1 : n);
}

template <int W, int G, int E, bool FULL>
static int run_bwd(const NormBwdParams& p, unsigned ctas, cudaStream_t st) {
  constexpr int kThreads = G < 128 ? 128 : G, kGroups = kThreads / G;
  static_assert(kGroups * E * G * 4 <= kNormSmem, "sums of the groups");
  S3R_CUDA(cudaFuncSetAttribute(norm_bwd_kernel<W, G, E, FULL>, cudaFuncAttributeMaxDynamicSharedMemorySize, kNormSmem));
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
  if (G == 128) return run_bwd<W, 128, 8, FULL>(p, ctas, st);
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
  const NormParams p = {a, a.batch * a.tokens, 1.f / static_cast<float>(a.channels)};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return w == 8 ? pick_fwd<8>(p, st) : w == 4 ? pick_fwd<4>(p, st) : pick_fwd<1>(p, st);
}

extern "C" size_t s3r_residual_norm_bwd_workspace_bytes(int64_t batch, int64_t tokens, int channels, int gate_mode) {
  if (batch <= 0 || tokens <= 0 || channels <= 0 || channels > kNormMaxChannels || batch > (1ll << 31) / tokens) return 0;
  int G, E;
  bwd_shape(channels, &G, &E);
  const int64_t entries = gate_mode == S3R_GATE_CHANNEL ? batch : 1, span = gate_mode == S3R_GATE_CHANNEL ? tokens : batch * tokens;
  return static_cast<size_t>(entries) * bwd_slices(entries, span, G) * kSums * channels * sizeof(float);
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
  bwd_shape(f.channels, &G, &E);
  p.slices = bwd_slices(entries, p.span, G);
  const bool sums = g.d_weight || g.d_bias || g.d_scale || g.d_post_weight || g.d_post_bias || g.d_gate_channel;
  const size_t need = s3r_residual_norm_bwd_workspace_bytes(f.batch, f.tokens, f.channels, f.gate_mode);
  S3R_REQUIRE(!sums || (g.workspace && g.workspace_bytes >= need && reinterpret_cast<uintptr_t>(g.workspace) % 4 == 0), S3R_ERR_TOO_LARGE,
              "s3r_residual_norm_bwd: workspace of %zu bytes is smaller than the %zu needed", g.workspace ? g.workspace_bytes : 0, need);
  p.partial = static_cast<float*>(g.workspace);
  p.inv_n = 1.f / static_cast<float>(f.channels);
  const uint32_t row = (static_cast<uint32_t>(f.channels) + 7) / 8 * 8;
  p.at_y = row * type_bytes(f.x_type);
  p.at_dr = p.at_y + row * type_bytes(f.y_type);
  p.at_dh = p.at_dr + row * type_bytes(f.x_type);
  p.stage_bytes = p.at_dh + row * type_bytes(f.h_type);
  const int threads = G < 128 ? 128 : G, resident = 512 / threads;
  const uint32_t room = kNormSmem / resident / (threads / G);
  p.stages = static_cast<int>(room / p.stage_bytes < 4 ? room / p.stage_bytes : 4);
  S3R_REQUIRE(p.stages >= 1, S3R_ERR_TOO_LARGE, "s3r_residual_norm_bwd: rows do not fit shared memory");

  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned ctas = static_cast<unsigned>(entries * p.slices);
  const bool full = f.post || per_entry;
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
  void* out[] = {g.d_weight, g.d_bias, g.d_scale, g.d_post_weight, g.d_post_bias};
  for (int i = 0; i < 5; ++i)
    if (out[i]) s.which[s.n] = i, s.out[s.n++] = out[i];
  s.out[s.n] = g.d_gate_channel;
  const int64_t jobs = s.n + (g.d_gate_channel ? entries : 0), blocks = jobs * ((f.channels + 31) / 32);
  S3R_REQUIRE(blocks < (1ll << 31), S3R_ERR_TOO_LARGE, "s3r_residual_norm_bwd: grid too large");
  return launch(norm_sums_kernel, static_cast<unsigned>(blocks), 256, 0, st, s);
}
