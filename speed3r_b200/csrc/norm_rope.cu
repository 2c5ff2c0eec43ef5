// The packed projection [batch, tokens, heads of q, k and v] as q, k and v [batch, heads, tokens, head_dim]: every head of q and k normalised
// (LayerNorm or by the root of its mean square) and turned by the rotary embedding, in one pass, and the gradient of that.
// Bound: HBM, every element is read once and written once (backward: x and its gradient read, one gradient written).
//
// A head's columns are pairs (i, i + pairs) that rotation turns, so a thread takes both members: V columns of the first kind and the V columns
// `pairs` further, two vectors, and needs nobody else's for the rotation.  G threads share a head; sums over it are log2 G shuffles.
// Columns that are not turned are taken as two neighbouring vectors.  A group of G threads stays with one token and walks over heads, so that the
// token's sines and cosines, the parameters and the sums over rows stay in registers; the groups of a warp have neighbouring tokens, whose
// results lie one behind the other.
// Memory is read and written by whole rows: the heads of a warp's tokens come by cp.async, neighbouring lanes neighbouring chunks, four heads
// ahead, and results leave the same way through shared memory.
//
// 64 512 tokens of 16 heads of 64 in bf16, LayerNorm with weight and bias, two axes: forward 133 us (793 MB, 6.0 TB/s; a copy by the same route 123);
// backward 216 us (1.19 GB read and written with the gradients of q, k and v, 5.5 TB/s; the rest is latency, at 16 warps per SM).
// Tried there, and slower: a thread's own vectors, pieces of 32 bytes, by cp.async 150 to 156 (where these took 139), and in registers four heads ahead
// 173; vectors of eight elements 153; a CTA that walks over q, k and v 155 to 191; three heads ahead 141, eight 143; backward two heads ahead 271 for 252.
#include <type_traits>

#include "rows.cuh"

namespace s3r {

struct NrParams {
  const void *qkv, *cos, *sin;
  const int64_t* pos;
  const void *weight[2], *bias[2];     // of q and k
  void* out[3];                        // q, k, v
  const void* d_out[3];                // backward: their gradients
  int64_t d_strides[3][3];
  void* d_qkv;
  float* sums;                         // [head chunks of q, then of k][CTAs of a chunk][weight, bias][head_dim]
  int64_t stride_b, stride_t, pos_stride_b, pos_stride_t, cos_pitch, sin_pitch, rows_of_tokens;
  uint32_t tokens;
  int heads, kv_heads, head_dim, kind, type, param_type, table_type, axes, pairs, rows;
  int normed[2];
  float eps[2], inverse_dim;
  int per_chunk, q_chunks, kv_chunks;
  uint32_t* status;
};

// A vector of V elements of 16 or 32 bits, as it lies in memory.
template <int V, int BYTES>
struct Vec {
  static constexpr int kWords = V * BYTES / 4 < 1 ? 1 : V * BYTES / 4;
  uint32_t w[kWords];
};
template <int V, int BYTES>
__device__ __forceinline__ void take_vec(Vec<V, BYTES>& v, uint32_t at) {
  if constexpr (V * BYTES == 2) {
    uint16_t h;
    asm volatile("ld.shared.b16 %0, [%1];" : "=h"(h) : "r"(at) : "memory");
    v.w[0] = h;
  } else if constexpr (V * BYTES == 4) {
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v.w[0]) : "r"(at) : "memory");
  } else if constexpr (V * BYTES == 8) {
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.w[0]), "=r"(v.w[1]) : "r"(at) : "memory");
  } else {
#pragma unroll
    for (int k = 0; k < V * BYTES / 16; ++k) {
      const uint4 u = lds128(at + 16 * k);
      v.w[4 * k] = u.x, v.w[4 * k + 1] = u.y, v.w[4 * k + 2] = u.z, v.w[4 * k + 3] = u.w;
    }
  }
}
template <int V, int BYTES>
__device__ __forceinline__ void put_vec(const Vec<V, BYTES>& v, uint32_t at) {
  if constexpr (V * BYTES == 2) asm volatile("st.shared.b16 [%0], %1;" ::"r"(at), "h"(static_cast<uint16_t>(v.w[0])) : "memory");
  else if constexpr (V * BYTES == 4) sts32(at, v.w[0]);
  else if constexpr (V * BYTES == 8) sts64(at, v.w[0], v.w[1]);
  else
#pragma unroll
    for (int k = 0; k < V * BYTES / 16; ++k) sts128(at + 16 * k, v.w[4 * k], v.w[4 * k + 1], v.w[4 * k + 2], v.w[4 * k + 3]);
}

constexpr int kNrThreads = 128, kNrWarps = kNrThreads / 32;

// One head of a warp's tokens: rows of a constant pitch, 16 bytes longer than the longest, so that rows begin in different banks.
// CB: bytes that a lane copies at a time; chunk n of a lane is number 32 n + lane, row by row.
template <int V, int G, int E, int BYTES, int CB, int INPUTS>
struct Tile {
  static constexpr int kZeros = V * BYTES < 16 ? 16 : V * BYTES;       // behind the tiles: what lanes without columns read
  static constexpr int kRows = 32 / G, kPitch = 2 * V * G * E * BYTES + 16, kBytes = kRows * kPitch;
  static constexpr int kChunks = (kRows * (kPitch - 16) + 32 * CB - 1) / (32 * CB);
  static constexpr int kAhead = 4, kSmem = kNrWarps * kBytes * (kAhead * INPUTS + 1) + kZeros;
  struct Chunk {
    int row, byte;           // byte: in the row
    uint32_t at;             // in the tile
    bool in;
  };
  static __device__ __forceinline__ Chunk chunk(int n, int lane, int row_bytes) {
    const int per = row_bytes / CB, i = 32 * n + lane, row = i / per, byte = (i - row * per) * CB;
    return {row, byte, static_cast<uint32_t>(row * kPitch + byte), row < kRows};
  }
  static __device__ __forceinline__ void ask(uint32_t to, const char* from) {
    if constexpr (CB == 16) {
      cp_async16(to, from);
    } else if constexpr (CB == 8) {
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
    } else if constexpr (CB == 4) {
      cp_async4(to, from);
    } else {
      asm volatile("st.shared.b16 [%0], %1;" ::"r"(to), "h"(__ldg(reinterpret_cast<const uint16_t*>(from))) : "memory");
    }
  }
  static __device__ __forceinline__ void leave(char* to, uint32_t from) {
    Vec<CB / 2, 2> v;
    take_vec<CB / 2, 2>(v, from);
    if constexpr (CB == 16) *reinterpret_cast<uint4*>(to) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
    else if constexpr (CB == 8) *reinterpret_cast<uint2*>(to) = make_uint2(v.w[0], v.w[1]);
    else if constexpr (CB == 4) *reinterpret_cast<uint32_t*>(to) = v.w[0];
    else *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(v.w[0]);
  }
};

// Where a thread's E slots lie: columns c0 .. c0 + V and c1 .. c1 + V, the axis that turns them (-1: none), column of the tables.
struct Slot {
  int c0, c1, axis, column;
};
template <int V>
__device__ __forceinline__ Slot slot_of(int s, const NrParams& p) {
  const int per = p.axes ? p.pairs / V : 1, turned = p.axes * per;
  if (s < turned) {
    const int a = s / per, j = (s - a * per) * V;
    return {2 * p.pairs * a + j, 2 * p.pairs * a + p.pairs + j, a, j};
  }
  const int c = 2 * p.pairs * p.axes + (s - turned) * 2 * V;
  return {c, c + V, -1, 0};
}

template <int G, int N>
__device__ __forceinline__ void group_sum(float (&s)[N]) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) s[k] += __shfl_xor_sync(0xffffffffu, s[k], o);
}

// Values of a slot in packed pairs: H of the first member, H of the second; V = 1: the two members are the one pair.
template <int V>
constexpr int kHalf = V == 1 ? 1 : V / 2;
template <int V>
constexpr int kSides = V == 1 ? 1 : 2;
template <int BYTES>
__device__ __forceinline__ float one_value(uint32_t w, int type) {
  return BYTES == 4 ? __uint_as_float(w) : type == S3R_BF16 ? bf16_lo(w) : half_lo(w);
}
template <int V, int BYTES>
__device__ __forceinline__ void take_slot(float2 (&x)[kSides<V>][kHalf<V>], uint32_t at0, uint32_t at1, int type) {
  Vec<V, BYTES> v[2];
  take_vec<V, BYTES>(v[0], at0);
  take_vec<V, BYTES>(v[1], at1);
  if constexpr (V == 1) {
    x[0][0] = make_float2(one_value<BYTES>(v[0].w[0], type), one_value<BYTES>(v[1].w[0], type));
  } else {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int k = 0; k < V / 2; ++k) {
        if constexpr (BYTES == 4) x[m][k] = make_float2(__uint_as_float(v[m].w[2 * k]), __uint_as_float(v[m].w[2 * k + 1]));
        else x[m][k] = type == S3R_BF16 ? make_float2(bf16_lo(v[m].w[k]), bf16_hi(v[m].w[k])) : make_float2(half_lo(v[m].w[k]), half_hi(v[m].w[k]));
      }
  }
}
template <int V, int BYTES>
__device__ __forceinline__ void put_slot(const float2 (&x)[kSides<V>][kHalf<V>], uint32_t at0, uint32_t at1, int type) {
  Vec<V, BYTES> v[2];
  if constexpr (V == 1) {
    if constexpr (BYTES == 4) {
      v[0].w[0] = __float_as_uint(x[0][0].x), v[1].w[0] = __float_as_uint(x[0][0].y);
    } else {
      const uint32_t w = type == S3R_BF16 ? pack_bf16(x[0][0].x, x[0][0].y) : pack_half(x[0][0].x, x[0][0].y);
      v[0].w[0] = w & 0xffffu, v[1].w[0] = w >> 16;
    }
  } else {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int k = 0; k < V / 2; ++k) {
        if constexpr (BYTES == 4) v[m].w[2 * k] = __float_as_uint(x[m][k].x), v[m].w[2 * k + 1] = __float_as_uint(x[m][k].y);
        else v[m].w[k] = type == S3R_BF16 ? pack_bf16(x[m][k].x, x[m][k].y) : pack_half(x[m][k].x, x[m][k].y);
      }
  }
  put_vec<V, BYTES>(v[0], at0);
  put_vec<V, BYTES>(v[1], at1);
}
__device__ __forceinline__ float2 twice(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 minus(float2 v) { return make_float2(-v.x, -v.y); }
// What a quarter turn makes of a slot, (a, b) -> (-b, a), and with `back` of its gradient, (a, b) -> (b, -a)
template <int V>
__device__ __forceinline__ float2 quarter(const float2 (&x)[kSides<V>][kHalf<V>], int m, int k, bool back) {
  if constexpr (V == 1) return back ? make_float2(x[0][0].y, -x[0][0].x) : make_float2(-x[0][0].y, x[0][0].x);
  else return (m == 0) != back ? minus(x[1 - m][k]) : x[1 - m][k];
}

// What a thread keeps of its columns, in the order of values(): member m of slot e in [e][m]
template <int V, int E>
struct Lane {
  Slot slot[E];
  bool on[E];
  float share[E];        // -1 / head_dim, 0 for columns that are not there, which stay 0 when the mean is taken off
};
template <int V, int G, int E>
__device__ __forceinline__ void place(Lane<V, E>& l, const NrParams& p, int t) {
#pragma unroll
  for (int e = 0; e < E; ++e) {
    l.slot[e] = slot_of<V>(t + e * G, p);
    l.on[e] = (t + e * G) * 2 * V < p.head_dim;
    l.share[e] = l.on[e] ? -p.inverse_dim : 0.f;
  }
}
// columns of the two values of pair [m][k] of a slot
template <int V>
__device__ __forceinline__ int column_x(const Slot& s, int m, int k) { return (m ? s.c1 : s.c0) + 2 * k; }
template <int V>
__device__ __forceinline__ int column_y(const Slot& s, int m, int k) { return V == 1 ? s.c1 : column_x<V>(s, m, k) + 1; }
template <int V, int E>
__device__ __forceinline__ void parameter(float2 (&f)[E][kSides<V>][kHalf<V>], const Lane<V, E>& l, const void* from, int type, float other) {
  uint32_t raw[E][kSides<V>][kHalf<V>][2];
  with_width(type, [&](auto width) {
    const auto* at = static_cast<const decltype(width)*>(from);
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int m = 0; m < kSides<V>; ++m)
#pragma unroll
        for (int k = 0; k < kHalf<V>; ++k) {
          raw[e][m][k][0] = from && l.on[e] ? __ldg(at + column_x<V>(l.slot[e], m, k)) : 0;
          raw[e][m][k][1] = from && l.on[e] ? __ldg(at + column_y<V>(l.slot[e], m, k)) : 0;
        }
  });
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int m = 0; m < kSides<V>; ++m)
#pragma unroll
      for (int k = 0; k < kHalf<V>; ++k)
        f[e][m][k] = from && l.on[e] ? make_float2(any_value(raw[e][m][k][0], type), any_value(raw[e][m][k][1], type)) : make_float2(other, other);
}
template <int V, int E>
__device__ __forceinline__ void angles(float2 (&c)[E][kHalf<V>], float2 (&s)[E][kHalf<V>], const Lane<V, E>& l, const NrParams& p, int64_t b, int t, bool in) {
  constexpr int N = V == 1 ? 1 : 2;                                // values of a pair that differ
  int64_t row[E];
  bool turned[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    turned[e] = in && l.on[e] && l.slot[e].axis >= 0;
    row[e] = turned[e] ? __ldg(p.pos + b * p.pos_stride_b + t * p.pos_stride_t + l.slot[e].axis) : 0;
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (row[e] < 0 || row[e] >= p.rows) {
      if (turned[e]) atomicOr(p.status, kStatusBadIndex);
      row[e] = row[e] < 0 ? 0 : p.rows - 1;
    }
  uint32_t cr[E][kHalf<V>][N], sr[E][kHalf<V>][N];
  with_width(p.table_type, [&](auto width) {
    const auto *cos = static_cast<const decltype(width)*>(p.cos), *sin = static_cast<const decltype(width)*>(p.sin);
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int k = 0; k < kHalf<V>; ++k)
#pragma unroll
        for (int n = 0; n < N; ++n) {
          cr[e][k][n] = turned[e] ? __ldg(cos + row[e] * p.cos_pitch + l.slot[e].column + 2 * k + n) : 0;
          sr[e][k][n] = turned[e] ? __ldg(sin + row[e] * p.sin_pitch + l.slot[e].column + 2 * k + n) : 0;
        }
  });
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int k = 0; k < kHalf<V>; ++k) {
      c[e][k] = turned[e] ? make_float2(any_value(cr[e][k][0], p.table_type), any_value(cr[e][k][N - 1], p.table_type)) : twice(1.f);
      s[e][k] = turned[e] ? make_float2(any_value(sr[e][k][0], p.table_type), any_value(sr[e][k][N - 1], p.table_type)) : twice(0.f);
    }
}

// Heads of a CTA: part 0 q, 1 k, 2 v; heads first .. first + count of it.
struct Heads {
  int part, first, count;
};
__device__ __forceinline__ Heads heads_of(int chunk, const NrParams& p) {
  int part = 0, n = p.heads;
  if (chunk >= p.q_chunks) {
    chunk -= p.q_chunks;
    part = 1;
    n = p.kv_heads;
    if (chunk >= p.kv_chunks) chunk -= p.kv_chunks, part = 2;
  }
  const int first = chunk * p.per_chunk;
  return {part, first, min(p.per_chunk, n - first)};
}
__device__ __forceinline__ int packed_head(const Heads& h, const NrParams& p) { return h.first + (h.part > 0 ? p.heads : 0) + (h.part > 1 ? p.kv_heads : 0); }

// (x - mean) * inverse in place; returns the inverse.  The variance is that of centred values.
template <int V, int G, int E>
__device__ __forceinline__ float normalise(float2 (&x)[E][kSides<V>][kHalf<V>], const Lane<V, E>& l, const NrParams& p, float eps) {
  float s[1];
  float2 t;
  if (p.kind == S3R_NORM_LAYER) {
    t = twice(0.f);
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int k = 0; k < kHalf<V>; ++k) t = fadd2(t, V == 1 ? x[e][0][k] : fadd2(x[e][0][k], x[e][kSides<V> - 1][k]));
    s[0] = t.x + t.y;
    group_sum<G>(s);
    float minus_mean[E];
#pragma unroll
    for (int e = 0; e < E; ++e) minus_mean[e] = s[0] * l.share[e];
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int m = 0; m < kSides<V>; ++m)
#pragma unroll
        for (int k = 0; k < kHalf<V>; ++k) x[e][m][k] = fadd2(x[e][m][k], twice(minus_mean[e]));
  }
  t = twice(0.f);
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int m = 0; m < kSides<V>; ++m)
#pragma unroll
      for (int k = 0; k < kHalf<V>; ++k) t = ffma2(x[e][m][k], x[e][m][k], t);
  s[0] = t.x + t.y;
  group_sum<G>(s);
  const float inverse = rsqrtf(fmaf(s[0], p.inverse_dim, eps));
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int m = 0; m < kSides<V>; ++m)
#pragma unroll
      for (int k = 0; k < kHalf<V>; ++k) x[e][m][k] = fmul2(x[e][m][k], twice(inverse));
  return inverse;
}

// Rotation and the norm's weight and bias are one linear map of a pair of normalised values, of which a thread keeps six numbers per token:
//   out1 = n1 (w1 c) - n2 (w2 s) + (b1 c - b2 s),  out2 = n2 (w2 c) + n1 (w1 s) + (b2 c + b1 s)
// Columns that no axis turns have no partner, not one times 0: 0 * infinity would be NaN.  What is added to them without a bias is -0, which leaves
// every value as it is, -0 too.  The step with the partner is taken back for them: a selection of each result took 133.9 us where this takes 132.8 (64 512
// tokens, all columns turned), and 100.1 for 95.4 with heads of 100.
template <int V, int G, int E, int BYTES, int CB>
__global__ void __launch_bounds__(kNrThreads, E * V > 4 || Tile<V, G, E, BYTES, CB, 1>::kChunks > 4 ? 4 : 6) norm_rope_fwd_kernel(const __grid_constant__ NrParams p) {
  using T = Tile<V, G, E, BYTES, CB, 1>;
  constexpr int H = kHalf<V>, S = kSides<V>, kChunks = T::kChunks;
  extern __shared__ __align__(16) char smem[];
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * kNrWarps + warp) * T::kRows;       // token of the warp's first row
  const int64_t token = first + lane / G, b = static_cast<uint32_t>(token) / p.tokens;
  const bool in = token < p.rows_of_tokens;
  const int at = static_cast<int>(token - b * p.tokens);
  const Heads h = heads_of(blockIdx.y, p);
  Lane<V, E> l;
  place<V, G, E>(l, p, lane % G);
  const int64_t row_bytes = p.head_dim * BYTES, plane = p.tokens * row_bytes;
  const uint32_t ring = smem_u32(smem) + warp * T::kBytes * (T::kAhead + 1), last = ring + T::kAhead * T::kBytes;
  const char* from[kChunks];
  char* to[kChunks];
  uint32_t place_of[kChunks];
#pragma unroll
  for (int n = 0; n < kChunks; ++n) {
    const auto c = T::chunk(n, lane, static_cast<int>(row_bytes));
    const uint32_t tok = static_cast<uint32_t>(first) + c.row, cb = tok / p.tokens, ct = tok - cb * p.tokens;       // fewer than 2^31
    const bool there = c.in && tok < p.rows_of_tokens;
    from[n] = there ? static_cast<const char*>(p.qkv) + (static_cast<int64_t>(cb) * p.stride_b + static_cast<int64_t>(ct) * p.stride_t) * BYTES + packed_head(h, p) * row_bytes + c.byte : nullptr;
    to[n] = static_cast<char*>(p.out[h.part]) + (static_cast<int64_t>(cb) * (h.part == 0 ? p.heads : p.kv_heads) + h.first) * plane + ct * row_bytes + c.byte;
    place_of[n] = c.at;
  }
  int left = h.count;                                              // heads that are still to be asked for
  uint32_t free = 0, full = 0;                                     // places in the ring
  auto next = [&](uint32_t& place) { place = place == (T::kAhead - 1) * T::kBytes ? 0 : place + T::kBytes; };
  auto fetch = [&] {
    if (left > 0)
#pragma unroll
      for (int n = 0; n < kChunks; ++n)
        if (from[n]) {
          T::ask(ring + free + place_of[n], from[n]);
          from[n] += row_bytes;
        }
    --left;
    next(free);
    cp_async_commit();
  };
  auto leave = [&](uint32_t tile) {
#pragma unroll
    for (int n = 0; n < kChunks; ++n)
      if (from[n]) {
        T::leave(to[n], tile + place_of[n]);
        to[n] += plane;
      }
  };
#pragma unroll
  for (int u = 0; u < T::kAhead; ++u) fetch();
  if (h.part == 2) {
    for (int i = 0; i < h.count; ++i) {
      cp_async_wait<T::kAhead - 1>();
      leave(ring + full);
      next(full);
      fetch();
    }
    return;
  }
  const bool normed = p.normed[h.part];
  float2 own[E][S][H], other[E][S][H], add[E][S][H];               // what multiplies a member, its partner, and what is added
  {
    float2 c[E][H], s[E][H], w[E][S][H], bias[E][S][H];
    angles<V, E>(c, s, l, p, b, at, in);
    parameter<V, E>(w, l, p.weight[h.part], p.param_type, 1.f);
    parameter<V, E>(bias, l, p.bias[h.part], p.param_type, 0.f);
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int m = 0; m < S; ++m)
#pragma unroll
        for (int k = 0; k < H; ++k) {
          const bool turned = l.slot[e].axis >= 0;
          own[e][m][k] = turned ? fmul2(w[e][m][k], c[e][k]) : w[e][m][k];
          other[e][m][k] = fmul2(quarter<V>(w[e], m, k, false), s[e][k]);
          add[e][m][k] = turned ? ffma2(bias[e][m][k], c[e][k], fmul2(quarter<V>(bias[e], m, k, false), s[e][k])) : p.bias[h.part] ? bias[e][m][k] : twice(-0.f);
        }
  }
  const uint32_t mine = lane / G * T::kPitch, zeros = smem_u32(smem) + T::kSmem - T::kZeros;
  uint32_t in_tile[E][2];                                          // its vectors in the first place; without columns: the zeros, whatever the place
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int m = 0; m < 2; ++m) in_tile[e][m] = l.on[e] ? ring + mine + (m ? l.slot[e].c1 : l.slot[e].c0) * BYTES : zeros;
  if (threadIdx.x < T::kZeros / 4) sts32(zeros + 4 * threadIdx.x, 0);
  __syncthreads();
  const float eps = p.eps[h.part];
  const int turned_slots = p.axes * (p.pairs / V);                 // a slot's number tells whether an axis turns it: no register for each
#pragma unroll 1
  for (int i = 0; i < h.count; ++i) {
    cp_async_wait<T::kAhead - 1>();
    __syncwarp();                                                  // every lane's copies are there, and the last head's results have left
    float2 x[E][S][H];
#pragma unroll
    for (int e = 0; e < E; ++e) take_slot<V, BYTES>(x[e], in_tile[e][0] + (l.on[e] ? full : 0), in_tile[e][1] + (l.on[e] ? full : 0), p.type);
    next(full);
    __syncwarp();
    fetch();
    if (normed) normalise<V, G, E>(x, l, p, eps);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float2 y[S][H];
#pragma unroll
      for (int m = 0; m < S; ++m)
#pragma unroll
        for (int k = 0; k < H; ++k) {
          const float2 partner = V == 1 ? make_float2(x[e][m][k].y, x[e][m][k].x) : x[e][S - 1 - m][k];
          y[m][k] = ffma2(x[e][m][k], own[e][m][k], ffma2(partner, other[e][m][k], add[e][m][k]));
          if (lane % G + e * G >= turned_slots) y[m][k] = ffma2(x[e][m][k], own[e][m][k], add[e][m][k]);
        }
      if (l.on[e]) put_slot<V, BYTES>(y, last + mine + l.slot[e].c0 * BYTES, last + mine + l.slot[e].c1 * BYTES, p.type);
    }
    __syncwarp();
    leave(last);
  }
}

// The gradient of a head: turned back, then through the norm as computed again from x.  Sums for weight and bias: over the CTA's tokens and heads in
// registers, over the warp's groups by shuffles, over warps in shared memory, over CTAs by norm_rope_sums_kernel.
template <int V, int G, int E, int BYTES, int CB>
__global__ void __launch_bounds__(kNrThreads, E * V > 4 || (V == 1 && E == 4) || Tile<V, G, E, BYTES, CB, 2>::kChunks > 4 ? 3 : 4) norm_rope_bwd_kernel(const __grid_constant__ NrParams p) {
  using T = Tile<V, G, E, BYTES, CB, 2>;
  constexpr int H = kHalf<V>, S = kSides<V>, kChunks = T::kChunks;
  extern __shared__ __align__(16) char smem[];
  __shared__ float red[2][kNrWarps][2 * V * G * E];
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Heads h = heads_of(blockIdx.y, p);
  const bool normed = h.part < 2 && p.normed[h.part < 2 ? h.part : 0];
  Lane<V, E> l;
  place<V, G, E>(l, p, lane % G);
  float2 w[E][S][H], dw[E][S][H], db[E][S][H];
  if (normed) parameter<V, E>(w, l, p.weight[h.part], p.param_type, 1.f);
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int m = 0; m < S; ++m)
#pragma unroll
      for (int k = 0; k < H; ++k) dw[e][m][k] = db[e][m][k] = twice(0.f);
  const char* d_out = static_cast<const char*>(p.d_out[h.part]);
  const int64_t row_bytes = p.head_dim * BYTES, width = (p.heads + 2 * p.kv_heads) * row_bytes, column = packed_head(h, p) * row_bytes;
  const int64_t d_head = p.d_strides[h.part][1] * BYTES;
  const int turned_slots = p.axes * (p.pairs / V);
  const uint32_t ring = smem_u32(smem) + warp * T::kBytes * (2 * T::kAhead + 1), last = ring + 2 * T::kAhead * T::kBytes, mine = lane / G * T::kPitch;
  const uint32_t zeros = smem_u32(smem) + T::kSmem - T::kZeros;
  uint32_t in_tile[E][2];                                          // its vectors in the first place; without columns: the zeros, whatever the place
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int m = 0; m < 2; ++m) in_tile[e][m] = l.on[e] ? ring + mine + (m ? l.slot[e].c1 : l.slot[e].c0) * BYTES : zeros;
  if (threadIdx.x < T::kZeros / 4) sts32(zeros + 4 * threadIdx.x, 0);
  __syncthreads();
  for (int64_t begin = static_cast<int64_t>(blockIdx.x) * kNrWarps * T::kRows; begin < p.rows_of_tokens; begin += static_cast<int64_t>(gridDim.x) * kNrWarps * T::kRows) {
    const int64_t first = begin + warp * T::kRows, token = first + lane / G, b = static_cast<uint32_t>(token) / p.tokens;
    const bool in = token < p.rows_of_tokens;
    const int at = static_cast<int>(token - b * p.tokens);
    const char *from[kChunks], *d_from[kChunks];
    char* to[kChunks];                                             // NULL: not there
    uint32_t place_of[kChunks];
#pragma unroll
    for (int n = 0; n < kChunks; ++n) {
      const auto c = T::chunk(n, lane, static_cast<int>(row_bytes));
      const uint32_t tok = static_cast<uint32_t>(first) + c.row, cb = tok / p.tokens, ct = tok - cb * p.tokens;       // fewer than 2^31
      from[n] = static_cast<const char*>(p.qkv) + (static_cast<int64_t>(cb) * p.stride_b + static_cast<int64_t>(ct) * p.stride_t) * BYTES + column + c.byte;
      d_from[n] = d_out + (static_cast<int64_t>(cb) * p.d_strides[h.part][0] + static_cast<int64_t>(ct) * p.d_strides[h.part][2]) * BYTES + h.first * d_head + c.byte;
      to[n] = c.in && tok < p.rows_of_tokens ? static_cast<char*>(p.d_qkv) + tok * width + column + c.byte : nullptr;
      place_of[n] = c.at;
    }
    int left = h.count;                                            // heads that are still to be asked for
    uint32_t free = 0, full = 0;                                   // places in the ring
    auto next = [&](uint32_t& place) { place = place == (T::kAhead - 1) * 2 * T::kBytes ? 0 : place + 2 * T::kBytes; };
    auto fetch = [&] {
      if (left > 0)
#pragma unroll
        for (int n = 0; n < kChunks; ++n)
          if (to[n]) {
            if (d_out) T::ask(ring + free + place_of[n], d_from[n]);
            if (normed) T::ask(ring + free + T::kBytes + place_of[n], from[n]);
            d_from[n] += d_head;
            from[n] += row_bytes;
          }
      --left;
      next(free);
      cp_async_commit();
    };
    auto leave = [&](uint32_t tile) {
#pragma unroll
      for (int n = 0; n < kChunks; ++n)
        if (to[n]) {
          T::leave(to[n], tile + place_of[n]);
          to[n] += row_bytes;
        }
    };
    __syncwarp();                                                  // the last tokens' tiles are read
#pragma unroll
    for (int u = 0; u < T::kAhead; ++u) fetch();
    float2 c[E][H], s[E][H];
    if (h.part < 2) angles<V, E>(c, s, l, p, b, at, in);
#pragma unroll 1
    for (int i = 0; i < h.count; ++i) {
      cp_async_wait<T::kAhead - 1>();
      if (h.part == 2) {
        if (!d_out)                                                // zeros, by way of the results' tile
#pragma unroll
          for (int n = 0; n < kChunks; ++n) {
            Vec<CB / 2, 2> zero;
#pragma unroll
            for (int k = 0; k < Vec<CB / 2, 2>::kWords; ++k) zero.w[k] = 0;
            if (to[n]) put_vec<CB / 2, 2>(zero, last + place_of[n]);
          }
        leave(d_out ? ring + full : last);
        next(full);
        fetch();
        continue;
      }
      __syncwarp();                                                // every lane's copies are there, and the last head's results have left
      float2 d[E][S][H], x[E][S][H];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        // a token that is not there has whatever was in the tile
        const uint32_t of = l.on[e] ? full : 0, there = in ? l.on[e] ? full + T::kBytes : 0 : 0;
        take_slot<V, BYTES>(d[e], in && d_out ? in_tile[e][0] + of : zeros, in && d_out ? in_tile[e][1] + of : zeros, p.type);
        if (normed) take_slot<V, BYTES>(x[e], in ? in_tile[e][0] + there : zeros, in ? in_tile[e][1] + there : zeros, p.type);
      }
      next(full);
      __syncwarp();
      fetch();
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float2 partner[S][H];
#pragma unroll
        for (int m = 0; m < S; ++m)
#pragma unroll
          for (int k = 0; k < H; ++k) partner[m][k] = fmul2(quarter<V>(d[e], m, k, true), s[e][k]);
        if (lane % G + e * G >= turned_slots) continue;            // no partner where nothing turns, as in the forward
#pragma unroll
        for (int m = 0; m < S; ++m)
#pragma unroll
          for (int k = 0; k < H; ++k) d[e][m][k] = ffma2(d[e][m][k], c[e][k], partner[m][k]);
      }
      if (normed) {
        const float inverse = normalise<V, G, E>(x, l, p, in ? p.eps[h.part] : 1.f);
        float2 t0 = twice(0.f), t1 = twice(0.f);                   // sums of e and of e n, e = d * weight
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
          for (int m = 0; m < S; ++m)
#pragma unroll
            for (int k = 0; k < H; ++k) {
              dw[e][m][k] = ffma2(d[e][m][k], x[e][m][k], dw[e][m][k]);
              db[e][m][k] = fadd2(db[e][m][k], d[e][m][k]);
              d[e][m][k] = fmul2(d[e][m][k], w[e][m][k]);
              t0 = fadd2(t0, d[e][m][k]);
              t1 = ffma2(d[e][m][k], x[e][m][k], t1);
            }
        float sums[2] = {t0.x + t0.y, t1.x + t1.y};
        group_sum<G>(sums);
        const float mean = p.kind == S3R_NORM_LAYER ? -sums[0] * p.inverse_dim * inverse : 0.f, along = -sums[1] * p.inverse_dim * inverse;
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
          for (int m = 0; m < S; ++m)
#pragma unroll
            for (int k = 0; k < H; ++k) d[e][m][k] = ffma2(d[e][m][k], twice(inverse), ffma2(x[e][m][k], twice(along), twice(mean)));
      }
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (l.on[e]) put_slot<V, BYTES>(d[e], last + mine + l.slot[e].c0 * BYTES, last + mine + l.slot[e].c1 * BYTES, p.type);
      __syncwarp();
      leave(last);
    }
  }
  if (!p.sums || !normed) return;                            // the same for the whole CTA
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int m = 0; m < S; ++m)
#pragma unroll
      for (int k = 0; k < H; ++k) {
#pragma unroll
        for (int o = 16; o >= G; o >>= 1) {
          dw[e][m][k] = fadd2(dw[e][m][k], make_float2(__shfl_xor_sync(0xffffffffu, dw[e][m][k].x, o), __shfl_xor_sync(0xffffffffu, dw[e][m][k].y, o)));
          db[e][m][k] = fadd2(db[e][m][k], make_float2(__shfl_xor_sync(0xffffffffu, db[e][m][k].x, o), __shfl_xor_sync(0xffffffffu, db[e][m][k].y, o)));
        }
        if ((threadIdx.x & 31) < G && l.on[e]) {
          const int x = column_x<V>(l.slot[e], m, k), y = column_y<V>(l.slot[e], m, k);
          red[0][threadIdx.x >> 5][x] = dw[e][m][k].x;
          red[1][threadIdx.x >> 5][x] = db[e][m][k].x;
          red[0][threadIdx.x >> 5][y] = dw[e][m][k].y;
          red[1][threadIdx.x >> 5][y] = db[e][m][k].y;
        }
      }
  __syncthreads();
  float* to = p.sums + (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * 2 * p.head_dim;
  for (int c = threadIdx.x; c < 2 * p.head_dim; c += kNrThreads) {
    const int which = c >= p.head_dim, col = c - which * p.head_dim;
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < kNrWarps; ++k) total += red[which][k][col];
    to[c] = total;
  }
}

// The CTAs' sums, in a fixed order: a CTA has 32 of a part's 2 * head_dim columns, a warp every 32nd row.
struct NrSums {
  const float* sums;
  void* out[2][2];                   // of q and k: weight, bias
  int64_t first[2], rows[2];
  int head_dim, type;
};
__global__ void __launch_bounds__(1024) norm_rope_sums_kernel(const __grid_constant__ NrSums p) {
  __shared__ float red[32][33];
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = blockIdx.y, col = blockIdx.x * 32 + lane;
  const bool in = col < 2 * p.head_dim;
  float total = 0.f;
  if (in)
    for (int64_t i = warp; i < p.rows[part]; i += 32 * 8) {        // eight on their way at a time
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = i + 32 * k < p.rows[part] ? __ldg(p.sums + (p.first[part] + i + 32 * k) * 2 * p.head_dim + col) : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) total += v[k];
    }
  red[warp][lane] = total;
  __syncthreads();
  const int which = col >= p.head_dim;
  void* out = p.out[part][which];
  if (warp == 0 && in && out) {
    float v[1] = {0.f};
#pragma unroll
    for (int i = 0; i < 32; ++i) v[0] += red[i][lane];
    Raw<1> o;
    pack<1>(o, v, p.type);
    store_raw<1>(o, out, p.type, col - which * p.head_dim);
  }
}

template <int V, int G, int E, int BYTES, int CB>
static int run_norm_rope(const NrParams& p, bool backward, unsigned ctas, cudaStream_t st) {
  const dim3 grid(ctas, static_cast<unsigned>(p.q_chunks + 2 * p.kv_chunks));
  constexpr int kForward = Tile<V, G, E, BYTES, CB, 1>::kSmem, kBackward = Tile<V, G, E, BYTES, CB, 2>::kSmem;
  static std::atomic<uint64_t> ready[2];
  if (attributes_missing(ready[backward])) {
    if (backward) S3R_CUDA(cudaFuncSetAttribute(norm_rope_bwd_kernel<V, G, E, BYTES, CB>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBackward));
    else S3R_CUDA(cudaFuncSetAttribute(norm_rope_fwd_kernel<V, G, E, BYTES, CB>, cudaFuncAttributeMaxDynamicSharedMemorySize, kForward));
    attributes_set(ready[backward]);
  }
  if (backward) return launch(norm_rope_bwd_kernel<V, G, E, BYTES, CB>, grid, kNrThreads, kBackward, st, p);
  return launch(norm_rope_fwd_kernel<V, G, E, BYTES, CB>, grid, kNrThreads, kForward, st, p);
}
// The widest copy of at most 16 bytes that divides rows, addresses and strides, and no narrower than a vector
template <int V, int G, int E, int BYTES>
static int by_chunk(const NrParams& p, int bytes, bool backward, unsigned ctas, cudaStream_t st) {
  constexpr int kVector = V * BYTES > 16 ? 16 : V * BYTES;
  if (bytes >= 16) return run_norm_rope<V, G, E, BYTES, 16>(p, backward, ctas, st);
  if constexpr (kVector <= 8) {
    if (bytes == 8) return run_norm_rope<V, G, E, BYTES, 8>(p, backward, ctas, st);
  }
  if constexpr (kVector <= 4) {
    if (bytes == 4) return run_norm_rope<V, G, E, BYTES, 4>(p, backward, ctas, st);
  }
  return run_norm_rope<V, G, E, BYTES, kVector>(p, backward, ctas, st);
}
// Elements of a thread's vectors, threads of a head (a power of two), pairs of vectors of each, bytes of a copy.
struct NrShape {
  int vector, group, each, bytes;
};
template <int BYTES>
static int pick_norm_rope(const NrParams& p, NrShape s, bool backward, unsigned ctas, cudaStream_t st) {
  switch (s.vector * 1000 + s.group * 10 + s.each) {
    case 4081: return by_chunk<4, 8, 1, BYTES>(p, s.bytes, backward, ctas, st);
    case 4161: return by_chunk<4, 16, 1, BYTES>(p, s.bytes, backward, ctas, st);
    case 4321: return by_chunk<4, 32, 1, BYTES>(p, s.bytes, backward, ctas, st);
    case 2082: return by_chunk<2, 8, 2, BYTES>(p, s.bytes, backward, ctas, st);
    case 2083: return by_chunk<2, 8, 3, BYTES>(p, s.bytes, backward, ctas, st);
    case 2162: return by_chunk<2, 16, 2, BYTES>(p, s.bytes, backward, ctas, st);
    case 2163: return by_chunk<2, 16, 3, BYTES>(p, s.bytes, backward, ctas, st);
    case 2322: return by_chunk<2, 32, 2, BYTES>(p, s.bytes, backward, ctas, st);
    case 1083: return by_chunk<1, 8, 3, BYTES>(p, s.bytes, backward, ctas, st);
    case 1084: return by_chunk<1, 8, 4, BYTES>(p, s.bytes, backward, ctas, st);
    case 1163: return by_chunk<1, 16, 3, BYTES>(p, s.bytes, backward, ctas, st);
    case 1164: return by_chunk<1, 16, 4, BYTES>(p, s.bytes, backward, ctas, st);
    case 1323: return by_chunk<1, 32, 3, BYTES>(p, s.bytes, backward, ctas, st);
    default: return by_chunk<1, 32, 4, BYTES>(p, s.bytes, backward, ctas, st);
  }
}

// Heads are split over CTAs until there are `per_sm` for every SM; no further than that, a token's angles are found once per CTA, and the backward has
// a row of sums for each.  Forward / backward: 3 x 1041 tokens of 12 + 4 heads of 80, four per SM 13.8 / 19, eight 10.2 / 22.5, twelve 14 / 26; 1041 of
// 16 heads of 64, four 8.2 / 11.3, eight 7.2 / 15; 300 of them backward, two or three 7.9, four 11.1; 2 x 1041 backward, two 15.5, three 14.4, six 18.1.
constexpr int kNrForwardSplit = 8, kNrBackwardSplit = 3;
static void norm_rope_chunks(int64_t token_ctas, int heads, int kv_heads, int per_sm, int* per_chunk, int* q_chunks, int* kv_chunks) {
  int per = heads;
  while (per > 1) {
    const int64_t chunks = (heads + per - 1) / per + 2 * ((kv_heads + per - 1) / per);
    if (chunks * token_ctas >= static_cast<int64_t>(per_sm) * sm_count()) break;
    per = (per + 1) / 2;
  }
  *per_chunk = per;
  *q_chunks = (heads + per - 1) / per;
  *kv_chunks = (kv_heads + per - 1) / per;
}
// CTAs of the backward along the tokens: each walks over its share of them and leaves one row of sums.  Three times what is resident, so that v's,
// which do least and come last, fill the gaps of the others: 64 x 1008 tokens 231 us, all resident 270, twice 250, four times 231 to 238; 48 x 256
// 53.7, 59.4, 56.9, 55.3.
constexpr int kNrBackwardCtas = 12;      // per SM
static unsigned norm_rope_bwd_ctas(int64_t token_ctas, int chunks) {
  const int64_t most = kNrBackwardCtas * static_cast<int64_t>(sm_count()) / chunks;
  return static_cast<unsigned>(token_ctas < most ? token_ctas : most < 1 ? 1 : most);
}

static int check_norm_rope(const s3r_qkv_norm_rope* f, const char* what) {
  S3R_REQUIRE(f && f->qkv, S3R_ERR_NULL, "%s: NULL pointer", what);
  S3R_REQUIRE(f->batch > 0 && f->tokens > 0 && f->heads > 0 && f->kv_heads > 0, S3R_ERR_SHAPE, "%s: sizes must be positive", what);
  S3R_REQUIRE(f->head_dim >= 2 && f->head_dim <= 256 && f->head_dim % 2 == 0, S3R_ERR_UNSUPPORTED, "%s: head_dim %d (even, 2 to 256)", what, f->head_dim);
  S3R_REQUIRE(f->heads <= 4096 && f->kv_heads <= 4096 && f->tokens < (1ll << 31) - 1024 && f->batch < (1ll << 31) - 1024 && f->batch * f->tokens < (1ll << 31) - 1024,
              S3R_ERR_TOO_LARGE, "%s: too many heads or tokens", what);
  S3R_REQUIRE(known_type(f->type), S3R_ERR_UNSUPPORTED, "%s: types are fp32, bf16 and fp16", what);
  S3R_REQUIRE(f->kind == S3R_NORM_LAYER || f->kind == S3R_NORM_RMS, S3R_ERR_UNSUPPORTED, "%s: kind %d", what, f->kind);
  S3R_REQUIRE((f->q_normed || (!f->q_weight && !f->q_bias)) && (f->k_normed || (!f->k_weight && !f->k_bias)), S3R_ERR_SHAPE, "%s: weight and bias belong to a norm", what);
  S3R_REQUIRE(!(f->q_weight || f->q_bias || f->k_weight || f->k_bias) || known_type(f->param_type), S3R_ERR_UNSUPPORTED, "%s: types are fp32, bf16 and fp16", what);
  S3R_REQUIRE(f->axes >= 0 && (f->axes == 0 || (f->pairs > 0 && f->rows > 0 && f->pos && f->cos && f->sin)), S3R_ERR_SHAPE, "%s: a rotation needs positions and tables", what);
  S3R_REQUIRE(f->axes == 0 || (f->axes <= 128 && f->pairs <= 128 && 2 * f->axes * f->pairs <= f->head_dim), S3R_ERR_SHAPE, "%s: %d axes of %d pairs in %d columns", what,
              f->axes, f->pairs, f->head_dim);
  S3R_REQUIRE(f->axes == 0 || known_type(f->table_type), S3R_ERR_UNSUPPORTED, "%s: types are fp32, bf16 and fp16", what);
  const void* params[] = {f->q_weight, f->q_bias, f->k_weight, f->k_bias};
  for (const void* t : params) S3R_REQUIRE(!t || reinterpret_cast<uintptr_t>(t) % type_bytes(f->param_type) == 0, S3R_ERR_ALIGNMENT, "%s: elements must be aligned", what);
  S3R_REQUIRE(reinterpret_cast<uintptr_t>(f->qkv) % type_bytes(f->type) == 0 &&
                  (f->axes == 0 || ((reinterpret_cast<uintptr_t>(f->cos) | reinterpret_cast<uintptr_t>(f->sin)) % type_bytes(f->table_type) == 0 &&
                                    reinterpret_cast<uintptr_t>(f->pos) % 8 == 0)), S3R_ERR_ALIGNMENT, "%s: elements must be aligned", what);
  return 0;
}

// The largest vector, up to four elements, that divides pairs, what is not turned, addresses and strides, and groups of threads that hold a head with
// eight to sixteen values each: a thread with less repeats the sums' shuffles for little (16 128 tokens of 16 heads, forward / backward: 50 channels, one
// pair for each of 32 threads 73 / 156, four for each of 8 64 / 135; 72 channels 87 / 188 and 53 / 104).  In a few tokens' work it costs a microsecond.
static NrShape norm_rope_shape(const s3r_qkv_norm_rope* f, const void* const* pointers, int n_pointers, const int64_t* strides, int n_strides) {
  const int turned = 2 * f->axes * f->pairs, size = type_bytes(f->type);
  uint64_t grid = 16 | static_cast<uint64_t>(f->head_dim) * size;      // its lowest bit: what rows, addresses and strides are multiples of
  for (int i = 0; i < n_pointers; ++i) grid |= reinterpret_cast<uintptr_t>(pointers[i]);
  for (int i = 0; i < n_strides; ++i) grid |= static_cast<uint64_t>(strides[i]) * size;
  const int bytes = static_cast<int>(grid & (~grid + 1));
  int v = 4;
  while (v > 1 && ((f->axes && f->pairs % v) || (f->head_dim - turned) % (2 * v) || (v * size < 16 ? v * size : 16) > bytes)) v /= 2;
  int slots = f->head_dim / (2 * v);
  if (v == 4) {
    // A quarter of the threads or more without columns: three vectors of two for half as many threads, where those still fill the GPU (96 channels,
    // 16 128 tokens 63 / 117 and 58 / 107; 6246 tokens 27.3 / 51.7 and 27.9 / 48.2)
    const int group = slots <= 8 ? 8 : slots <= 16 ? 16 : 32;
    const int64_t halved = (f->batch * f->tokens * (group / 2) + kNrThreads - 1) / kNrThreads;      // CTAs of groups of half as many threads
    if (group == 8 || 4 * slots > 3 * group || halved < 2 * static_cast<int64_t>(sm_count())) return {4, group, 1, bytes};
    v = 2, slots *= 2;
  }
  int group = 8;
  const int most = v == 2 ? 3 : 4, least = most - 1;
  while (group < 32 && slots > group * most) group *= 2;
  return {v, group, slots <= group * least ? least : most, bytes};
}

static NrParams norm_rope_params(const s3r_qkv_norm_rope* f) {
  NrParams p = {};
  p.qkv = f->qkv;
  p.cos = f->cos;
  p.sin = f->sin;
  p.pos = f->pos;
  p.weight[0] = f->q_weight;
  p.weight[1] = f->k_weight;
  p.bias[0] = f->q_bias;
  p.bias[1] = f->k_bias;
  p.stride_b = f->stride_b;
  p.stride_t = f->stride_t;
  p.pos_stride_b = f->pos_stride_b;
  p.pos_stride_t = f->pos_stride_t;
  p.cos_pitch = f->cos_pitch;
  p.sin_pitch = f->sin_pitch;
  p.rows_of_tokens = f->batch * f->tokens;
  p.tokens = static_cast<uint32_t>(f->tokens);
  p.heads = f->heads;
  p.kv_heads = f->kv_heads;
  p.head_dim = f->head_dim;
  p.kind = f->kind;
  p.type = f->type;
  p.param_type = f->param_type;
  p.table_type = f->table_type;
  p.axes = f->axes;
  p.pairs = f->axes ? f->pairs : 0;
  p.rows = f->rows;
  p.normed[0] = f->q_normed;
  p.normed[1] = f->k_normed;
  p.eps[0] = f->q_eps;
  p.eps[1] = f->k_eps;
  p.inverse_dim = 1.f / static_cast<float>(f->head_dim);
  p.status = device_status_ptr();
  return p;
}

}  // namespace s3r

using namespace s3r;

extern "C" int s3r_qkv_norm_rope_fwd(const s3r_qkv_norm_rope* f, void* stream) {
  if (const int rc = check_norm_rope(f, "s3r_qkv_norm_rope_fwd")) return rc;
  S3R_REQUIRE(f->q && f->k && f->v, S3R_ERR_NULL, "s3r_qkv_norm_rope_fwd: NULL pointer");
  for (const void* t : {f->q, f->k, f->v}) S3R_REQUIRE(reinterpret_cast<uintptr_t>(t) % type_bytes(f->type) == 0, S3R_ERR_ALIGNMENT, "s3r_qkv_norm_rope_fwd: elements must be aligned");
  NrParams p = norm_rope_params(f);
  S3R_REQUIRE(p.status, S3R_ERR_DRIVER, "s3r_qkv_norm_rope_fwd: no status word");
  p.out[0] = f->q;
  p.out[1] = f->k;
  p.out[2] = f->v;
  const void* pointers[] = {f->qkv, f->q, f->k, f->v};
  const int64_t strides[] = {f->batch > 1 ? f->stride_b : 0, f->tokens > 1 ? f->stride_t : 0};
  const NrShape s = norm_rope_shape(f, pointers, 4, strides, 2);
  const int64_t per = kNrThreads / s.group, ctas = (p.rows_of_tokens + per - 1) / per;
  norm_rope_chunks(ctas, f->heads, f->kv_heads, kNrForwardSplit, &p.per_chunk, &p.q_chunks, &p.kv_chunks);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return f->type == S3R_F32 ? pick_norm_rope<4>(p, s, false, static_cast<unsigned>(ctas), st) : pick_norm_rope<2>(p, s, false, static_cast<unsigned>(ctas), st);
}

// Room for either shape of the grid: the chunks of heads depend on the vectors that addresses allow.
extern "C" size_t s3r_qkv_norm_rope_bwd_workspace_bytes(int64_t batch, int64_t tokens, int heads, int kv_heads, int head_dim) {
  if (batch <= 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0) return 0;
  // chunks of q and k times CTAs along the tokens: all of them together as many as there are, or one for each chunk of a head at least
  return static_cast<size_t>(kNrBackwardCtas * sm_count() + heads + 2 * kv_heads) * 2 * head_dim * sizeof(float);
}

extern "C" int s3r_qkv_norm_rope_bwd(const s3r_qkv_norm_rope* f, const s3r_qkv_norm_rope_grad* g, void* stream) {
  if (const int rc = check_norm_rope(f, "s3r_qkv_norm_rope_bwd")) return rc;
  S3R_REQUIRE(g && g->d_qkv, S3R_ERR_NULL, "s3r_qkv_norm_rope_bwd: NULL pointer");
  for (const void* t : {g->dq, g->dk, g->dv, static_cast<const void*>(g->d_qkv)})
    S3R_REQUIRE(reinterpret_cast<uintptr_t>(t) % type_bytes(f->type) == 0, S3R_ERR_ALIGNMENT, "s3r_qkv_norm_rope_bwd: elements must be aligned");
  S3R_REQUIRE((f->q_normed || (!g->d_q_weight && !g->d_q_bias)) && (f->k_normed || (!g->d_k_weight && !g->d_k_bias)), S3R_ERR_SHAPE,
              "s3r_qkv_norm_rope_bwd: weight and bias belong to a norm");
  const bool sums = g->d_q_weight || g->d_q_bias || g->d_k_weight || g->d_k_bias;
  const size_t need = s3r_qkv_norm_rope_bwd_workspace_bytes(f->batch, f->tokens, f->heads, f->kv_heads, f->head_dim);
  S3R_REQUIRE(!sums || known_type(f->param_type), S3R_ERR_UNSUPPORTED, "s3r_qkv_norm_rope_bwd: types are fp32, bf16 and fp16");
  S3R_REQUIRE(!sums || (g->workspace && g->workspace_bytes >= need && reinterpret_cast<uintptr_t>(g->workspace) % 4 == 0), S3R_ERR_TOO_LARGE,
              "s3r_qkv_norm_rope_bwd: workspace too small");
  NrParams p = norm_rope_params(f);
  S3R_REQUIRE(p.status, S3R_ERR_DRIVER, "s3r_qkv_norm_rope_bwd: no status word");
  const void* d_out[] = {g->dq, g->dk, g->dv};
  const int64_t* d_strides[] = {g->dq_strides, g->dk_strides, g->dv_strides};
  const void* pointers[5] = {f->qkv, g->d_qkv};
  int64_t strides[11] = {f->batch > 1 ? f->stride_b : 0, f->tokens > 1 ? f->stride_t : 0};
  int np = 2, ns = 2;
  for (int i = 0; i < 3; ++i) {
    p.d_out[i] = d_out[i];
    if (!d_out[i]) continue;
    pointers[np++] = d_out[i];
    const int64_t sizes[3] = {f->batch, i == 0 ? f->heads : f->kv_heads, f->tokens};
    for (int k = 0; k < 3; ++k) p.d_strides[i][k] = strides[ns++] = sizes[k] > 1 ? d_strides[i][k] : 0;
  }
  p.d_qkv = g->d_qkv;
  p.sums = sums ? static_cast<float*>(g->workspace) : nullptr;
  const NrShape s = norm_rope_shape(f, pointers, np, strides, ns);
  const int64_t per = kNrThreads / s.group, token_ctas = (p.rows_of_tokens + per - 1) / per;
  norm_rope_chunks(token_ctas, f->heads, f->kv_heads, kNrBackwardSplit, &p.per_chunk, &p.q_chunks, &p.kv_chunks);
  const int chunks = p.q_chunks + 2 * p.kv_chunks;
  const unsigned ctas = norm_rope_bwd_ctas(token_ctas, chunks);
  S3R_REQUIRE(!sums || static_cast<size_t>(p.q_chunks + p.kv_chunks) * ctas * 2 * f->head_dim * sizeof(float) <= need, S3R_ERR_TOO_LARGE,
              "s3r_qkv_norm_rope_bwd: workspace too small");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = f->type == S3R_F32 ? pick_norm_rope<4>(p, s, true, ctas, st) : pick_norm_rope<2>(p, s, true, ctas, st);
  if (rc || !sums) return rc;
  NrSums n = {};
  n.sums = p.sums;
  n.out[0][0] = g->d_q_weight;
  n.out[0][1] = g->d_q_bias;
  n.out[1][0] = g->d_k_weight;
  n.out[1][1] = g->d_k_bias;
  n.rows[0] = static_cast<int64_t>(p.q_chunks) * ctas;
  n.first[1] = n.rows[0];
  n.rows[1] = static_cast<int64_t>(p.kv_chunks) * ctas;
  n.head_dim = f->head_dim;
  n.type = f->param_type;
  return launch(norm_rope_sums_kernel, dim3(static_cast<unsigned>((2 * f->head_dim + 31) / 32), 2), 1024, 0, st, n);
}
