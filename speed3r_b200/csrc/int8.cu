// Products of 8-bit integers with a scale per token and per output channel, and the tokens they are made of.
//   quantise  scale[r] = max |x[r]| / 127, q = x / scale to nearest even.  Bound: HBM, a row is read once and kept in registers.
//   product   out[m, n] = (sum_k a[m, k] b[n, k]) a_scale[m] b_scale[n] + bias[n].  The sums are exact (32-bit integers), so that
//             no order of the k-steps changes a result.
#include <climits>
#include <type_traits>

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
      w[k / 4] = to_s8x4(f + k, inverse);
    if constexpr (W == 8) *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(q) = w[0];
  }
}

// Rows of a warp: short ones in CTAs of eight, which start half as often (100 000 x 256 bf16 27 -> 16 us, x 512 28.3 -> 27.4; x 1024 31 in CTAs
// of four, 33 in those).
__host__ __device__ constexpr int quantize_threads(int G, int E) { return G >= 128 ? G : E <= 16 ? 256 : 128; }
template <int W, int G, int E>
__global__ void __launch_bounds__(quantize_threads(G, E)) quantize_kernel(const __grid_constant__ QuantParams p) {
  constexpr int kRows = quantize_threads(G, E) / G, N = E / W;
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
        big = max_abs<W>(big, f);
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
      big = max_abs<W>(big, f);
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
  constexpr int kRows = quantize_threads(G, E) / G;
  const int64_t grid = (p.rows + kRows - 1) / kRows;
  return launch(quantize_kernel<W, G, E>, static_cast<unsigned>(grid), quantize_threads(G, E), 0, st, p);
}
template <int W>
static int pick_quantize(const QuantParams& p, cudaStream_t st) {
  const int C = p.channels;
  // 32 values per thread, all asked for at once: 64 512 x 4096 bf16 117 us (6.8 TB/s); with 16 135, and CTAs that stay with rows staged
  // ahead, as the norms have them, more.  A warp per row up to 2048 values, which needs no barrier (40 000 x 2048 41 us, 128 threads 44; x 1536
  // 35 and 44); a few rows, where latency counts, the other way round.
  const bool few = p.rows <= 2 * sm_count();
  if (C <= 256) return run_quantize<W, 32, 8>(p, st);
  if (C <= 1024 && few) return run_quantize<W, 128, 8>(p, st);
  if (C <= 512) return run_quantize<W, 32, 16>(p, st);
  if (C <= 1024) return run_quantize<W, 32, 32>(p, st);
  if (C <= 2048 && few) return run_quantize<W, 128, 16>(p, st);
  if (C <= 2048) return run_quantize<W, 32, 64>(p, st);
  if (C <= 4096) return run_quantize<W, 128, 32>(p, st);
  if (C <= 16384) return run_quantize<W, 512, 32>(p, st);
  return run_quantize<W, 1024, 0>(p, st);
}

// ---------------------------------------------------------------------------------------------------------------------
// 8-bit rows that begin anywhere, to rows at multiples of 16 bytes, as copies by TMA want them (zeros behind their end): 16 bytes per
// thread from five aligned words.  Bound: HBM, once in and once out (PyTorch's copy moves a byte per thread).
// ---------------------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) pad_rows_kernel(const int8_t* __restrict__ src, int64_t src_pitch, int8_t* __restrict__ dst, int64_t dst_pitch,
                                                       int64_t rows, int K, int chunks) {
  griddep_wait();
  griddep_launch();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, row = i / chunks;
  if (row >= rows) return;
  const int c = static_cast<int>(i - row * chunks) * 16;
  const int8_t* from = src + row * src_pitch + c;
  uint32_t w[4];
  const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(from) & 3);
  const int8_t *first = from - off, *begin = src, *end = src + (rows - 1) * src_pitch + K;
  if (c + 16 <= K && first >= begin && first + 20 <= end) {
    uint32_t v[5];
#pragma unroll
    for (int k = 0; k < 5; ++k) v[k] = __ldg(reinterpret_cast<const uint32_t*>(first) + k);
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(v[k], v[k + 1], off * 8);
  } else {                                               // the end of a row, and the first and last bytes of all
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      w[k] = 0;
      for (int b = 0; b < 4; ++b)
        if (c + 4 * k + b < K) w[k] |= static_cast<uint32_t>(static_cast<uint8_t>(from[4 * k + b])) << (8 * b);
    }
  }
  *reinterpret_cast<uint4*>(dst + row * dst_pitch + c) = make_uint4(w[0], w[1], w[2], w[3]);
}

// ---------------------------------------------------------------------------------------------------------------------
// product on tcgen05: persistent CTAs, K in steps of 128 bytes through a ring of TMA copies, the sums of two tiles in tensor memory
// so that one is written out while the next is summed.  One warp copies, one issues the products, eight take the sums (32 rows and
// half of the columns each), scale them and store through shared memory.
// At K = 1024 no unit is full (tensor pipe 0.72 busy, shared memory 0.55, L2 0.4, at 1.64 GHz under power), but the results' way out delays the
// copies in: 64 512 x 4096 take 155 us without the results' part, 166 without the stores at its end, 201 with them.  Tried and not kept: sixteen warps for the sums
// (220), stores from registers by way of shared memory (211) and, with a's rows of up to 1024 bytes staying where they are, half as
// many bytes to copy but three steps of the ring in place of five (234; 156 without the stores).
// CTAS = 2: a pair of CTAs multiplies 256 rows with TN columns; each holds 128 rows of a and half of b's rows, the products read both
// halves.  A k-step then brings half as much of b into either CTA's shared memory, whose bandwidth bounds one CTA alone.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kI8Warps = 8, kI8Threads = 64 + 32 * kI8Warps, kI8Piece = 4096;       // a warp's piece of the output: 32 rows of 128 bytes

struct I8Params {
  const float *a_scale, *b_scale, *bias;
  void* out;
  int64_t M;
  int N, K;
  int m_tiles, n_tiles;
  uint32_t copy_out;             // rows of the output are a multiple of 16 bytes: TMA stores
  uint32_t* status;
};

template <int TN, int CTAS>
struct I8Cfg {
  static constexpr int kABytes = 128 * 128, kBBytes = TN / CTAS * 128, kBytes = kABytes + kBBytes;
  static constexpr int kStages = 163840 / kBytes > 6 ? 6 : 163840 / kBytes;
  static constexpr int kOut = kStages * kBytes, kColumns = kOut + kI8Warps * kI8Piece;
  static constexpr int kSpan = TN / 2 < 64 ? 64 : TN / 2;       // columns of an epilogue warp: whole pieces
  static constexpr int kSmem = kColumns + kI8Warps * kSpan * 16 + 1024;
};

struct I8Ctl {
  uint64_t full[6], empty[6], acc_full[2], acc_empty[2], drained, pause;
  uint32_t tmem_base, abort_flag;
};

// kind::i8, signed x signed -> int32
__host__ __device__ constexpr uint32_t umma_idesc_i8(uint32_t M, uint32_t N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | ((M >> 4) << 24);
}
// Four k-steps of 32 bytes.
#define S3R_I8_K4(group)                                                     \
  asm volatile(                                                              \
      "{\n\t.reg .pred p, pt;\n\t.reg .b64 a, b;\n\t"                        \
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.u32 pt, 0, 0;\n\t"                   \
      "tcgen05.mma.cta_group::" group ".kind::i8 [%0], %1, %2, %3, p;\n\t"   \
      "add.s64 a, %1, 2;\n\tadd.s64 b, %2, 2;\n\t"                           \
      "tcgen05.mma.cta_group::" group ".kind::i8 [%0], a, b, %3, pt;\n\t"    \
      "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"                             \
      "tcgen05.mma.cta_group::" group ".kind::i8 [%0], a, b, %3, pt;\n\t"    \
      "add.s64 a, a, 2;\n\tadd.s64 b, b, 2;\n\t"                             \
      "tcgen05.mma.cta_group::" group ".kind::i8 [%0], a, b, %3, pt;\n\t}"   \
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accum)        \
      : "memory")
template <int CTAS>
__device__ __forceinline__ void umma_i8_k4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accum) {
  if constexpr (CTAS == 2) S3R_I8_K4("2");
  else S3R_I8_K4("1");
}
// arrives at this barrier of both CTAs of a pair (of this CTA's) once the products issued so far are done
template <int CTAS>
struct Ctas {};
template <int CTAS>
__device__ __forceinline__ void umma_commit(uint64_t* bar, Ctas<CTAS>) {
  if constexpr (CTAS == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                 "h"(static_cast<uint16_t>(3)) : "memory");
  else
    umma_commit(bar);
}
// address of `bar` in the pair's first CTA
template <int CTAS>
__device__ __forceinline__ uint32_t first_cta(uint64_t* bar) {
  uint32_t at = smem_u32(bar);
  if constexpr (CTAS == 2) asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(at));
  return at;
}
// What it tells of - sums read from tensor memory - is complete in front of it (tcgen05.wait::ld, tcgen05.fence) and is no memory of this
// thread, so that no release at the cluster's scope is needed: that waits for every store in flight, 2000 of a tile's 7000 cycles.
template <int CTAS>
__device__ __forceinline__ void arrive_first_cta(uint64_t* bar) {
  if constexpr (CTAS == 2)
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(first_cta<2>(bar)) : "memory");
  else
    mbar_arrive(bar);
}
// `bar`: address of a barrier of this CTA, or of the pair's other one
template <int CTAS>
__device__ __forceinline__ void tma_load_2d(uint32_t dst_smem, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  if constexpr (CTAS == 2)
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst_smem), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst_smem), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
// 32 lanes x 32 columns as four rows and eight columns per lane: register 16 h + 4 j + 2 i + e of lane l holds row 16 h + 8 i + l / 4,
// column 8 j + 2 (l % 4) + e.
__device__ __forceinline__ void tmem_ld_32x32(uint32_t taddr, uint32_t (&r)[32]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[16 * h]), "=r"(r[16 * h + 1]), "=r"(r[16 * h + 2]), "=r"(r[16 * h + 3]), "=r"(r[16 * h + 4]), "=r"(r[16 * h + 5]),
                   "=r"(r[16 * h + 6]), "=r"(r[16 * h + 7]), "=r"(r[16 * h + 8]), "=r"(r[16 * h + 9]), "=r"(r[16 * h + 10]), "=r"(r[16 * h + 11]),
                   "=r"(r[16 * h + 12]), "=r"(r[16 * h + 13]), "=r"(r[16 * h + 14]), "=r"(r[16 * h + 15])
                 : "r"(taddr + (static_cast<uint32_t>(16 * h) << 16)));
}
// The wait for it, tied to its registers: nothing that reads them moves in front of it.
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                 "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]),
                 "+r"(r[31])::"memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src_smem, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];"
               ::"l"(map), "r"(src_smem), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
template <int CTAS>
__device__ __forceinline__ void sync_pair() {
  if constexpr (CTAS == 2) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <int CTAS>
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns) {
  if constexpr (CTAS == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns) : "memory");
  else tmem_dealloc(at, columns);
}

// A piece (32 rows of 128 bytes, swizzled) to rows that begin anywhere: eight lanes per row move what lies in whole 16 bytes of memory, and
// element by element what is in front of them and behind.  64 512 x 1023, K = 1024, bf16: element by element alone 170 us, this way 89;
// 1024 columns by TMA 57 - sectors that two pieces share are written twice.
template <int TYPE>
__device__ __forceinline__ void store_lines(char* out, int64_t pitch, const char* piece, int columns, int rows, int lane) {
  constexpr int kSize = TYPE == S3R_F32 ? 4 : 2, kAtOnce = 4;
  using Word = std::conditional_t<kSize == 4, uint32_t, uint16_t>;
  const int j = lane & 7, bytes = columns * kSize;
  auto element = [&](int line, int byte) { return *reinterpret_cast<const Word*>(piece + swz128(line, byte >> 4) + (byte & 15)); };
  for (int i0 = 0; i0 < 8; i0 += kAtOnce) {
    uint4 inner[kAtOnce];
    Word front[kAtOnce], behind[kAtOnce];
    int skip[kAtOnce], tail[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int line = (i0 + i) * 4 + (lane >> 3);
      skip[i] = static_cast<int>(-reinterpret_cast<intptr_t>(out + line * pitch) & 15);        // where whole 16 bytes begin
      tail[i] = bytes > skip[i] ? (bytes - skip[i]) & 15 : 0;
      const uint4 a = *reinterpret_cast<const uint4*>(piece + swz128(line, j)), b = *reinterpret_cast<const uint4*>(piece + swz128(line, (j + 1) & 7));
      front[i] = element(line, j * kSize);
      behind[i] = element(line, min(bytes - tail[i] + j * kSize, 128 - kSize));
      uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      if (skip[i] & 8)
#pragma unroll
        for (int k = 0; k < 6; ++k) w[k] = w[k + 2];
      if (skip[i] & 4)
#pragma unroll
        for (int k = 0; k < 5; ++k) w[k] = w[k + 1];
      if (kSize == 2 && (skip[i] & 2))
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], 16);
      inner[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int line = (i0 + i) * 4 + (lane >> 3);
      char* to = out + line * pitch;
      if (line >= rows) continue;
      if (skip[i] + 16 * j + 16 <= bytes) *reinterpret_cast<uint4*>(to + skip[i] + 16 * j) = inner[i];
      if (j * kSize < min(skip[i], bytes)) *reinterpret_cast<Word*>(to + j * kSize) = front[i];
      if (j * kSize < tail[i]) *reinterpret_cast<Word*>(to + bytes - tail[i] + j * kSize) = behind[i];
    }
  }
}
// TYPE: of the output
template <int TN, int CTAS, int TYPE>
__global__ void __launch_bounds__(kI8Threads) int8_linear_kernel(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb,
                                                                 const __grid_constant__ CUtensorMap mo, const __grid_constant__ I8Params p) {
  using C = I8Cfg<TN, CTAS>;
  extern __shared__ char raw_smem[];
  __shared__ I8Ctl ctl;
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
      mbar_init(&ctl.acc_empty[s], CTAS * kI8Warps);
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
  const int tiles = p.m_tiles * p.n_tiles, steps = (p.K + 127) / 128, first = blockIdx.x / CTAS, stride = gridDim.x / CTAS;
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
          tma_load_2d<CTAS>(base + s * C::kBytes, &ma, bar, k * 128, m0);
          tma_load_2d<CTAS>(base + s * C::kBytes + C::kABytes, &mb, bar, k * 128, n0);
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
      constexpr uint32_t idesc = umma_idesc_i8(128 * CTAS, TN);
      const bool leader = elect_one_sync();
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
            umma_i8_k4<CTAS>(tmem + buf * TN, umma_desc_sw128(base + s * C::kBytes), umma_desc_sw128(base + s * C::kBytes + C::kABytes), idesc, k > 0);
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
    char* piece = smem + C::kOut + (warp - 2) * kI8Piece;
    const uint32_t stage = smem_u32(piece);
    // scales and biases of its columns, of this tile and the next one
    float* factors = reinterpret_cast<float*>(smem + C::kColumns) + (warp - 2) * 4 * C::kSpan;
    constexpr int per = TYPE == S3R_F32 ? 32 : 64;                 // columns of a piece
    const int from = half * C::kSpan;
    constexpr int kMine = C::kSpan / 32;
    // A lane's part of 32 rows x 32 columns: rows r, r + 8, r + 16, r + 24, of every eight columns two from c on.  With a row per lane
    // every lane would need every column's factors, and reading those (a wavefront per column and warp) kept shared memory busier
    // than the products at K = 1024 (64 512 x 4096: 248 us).
    const int r = lane >> 2, c = 2 * (lane & 3);
    float rows[4];                                                 // the next tile's row scales
    for (int i = lane; i < 4 * C::kSpan; i += 32) factors[i] = 0.f;
    __syncwarp();
    auto fetch = [&](int tile, Tile at, float* to) {
      const int64_t row = (static_cast<int64_t>(at.m) * CTAS + rank) * 128 + quarter * 32 + r;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int col = at.n * TN + from + i * 32 + lane;
        if (tile < tiles && col < p.N) {
          cp_async4(smem_u32(to + i * 32 + lane), p.b_scale + col);
          if (p.bias) cp_async4(smem_u32(to + C::kSpan + i * 32 + lane), p.bias + col);
        }
      }
      cp_async_commit();
#pragma unroll
      for (int i = 0; i < 4; ++i) rows[i] = tile < tiles && row + 8 * i < p.M ? __ldg(p.a_scale + row + 8 * i) : 0.f;
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
      float row[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) row[i] = rows[i];
      const float* columns = factors + buf * 2 * C::kSpan;
      cp_async_wait<0>();
      __syncwarp();
      advance(after);
      fetch(tile + stride, after, factors + (buf ^ 1) * 2 * C::kSpan);
      ok = mbar_wait_warp(&ctl.acc_full[buf], done >> 1 & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      // 32 columns' sums; once they are products the next 32 are asked for, under no condition, so that their registers have no other
      // writer to wait for, and are on their way while these are stored.
      const uint32_t sums = tmem + (static_cast<uint32_t>(quarter) << 21) + buf * TN + from;
      uint32_t v[32];
      if (from < TN) tmem_ld_32x32(sums, v);
#pragma unroll
      for (int g = 0; g < kMine; ++g) {
        float2 s[4], b[4], x[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[j] = *reinterpret_cast<const float2*>(columns + g * 32 + 8 * j + c);
          b[j] = *reinterpret_cast<const float2*>(columns + C::kSpan + g * 32 + 8 * j + c);
        }
        tmem_ld_wait_for(v);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = (i >> 1) * 16 + j * 4 + (i & 1) * 2;
            const float2 sum = make_float2(__int2float_rn(static_cast<int>(v[k])), __int2float_rn(static_cast<int>(v[k + 1])));
            x[j][i] = ffma2(fmul2(sum, make_float2(row[i], row[i])), s[j], b[j]);
          }
        if (g + 1 < kMine) {
          if (from < TN) tmem_ld_32x32(sums + g * 32 + 32, v);
        } else {                                                   // this warp's sums are in registers
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_first_cta<CTAS>(&ctl.acc_empty[buf]);
        }
        if (from + g * 32 < width) {
          const bool last = g + 1 == kMine || from + g * 32 + 32 >= width;
          if (per == 32 || !(g & 1)) {
            if (lane == 0) bulk_wait_read();                       // the store before has left this piece
            __syncwarp();
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            // row r + 8 i: 128 bytes, its 16-byte chunks swizzled by r
            char* to = piece + r * 128 + (TYPE == S3R_F32 ? (((2 * j + (c >> 2)) ^ r) << 4) + (c & 2) * 4 : ((((g & 1) * 4 + j) ^ r) << 4) + c * 2);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (TYPE == S3R_F32) *reinterpret_cast<float2*>(to + i * 1024) = x[j][i];
              else *reinterpret_cast<uint32_t*>(to + i * 1024) = TYPE == S3R_BF16 ? pack_bf16(x[j][i].x, x[j][i].y) : pack_half(x[j][i].x, x[j][i].y);
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
              store_lines<TYPE>(static_cast<char*>(p.out) + (m0 * p.N + n0 + c0) * type_bytes(TYPE), static_cast<int64_t>(p.N) * type_bytes(TYPE),
                                piece, min(per, width - c0), static_cast<int>(min(static_cast<int64_t>(32), p.M - m0)), lane);
              __syncwarp();                                        // read before the next piece is written
            }
          }
        }
      }
      __syncwarp();                                                // its factors are read
    }
    cp_async_wait<0>();
    if (lane == 0) bulk_wait_all();
    if (!ok && lane == 0) atomicOr(p.status, kStatusWaitTimeout);
  }
  tc_fence_before();
  __syncthreads();
  sync_pair<CTAS>();                                               // the other CTA's products and arrivals reach this one's memory
  if (warp == 1) tmem_free<CTAS>(tmem, 2 * TN);
}

template <int TN, int CTAS, int TYPE>
static int launch_int8(const int8_t* a, int64_t a_pitch, const int8_t* b, int64_t b_pitch, I8Params p, cudaStream_t st) {
  using C = I8Cfg<TN, CTAS>;
  CUtensorMap ma, mb, mo;
  {
    const uint64_t dims[2] = {static_cast<uint64_t>(p.K), static_cast<uint64_t>(p.M)}, strides[1] = {static_cast<uint64_t>(a_pitch)};
    const uint32_t box[2] = {128, 128};
    if (const int rc = make_tensor_map(&ma, a, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_DATA_TYPE_UINT8)) return rc;
  }
  {
    const uint64_t dims[2] = {static_cast<uint64_t>(p.K), static_cast<uint64_t>(p.N)}, strides[1] = {static_cast<uint64_t>(b_pitch)};
    const uint32_t box[2] = {128, TN / CTAS};
    if (const int rc = make_tensor_map(&mb, b, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_DATA_TYPE_UINT8)) return rc;
  }
  mo = ma;
  if (p.copy_out) {
    const uint64_t dims[2] = {static_cast<uint64_t>(p.N), static_cast<uint64_t>(p.M)};
    const uint64_t strides[1] = {static_cast<uint64_t>(p.N) * type_bytes(TYPE)};
    const uint32_t box[2] = {128 / type_bytes(TYPE), 32};
    const CUtensorMapDataType type = TYPE == S3R_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : TYPE == S3R_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if (const int rc = make_tensor_map(&mo, p.out, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, type)) return rc;
  }
  p.m_tiles = static_cast<int>((p.M + 128 * CTAS - 1) / (128 * CTAS));
  p.n_tiles = (p.N + TN - 1) / TN;
  const int64_t tiles = static_cast<int64_t>(p.m_tiles) * p.n_tiles, at_once = sm_count() / CTAS;
  S3R_REQUIRE(tiles < (1ll << 31) - 1024, S3R_ERR_TOO_LARGE, "s3r_int8_linear: too many tiles");
  static std::atomic<uint64_t> ready{0};
  if (attributes_missing(ready)) {
    S3R_CUDA(cudaFuncSetAttribute(int8_linear_kernel<TN, CTAS, TYPE>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    attributes_set(ready);
  }
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(static_cast<unsigned>((tiles < at_once ? tiles : at_once) * CTAS));
  c.blockDim = dim3(kI8Threads);
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
  return check_cuda(cudaLaunchKernelEx(&c, int8_linear_kernel<TN, CTAS, TYPE>, ma, mb, mo, p), "kernel launch");
}
template <int TN, int CTAS>
static int run_int8(const int8_t* a, int64_t a_pitch, const int8_t* b, int64_t b_pitch, int type, const I8Params& p, cudaStream_t st) {
  if (type == S3R_F32) return launch_int8<TN, CTAS, S3R_F32>(a, a_pitch, b, b_pitch, p, st);
  if (type == S3R_BF16) return launch_int8<TN, CTAS, S3R_BF16>(a, a_pitch, b, b_pitch, p, st);
  return launch_int8<TN, CTAS, S3R_F16>(a, a_pitch, b, b_pitch, p, st);
}

// ---------------------------------------------------------------------------------------------------------------------
// a few tokens: the weights are read once, at the rate of memory, and tensor cores would wait for tiles of them.  A warp has four output
// channels, a lane 16 bytes of each at a time; the tokens lie in shared memory.  One token x 4096 x 1024: 6.5 us on tcgen05, this way 3.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kFewTokens = 8, kFewBytes = 48 * 1024, kFewChannels = 4, kFewWarps = 8;

struct FewParams {
  const int8_t *a, *b;
  const float *a_scale, *b_scale, *bias;
  void* out;
  int64_t a_pitch, b_pitch;
  int N, K, type, M;
};

// 16 bytes from k on; what lies behind the row's end is 0 and not read
__device__ __forceinline__ uint4 load_16(const int8_t* row, int k, int K) {
  if (k + 16 <= K) return __ldg(reinterpret_cast<const uint4*>(row + k));
  uint32_t w[4] = {0, 0, 0, 0};
  for (int i = 0; k + i < K; ++i) w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(row[k + i])) << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int M>
__global__ void __launch_bounds__(32 * kFewWarps) int8_few_kernel(const __grid_constant__ FewParams p) {
  extern __shared__ __align__(16) char smem[];
  griddep_wait();
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, chunks = (p.K + 15) / 16;
  uint4* x = reinterpret_cast<uint4*>(smem);                       // [M][chunks]
  const int n0 = (blockIdx.x * kFewWarps + warp) * kFewChannels;
  // the first weights are on their way while the tokens are fetched
  uint4 w[kFewChannels];
  auto fetch = [&](int c) {
#pragma unroll
    for (int i = 0; i < kFewChannels; ++i) w[i] = n0 + i < p.N && c < chunks ? load_16(p.b + (n0 + i) * p.b_pitch, c * 16, p.K) : make_uint4(0, 0, 0, 0);
  };
  fetch(lane);
#pragma unroll
  for (int m = 0; m < M; ++m)
    for (int c = threadIdx.x; c < chunks; c += 32 * kFewWarps) x[m * chunks + c] = m < p.M ? load_16(p.a + m * p.a_pitch, c * 16, p.K) : make_uint4(0, 0, 0, 0);
  __syncthreads();
  int sum[kFewChannels][M];
#pragma unroll
  for (int i = 0; i < kFewChannels; ++i)
#pragma unroll
    for (int m = 0; m < M; ++m) sum[i][m] = 0;
  for (int c = lane; c < chunks; c += 32) {
    uint4 now[kFewChannels];
#pragma unroll
    for (int i = 0; i < kFewChannels; ++i) now[i] = w[i];
    fetch(c + 32);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const uint4 t = x[m * chunks + c];
#pragma unroll
      for (int i = 0; i < kFewChannels; ++i) {
        int s = sum[i][m];
        s = __dp4a(static_cast<int>(now[i].x), static_cast<int>(t.x), s);
        s = __dp4a(static_cast<int>(now[i].y), static_cast<int>(t.y), s);
        s = __dp4a(static_cast<int>(now[i].z), static_cast<int>(t.z), s);
        sum[i][m] = __dp4a(static_cast<int>(now[i].w), static_cast<int>(t.w), s);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kFewChannels; ++i)
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const int total = __reduce_add_sync(0xffffffffu, sum[i][m]);
      if (lane == i * M + m && m < p.M && n0 + i < p.N) {
        // the larger kernel's operations, so that a token's results do not depend on how many it comes with
        const float v[1] = {__fmaf_rn(__fmul_rn(__int2float_rn(total), __ldg(p.a_scale + m)), __ldg(p.b_scale + n0 + i), p.bias ? __ldg(p.bias + n0 + i) : 0.f)};
        Raw<1> o;
        pack<1>(o, v, p.type);
        store_raw<1>(o, p.out, p.type, static_cast<int64_t>(m) * p.N + n0 + i);
      }
    }
}

template <int M>
static int run_few(const FewParams& p, cudaStream_t st) {
  static_assert(M * kFewChannels <= 32, "a lane per result");
  const int per = kFewWarps * kFewChannels;
  return launch(int8_few_kernel<M>, static_cast<unsigned>((p.N + per - 1) / per), 32 * kFewWarps, static_cast<size_t>(M) * ((p.K + 15) / 16) * 16, st, p);
}

}  // namespace s3r

using namespace s3r;

extern "C" int s3r_quantize_rows(const void* x, int type, int64_t x_pitch, int8_t* q, int64_t q_pitch, float* scale, int64_t rows, int channels,
                                 void* stream) {
  S3R_REQUIRE(x && q && scale, S3R_ERR_NULL, "s3r_quantize_rows: NULL pointer");
  S3R_REQUIRE(rows > 0 && channels > 0 && x_pitch >= channels && q_pitch >= channels, S3R_ERR_SHAPE, "s3r_quantize_rows: sizes must be positive, pitches no shorter than rows");
  S3R_REQUIRE(known_type(type), S3R_ERR_UNSUPPORTED, "s3r_quantize_rows: types are fp32, bf16 and fp16");
  S3R_REQUIRE(rows < (1ll << 31), S3R_ERR_TOO_LARGE, "s3r_quantize_rows: too many rows");
  // a thread's next column, up to 1024 x 8 behind the last one, is an int too
  S3R_REQUIRE(channels <= INT_MAX - 8192, S3R_ERR_TOO_LARGE, "s3r_quantize_rows: %d channels (at most 2^31 - 8193)", channels);
  S3R_REQUIRE(reinterpret_cast<uintptr_t>(x) % type_bytes(type) == 0 && reinterpret_cast<uintptr_t>(scale) % 4 == 0, S3R_ERR_ALIGNMENT, "s3r_quantize_rows: elements must be aligned");
  const void* ptr[] = {x};
  int w = row_vector(channels, ptr, &type, 1);
  while (w > 1 && (x_pitch % w || (reinterpret_cast<uintptr_t>(q) | static_cast<uintptr_t>(q_pitch)) % w)) w = w == 8 ? 4 : 1;
  const QuantParams p = {x, q, scale, x_pitch, q_pitch, rows, type, channels};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return w == 8 ? pick_quantize<8>(p, st) : w == 4 ? pick_quantize<4>(p, st) : pick_quantize<1>(p, st);
}

extern "C" int s3r_pad_rows(const int8_t* src, int64_t src_pitch, int8_t* dst, int64_t dst_pitch, int64_t rows, int K, void* stream) {
  S3R_REQUIRE(src && dst, S3R_ERR_NULL, "s3r_pad_rows: NULL pointer");
  S3R_REQUIRE(rows > 0 && K > 0 && src_pitch >= 0 && dst_pitch >= K, S3R_ERR_SHAPE, "s3r_pad_rows: sizes must be positive, rows no longer than the pitch");
  S3R_REQUIRE(reinterpret_cast<uintptr_t>(dst) % 16 == 0 && dst_pitch % 16 == 0, S3R_ERR_ALIGNMENT, "s3r_pad_rows: rows must become multiples of 16 bytes");
  const int chunks = static_cast<int>((static_cast<int64_t>(K) + 15) / 16);
  const int64_t blocks = (rows * chunks + 255) / 256;
  S3R_REQUIRE(K <= 0x7fffff00 && blocks < (1ll << 31), S3R_ERR_TOO_LARGE, "s3r_pad_rows: grid too large");
  return launch(pad_rows_kernel, static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(stream), src, src_pitch, dst, dst_pitch, rows, K, chunks);
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (M <= kFewTokens && (M <= 2 ? M : M <= 4 ? 4 : 8) * ((static_cast<int64_t>(K) + 15) / 16 * 16) <= kFewBytes) {
    const FewParams f = {a, b, a_scale, b_scale, bias, out, a_pitch, b_pitch, N, K, type, static_cast<int>(M)};
    return M == 1 ? run_few<1>(f, st) : M == 2 ? run_few<2>(f, st) : M <= 4 ? run_few<4>(f, st) : run_few<8>(f, st);
  }
  I8Params p = {};
  p.a_scale = a_scale;
  p.b_scale = b_scale;
  p.bias = bias;
  p.out = out;
  p.M = M;
  p.N = N;
  p.K = K;
  p.copy_out = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && static_cast<int64_t>(N) * type_bytes(type) % 16 == 0;
  p.status = device_status_ptr();
  S3R_REQUIRE(p.status, S3R_ERR_DRIVER, "s3r_int8_linear: no status word");
  // The tile whose waves cost least: a wave of narrower tiles takes less, but not in proportion (the same rows of a).  Against the best tile of
  // each size (bf16, 16 to 33 000 tokens, N x K = 1024 x 1024, 4096 x 1024, 1024 x 4096, 3104 x 1024, 2000 x 2000, 512 x 500, 32 x 1024; 133
  // sizes) this choice takes 1 % longer in sum and 15 % at most (300 x 1024 x 4096: 12.7 us, by pairs of 128 columns 11.1); always 256 columns
  // by a pair is best from 4000 x 1024 x 1024 on and takes 16.6 instead of 12.5 us at 129 x 1024 x 4096.
  auto cost = [&](int tn, int ctas) {
    const int64_t tiles = (M + 128 * ctas - 1) / (128 * ctas) * ((N + tn - 1) / tn), at_once = sm_count() / ctas;
    return (tiles + at_once - 1) / at_once * (tn + (ctas == 2 ? 64 : 96));
  };
  const int64_t pair_256 = cost(256, 2), pair_128 = cost(128, 2), one_128 = cost(128, 1), one_64 = cost(64, 1);
  if (M > 128 && pair_256 <= pair_128 && pair_256 <= one_128 && pair_256 <= one_64) return run_int8<256, 2>(a, a_pitch, b, b_pitch, type, p, st);
  if (M > 128 && pair_128 <= one_128 && pair_128 <= one_64) return run_int8<128, 2>(a, a_pitch, b, b_pitch, type, p, st);
  if (one_128 <= one_64) return run_int8<128, 1>(a, a_pitch, b, b_pitch, type, p, st);
  return run_int8<64, 1>(a, a_pitch, b, b_pitch, type, p, st);
}
