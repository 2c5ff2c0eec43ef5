// What products of tiles by pairs of CTAs share (8-bit integers, bf16 and fp16): barriers and copies of a pair, sums on their way out of tensor
// memory, and pieces of the result on their way to rows that begin anywhere.
#pragma once

#include <type_traits>

#include "rows.cuh"

#ifdef __CUDACC__
namespace s3r {

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

}  // namespace s3r
#endif  // __CUDACC__
