// Products that are made again in the backward: dz from dy, and sums over rows.
#include "linear.cuh"

namespace s3r {

template <int OTHER>
static int dz(const LinOperand& a, const LinOperand& b, int64_t k, bool bf16, const LinParams& p, cudaStream_t st) {
  return with_act(p.act, [&](auto act) {
    return p.scale ? run_linear<decltype(act)::value, OTHER, false, 2>(a, b, k, bf16, p, st) : run_linear<decltype(act)::value, OTHER, false, 1>(a, b, k, bf16, p, st);
  });
}
int linear_dz(const LinOperand& a, const LinOperand& b, int64_t k, bool bf16, const LinParams& p, cudaStream_t st) {
  return p.other_type == S3R_F32 ? dz<S3R_F32>(a, b, k, bf16, p, st) : p.other_type == S3R_BF16 ? dz<S3R_BF16>(a, b, k, bf16, p, st) : dz<S3R_F16>(a, b, k, bf16, p, st);
}

}  // namespace s3r
