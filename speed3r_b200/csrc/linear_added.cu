// Products that are added to a residual.
#include "linear.cuh"

namespace s3r {

template <int OTHER>
static int added(const LinOperand& a, const LinOperand& b, int64_t k, bool bf16, const LinParams& p, cudaStream_t st) {
  return p.out_type == S3R_F32 ? run_linear<kAnyAct, OTHER, true, 0>(a, b, k, bf16, p, st) : run_linear<kAnyAct, OTHER, false, 0>(a, b, k, bf16, p, st);
}
int linear_added(const LinOperand& a, const LinOperand& b, int64_t k, bool bf16, const LinParams& p, cudaStream_t st) {
  return p.other_type == S3R_F32 ? added<S3R_F32>(a, b, k, bf16, p, st) : p.other_type == S3R_BF16 ? added<S3R_BF16>(a, b, k, bf16, p, st) : added<S3R_F16>(a, b, k, bf16, p, st);
}

}  // namespace s3r
