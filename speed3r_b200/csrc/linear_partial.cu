// Products whose contraction is cut into parts: fp32 sums of each.
#include "linear.cuh"

namespace s3r {

int linear_partial(const LinOperand& a, const LinOperand& b, int64_t k, bool bf16, const LinParams& p, cudaStream_t st) {
  return run_linear<kPartial, kNoOther, true, 0>(a, b, k, bf16, p, st);
}

}  // namespace s3r
