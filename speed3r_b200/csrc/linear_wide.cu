// Products whose result is fp32.
#include "linear.cuh"

namespace s3r {

int linear_wide(const LinOperand& a, const LinOperand& b, int64_t k, bool bf16, const LinParams& p, cudaStream_t st) {
  return with_act(p.act, [&](auto act) { return run_linear<decltype(act)::value, kNoOther, true, 0>(a, b, k, bf16, p, st); });
}

}  // namespace s3r
