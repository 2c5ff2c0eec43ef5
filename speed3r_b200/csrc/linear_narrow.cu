// Products whose result is bf16 or fp16.
#include "linear.cuh"

namespace s3r {

int linear_narrow(const LinOperand& a, const LinOperand& b, int64_t k, bool bf16, const LinParams& p, cudaStream_t st) {
  return with_act(p.act, [&](auto act) { return run_linear<decltype(act)::value, kNoOther, false, 0>(a, b, k, bf16, p, st); });
}

}  // namespace s3r
