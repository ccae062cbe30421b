// The argument rules of csrc/gx_checks.h behind C entry points, for CPU tests.
#include "../gyro-dx_b200/csrc/gx_checks.h"

extern "C" {
int chk_linear(uint32_t rows, uint32_t cols, const void *x, uint32_t xd, uint64_t xs, uint32_t n, const void *y,
               uint32_t yd, uint64_t ys) {
    return gx::linear_args_ok(rows, cols, x, xd, xs, n, y, yd, ys);
}
int chk_norm(const gx_norm_desc *d, uint32_t n) { return gx::norm_args_ok(*d, n); }
int chk_residual(const gx_residual_desc *d, uint32_t n) { return gx::residual_args_ok(*d, n); }
int chk_logprobs(const gx_logprobs_desc *d, uint32_t n) { return gx::logprobs_args_ok(*d, n); }
int chk_norms(const gx_norms_desc *d) { return gx::norms_args_ok(*d); }
}
