// Per-pixel products (linear.hpp) for f16.
#include "linear.hpp"

namespace gs3d {

size_t linear_fwd_bytes_f16(int64_t rows, int K, int N) { return fwd_bytes<f16_t>(rows, K, N); }

int linear_fwd_f16(const gs3d_linear_args& g, void* scratch, hipStream_t stream) {
    return linear_fwd<f16_t>(g, scratch, stream);
}

int linear_bwd_f16(const gs3d_linear_bwd_args& g, char* scratch, hipStream_t stream) {
    return g.codes ? linear_bwd<f16_t, true>(g, scratch, stream) : linear_bwd<f16_t, false>(g, scratch, stream);
}

size_t linear_bwd_bytes_f16(int64_t rows, int K, int N, bool act, bool params, bool dx) {
    return bwd_scratch<f16_t>(rows, K, N, act, params, dx).total;
}

}  // namespace gs3d
