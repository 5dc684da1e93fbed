// Per-pixel products (linear.hpp) for f32.
#include "linear.hpp"

namespace gs3d {

size_t linear_fwd_bytes_f32(int64_t rows, int K, int N) { return fwd_bytes<float>(rows, K, N); }

int linear_fwd_f32(const gs3d_linear_args& g, void* scratch, hipStream_t stream) {
    return linear_fwd<float>(g, scratch, stream);
}

int linear_bwd_f32(const gs3d_linear_bwd_args& g, char* scratch, hipStream_t stream) {
    return g.codes ? linear_bwd<float, true>(g, scratch, stream) : linear_bwd<float, false>(g, scratch, stream);
}

size_t linear_bwd_bytes_f32(int64_t rows, int K, int N, bool act, bool params, bool dx) {
    return bwd_scratch<float>(rows, K, N, act, params, dx).total;
}

}  // namespace gs3d
