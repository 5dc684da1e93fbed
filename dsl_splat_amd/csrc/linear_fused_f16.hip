// The fused backward pass of products (linear_fused.hpp) for f16.
#include "linear_fused.hpp"

namespace gs3d {

template <>
void fused_launch<f16_t>(const LinearFused& a, bool q8, int blocks, hipStream_t stream) {
    if (q8) launch_fused<f16_t, true>(a, blocks, stream);
    else launch_fused<f16_t, false>(a, blocks, stream);
}

}  // namespace gs3d
