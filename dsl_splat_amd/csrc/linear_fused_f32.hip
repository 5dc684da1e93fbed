// The fused backward pass of products (linear_fused.hpp) for f32.
#include "linear_fused.hpp"

namespace gs3d {

template <>
void fused_launch<float>(const LinearFused& a, bool q8, int blocks, hipStream_t stream) {
    if (q8) launch_fused<float, true>(a, blocks, stream);
    else launch_fused<float, false>(a, blocks, stream);
}

}  // namespace gs3d
