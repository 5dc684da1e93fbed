// C entry points of the per-pixel products (linear.hpp).
#include "common.hpp"

namespace gs3d {

// Defined by linear_f32.hip, linear_bf16.hip, linear_f16.hip.
size_t linear_fwd_bytes_f32(int64_t rows, int K, int N);
int linear_fwd_f32(const gs3d_linear_args& g, void* scratch, hipStream_t stream);
size_t linear_fwd_bytes_bf16(int64_t rows, int K, int N);
int linear_fwd_bf16(const gs3d_linear_args& g, void* scratch, hipStream_t stream);
size_t linear_fwd_bytes_f16(int64_t rows, int K, int N);
int linear_fwd_f16(const gs3d_linear_args& g, void* scratch, hipStream_t stream);
int linear_bwd_f32(const gs3d_linear_bwd_args& g, char* scratch, hipStream_t stream);
int linear_bwd_bf16(const gs3d_linear_bwd_args& g, char* scratch, hipStream_t stream);
int linear_bwd_f16(const gs3d_linear_bwd_args& g, char* scratch, hipStream_t stream);
size_t linear_bwd_bytes_f32(int64_t rows, int K, int N, bool act, bool params, bool dx);
size_t linear_bwd_bytes_bf16(int64_t rows, int K, int N, bool act, bool params, bool dx);
size_t linear_bwd_bytes_f16(int64_t rows, int K, int N, bool act, bool params, bool dx);

static bool linear_sizes_ok(int64_t rows, int K, int N, int dtype, int activation) {
    return rows >= 0 && rows <= GS3D_MAX_ROWS && K >= 1 && N >= 1 && K <= GS3D_MAX_CHANNELS &&
           N <= GS3D_MAX_CHANNELS && dtype >= 0 && dtype <= 2 && activation >= 0 && activation <= 3;
}

static size_t linear_bwd_bytes(int64_t rows, int K, int N, int dtype, bool act, bool params, bool dx) {
    if (dtype == GS3D_F32) return linear_bwd_bytes_f32(rows, K, N, act, params, dx);
    return dtype == GS3D_BF16 ? linear_bwd_bytes_bf16(rows, K, N, act, params, dx)
                              : linear_bwd_bytes_f16(rows, K, N, act, params, dx);
}

}  // namespace gs3d

extern "C" size_t gs3d_linear_fwd_scratch_bytes(int64_t rows, int32_t inner, int32_t outer, int32_t dtype) {
    if (!gs3d::linear_sizes_ok(rows, inner, outer, dtype, 0)) return 0;
    if (dtype == GS3D_F32) return gs3d::linear_fwd_bytes_f32(rows, inner, outer);
    return dtype == GS3D_BF16 ? gs3d::linear_fwd_bytes_bf16(rows, inner, outer)
                              : gs3d::linear_fwd_bytes_f16(rows, inner, outer);
}

extern "C" int gs3d_linear_fwd(const gs3d_linear_args* g, void* scratch, size_t scratch_bytes, void* stream) {
    if (!g || !gs3d::linear_sizes_ok(g->rows, g->inner, g->outer, g->dtype, g->activation)) return GS3D_ERR_ARGUMENT;
    if (g->x_stride < g->inner || (g->residual && g->residual_stride < g->outer)) return GS3D_ERR_ARGUMENT;
    if (g->rows == 0) return GS3D_OK;
    if (!g->x || !g->weight || !g->y || !g->codes != !g->scales) return GS3D_ERR_ARGUMENT;
    const size_t needed = gs3d_linear_fwd_scratch_bytes(g->rows, g->inner, g->outer, g->dtype);
    if (needed > 0 && (!scratch || scratch_bytes < needed)) return GS3D_ERR_SCRATCH;
    const hipStream_t s = gs3d::as_stream(stream);
    if (g->dtype == GS3D_F32) return gs3d::linear_fwd_f32(*g, scratch, s);
    return g->dtype == GS3D_BF16 ? gs3d::linear_fwd_bf16(*g, scratch, s) : gs3d::linear_fwd_f16(*g, scratch, s);
}

extern "C" size_t gs3d_linear_bwd_scratch_bytes(int64_t rows, int32_t inner, int32_t outer, int32_t dtype) {
    if (!gs3d::linear_sizes_ok(rows, inner, outer, dtype, 0)) return 0;
    return gs3d::linear_bwd_bytes(rows, inner, outer, dtype, true, true, true);
}

extern "C" size_t gs3d_linear_bwd_call_scratch_bytes(const gs3d_linear_bwd_args* g) {
    if (!g || !gs3d::linear_sizes_ok(g->rows, g->inner, g->outer, g->dtype, g->activation) || g->rows == 0) return 0;
    return gs3d::linear_bwd_bytes(g->rows, g->inner, g->outer, g->dtype, g->activation != GS3D_ACT_NONE,
                                  g->grad_weight || g->grad_bias, g->grad_x != nullptr);
}

extern "C" int gs3d_linear_bwd(const gs3d_linear_bwd_args* g, void* scratch, size_t scratch_bytes, void* stream) {
    if (!g || !gs3d::linear_sizes_ok(g->rows, g->inner, g->outer, g->dtype, g->activation)) return GS3D_ERR_ARGUMENT;
    const bool q8 = g->codes != nullptr;
    if (q8 != (g->scales != nullptr) || (q8 && g->x)) return GS3D_ERR_ARGUMENT;
    const bool sees_input = g->grad_weight || g->activation != GS3D_ACT_NONE;
    if (g->rows > 0 && (!g->weight || !g->upstream || g->upstream_stride < g->outer ||
                        (sees_input && !q8 && (!g->x || g->x_stride < g->inner))))
        return GS3D_ERR_ARGUMENT;
    const size_t needed = gs3d_linear_bwd_call_scratch_bytes(g);
    if (needed > 0 && (!scratch || scratch_bytes < needed)) return GS3D_ERR_SCRATCH;
    const hipStream_t s = gs3d::as_stream(stream);
    char* p = static_cast<char*>(scratch);
    if (g->dtype == GS3D_F32) return gs3d::linear_bwd_f32(*g, p, s);
    return g->dtype == GS3D_BF16 ? gs3d::linear_bwd_bf16(*g, p, s) : gs3d::linear_bwd_f16(*g, p, s);
}
