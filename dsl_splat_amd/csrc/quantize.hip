// Activations in 8 bits and back (the form is described in decode.hpp).
//
// Four lanes share a block of 32 channels, eight channels a lane: the block's
// largest magnitude takes two exchanges inside the quad, and each lane writes
// its eight codes at once.  Both directions stream: one read, one write, no
// reuse, so HBM bounds them: 1.92 M rows of 128 bfloat16 151 us one way, 120
// back (4.9 and 6.2 TB/s).
#include "decode.hpp"

namespace gs3d {

// Eight elements from `at` on as floats, zero past the row's end.
template <class T>
GS3D_DEV void load8(const T* row, int at, int count, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        float lo[4], hi[4];
        unpack(load_row(row, at, count), lo);
        unpack(load_row(row, at + 4, count), hi);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
    } else {
        unpack<T>(load_row(row, at, count), v);
    }
}

template <class T>
__global__ __launch_bounds__(256) void quantize_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int channels,
                                                       int8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const int blocks = (channels + 31) >> 5;
    const int64_t total = rows * blocks * 4;
    const int64_t step = (int64_t)gridDim.x * 256;
    // A whole wavefront runs the loop together (the quads exchange maxima).
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i - (threadIdx.x & 63) < total; i += step) {
        const bool live = i < total;
        const int64_t unit = (live ? i : total - 1) >> 2;
        const int64_t row = unit / blocks;
        const int block = (int)(unit - row * blocks);
        const int at = 32 * block + 8 * (int)(i & 3);
        float v[8];
        load8(x + row * ldx, at, channels, v);
        uint32_t largest = 0u;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t m = magnitude_bits(v[k]);
            largest = m > largest ? m : largest;
        }
        const uint32_t byte = q8_scale_byte<T>(q8_block_max<4>(largest));
        const uint32_t words[2] = {q8_word(v, byte), q8_word(v + 4, byte)};
        if (live) {
            q8_store(codes + row * channels, at, channels, words);
            if ((i & 3) == 0) scales[unit] = (uint8_t)byte;
        }
    }
}

template <class T>
__global__ __launch_bounds__(256) void dequantize_kernel(Q8Rows q, int64_t rows, T* __restrict__ out) {
    constexpr int E = VEC<T>;
    const int vectors = (q.channels + E - 1) / E;
    const int64_t total = rows * vectors;
    const int64_t step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
        const int64_t row = i / vectors;
        const int at = E * (int)(i - row * vectors);
        store_row(out + row * q.channels, at, q.channels, load_row_q8<T>(q, row, at));
    }
}

template <class T>
static void launch_quantize(const void* x, int64_t ldx, int64_t rows, int channels, int8_t* codes, uint8_t* scales,
                            hipStream_t stream) {
    const int64_t lanes = rows * ((channels + 31) / 32) * 4;
    const int64_t blocks = (lanes + 255) / 256;
    hipLaunchKernelGGL(quantize_kernel<T>, dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, stream,
                       static_cast<const T*>(x), ldx, rows, channels, codes, scales);
}

template <class T>
static void launch_dequantize(const Q8Rows& q, int64_t rows, void* out, hipStream_t stream) {
    const int64_t lanes = rows * ((q.channels + VEC<T> - 1) / VEC<T>);
    const int64_t blocks = (lanes + 255) / 256;
    hipLaunchKernelGGL(dequantize_kernel<T>, dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, stream,
                       q, rows, static_cast<T*>(out));
}

void quantize_rows(const void* x, int64_t ldx, int64_t rows, int channels, int dtype, int8_t* codes, uint8_t* scales,
                   hipStream_t stream) {
    if (dtype == GS3D_F32) launch_quantize<float>(x, ldx, rows, channels, codes, scales, stream);
    if (dtype == GS3D_BF16) launch_quantize<bf16_t>(x, ldx, rows, channels, codes, scales, stream);
    if (dtype == GS3D_F16) launch_quantize<f16_t>(x, ldx, rows, channels, codes, scales, stream);
}

}  // namespace gs3d

extern "C" int gs3d_quantize_activations(const void* x, int64_t x_stride, int64_t rows, int32_t channels, int32_t dtype,
                                         int8_t* codes, uint8_t* scales, void* stream) {
    if (rows < 0 || channels < 1 || x_stride < channels || dtype < 0 || dtype > 2) return GS3D_ERR_ARGUMENT;
    if (rows == 0) return GS3D_OK;
    if (!x || !codes || !scales) return GS3D_ERR_ARGUMENT;
    gs3d::quantize_rows(x, x_stride, rows, channels, dtype, codes, scales, gs3d::as_stream(stream));
    return gs3d::launch_status("gs3d_quantize_activations");
}

extern "C" int gs3d_dequantize_activations(const int8_t* codes, const uint8_t* scales, int64_t rows, int32_t channels,
                                           int32_t dtype, void* out, void* stream) {
    if (rows < 0 || channels < 1 || dtype < 0 || dtype > 2) return GS3D_ERR_ARGUMENT;
    if (rows == 0) return GS3D_OK;
    if (!out || !codes || !scales) return GS3D_ERR_ARGUMENT;
    const gs3d::Q8Rows q{codes, scales, channels};
    const hipStream_t s = gs3d::as_stream(stream);
    if (dtype == GS3D_F32) gs3d::launch_dequantize<float>(q, rows, out, s);
    if (dtype == GS3D_BF16) gs3d::launch_dequantize<gs3d::bf16_t>(q, rows, out, s);
    if (dtype == GS3D_F16) gs3d::launch_dequantize<gs3d::f16_t>(q, rows, out, s);
    return gs3d::launch_status("gs3d_dequantize_activations");
}
