// What the feature-decoder kernels (linear.hip, group_norm.hip,
// quantize.hip) share: 16-byte vectors of the three element types, the
// activations and their slopes, matrix fragments, and the 8-bit form of
// activations.
//
// Element types: float, bfloat16, float16.  Everything is computed in 32
// bits; 16-bit values are converted on load and rounded once on store.
#pragma once

#include "common.hpp"

namespace gs3d {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x2 __attribute__((ext_vector_type(2)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

// Elements in 16 bytes: the width of every load, store and matrix fragment.
template <class T>
constexpr int VEC = 16 / (int)sizeof(T);

// Rows of channels start wherever the channel count puts them (33 channels of
// 2 bytes: every other row is off the 4-byte grid), so 16-byte accesses are
// declared with the element's alignment only; the device takes them as one
// instruction.
typedef u32x4 u32x4_at2 __attribute__((aligned(2), may_alias));
typedef u32x4 u32x4_at4 __attribute__((aligned(4), may_alias));
typedef u32x2 u32x2_at1 __attribute__((aligned(1), may_alias));
typedef uint32_t u32_at1 __attribute__((aligned(1), may_alias));

template <class T>
GS3D_DEV u32x4 load16(const T* p) {
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const u32x4_at4*>(p);
    else return *reinterpret_cast<const u32x4_at2*>(p);
}
template <class T>
GS3D_DEV void store16(T* p, u32x4 v) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<u32x4_at4*>(p) = v;
    else *reinterpret_cast<u32x4_at2*>(p) = v;
}

GS3D_DEV float to_f32(float v) { return v; }
GS3D_DEV float to_f32(bf16_t v) { return (float)v; }
GS3D_DEV float to_f32(f16_t v) { return (float)v; }

GS3D_DEV void unpack(u32x4 raw, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(raw[i]);
}
template <class T>
GS3D_DEV void unpack(u32x4 raw, float (&v)[8]) {
    if constexpr (__is_same(T, bf16_t)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(raw[i] << 16);
            v[2 * i + 1] = __uint_as_float(raw[i] & 0xFFFF0000u);
        }
    } else {
        const f16x8 h = __builtin_bit_cast(f16x8, raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
    }
}
template <class T>
GS3D_DEV void unpack(u32x4 raw, float (&v)[4]) {
    unpack(raw, v);
}

// Two floats to one 32-bit word of 16-bit values, round to nearest even.
template <class T>
GS3D_DEV uint32_t pack2(float a, float b) {
    if constexpr (__is_same(T, bf16_t))
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
    else
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
}
template <class T>
GS3D_DEV u32x4 pack(const float (&v)[4]) {
    return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}
template <class T>
GS3D_DEV u32x4 pack(const float (&v)[8]) {
    return u32x4{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7])};
}

// The VEC<T> elements of a row of `count` from element `at` on; those past
// the row's end are zero and never read.
template <class T>
GS3D_DEV u32x4 load_row(const T* row, int at, int count) {
    if (at + VEC<T> <= count) return load16(row + at);
    u32x4 raw = {0u, 0u, 0u, 0u};
    if (at < count) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (at + i < count) raw[i] = reinterpret_cast<const uint32_t*>(row)[at + i];
        } else {
            const uint16_t* half = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (at + i < count) raw[i / 2] |= (uint32_t)half[at + i] << (16 * (i & 1));
        }
    }
    return raw;
}

template <class T>
GS3D_DEV void store_row(T* row, int at, int count, u32x4 raw) {
    if (at + VEC<T> <= count) {
        store16(row + at, raw);
    } else if (at < count) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (at + i < count) reinterpret_cast<uint32_t*>(row)[at + i] = raw[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (at + i < count)
                    reinterpret_cast<uint16_t*>(row)[at + i] = (uint16_t)(raw[i / 2] >> (16 * (i & 1)));
        }
    }
}

// ---------------------------------------------------------------------------
// Activations (GS3D_ACT_*).  The kind is uniform over a launch.
// ---------------------------------------------------------------------------
GS3D_DEV float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

// Distribution function of the normal distribution.
GS3D_DEV float normal_below(float z) { return 0.5f + 0.5f * erff(z * 0.70710678f); }

GS3D_DEV float activate(float z, int kind) {
    if (kind == GS3D_ACT_SILU) return z * sigmoid(z);
    if (kind == GS3D_ACT_GELU) return z * normal_below(z);
    if (kind == GS3D_ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN stays
    return z;
}

// Derivative of activate at z.
GS3D_DEV float slope(float z, int kind) {
    if (kind == GS3D_ACT_SILU) {
        const float s = sigmoid(z);
        return s * __builtin_fmaf(z, 1.0f - s, 1.0f);
    }
    if (kind == GS3D_ACT_GELU) return __builtin_fmaf(z * 0.39894228f, __expf(-0.5f * z * z), normal_below(z));
    if (kind == GS3D_ACT_RELU) return z > 0.0f ? 1.0f : (z == z ? 0.0f : z);
    return 1.0f;
}

// ---------------------------------------------------------------------------
// The 8-bit form: 32 neighbouring channels of a row share a scale 2^e, stored
// as the byte e + 127; a value is the int8 code times 2^e.  e is the smallest
// with max |x| <= 127 * 2^e between -126 and TOP: past 127 * 2^TOP a code
// would stand for more than the type's largest value, so values there (the
// last percent of the type's range) keep the code 127.  A block with a value
// that is not finite has scale byte 255 and zero codes: 0 * inf reads back as
// NaN without a test.  Scales that are powers of two make the product with a
// code exact in every type (a code has 7 bits), so a matrix product or a norm
// that reads codes sees exactly the value that was kept.
// ---------------------------------------------------------------------------
constexpr int Q8_BLOCK = 32;
template <class T>
constexpr int Q8_TOP_BYTE = __is_same(T, f16_t) ? 9 + 127 : 121 + 127;

template <class T>
GS3D_DEV uint32_t q8_scale_byte(uint32_t largest_bits) {
    if (largest_bits >= 0x7F800000u) return 255u;
    // 127 = 1.1111110b * 2^6.
    const int byte = (int)(largest_bits >> 23) - 6 + ((largest_bits & 0x7FFFFFu) > 0x7E0000u ? 1 : 0);
    return byte < 1 ? 1u : byte > Q8_TOP_BYTE<T> ? (uint32_t)Q8_TOP_BYTE<T> : (uint32_t)byte;
}
GS3D_DEV float q8_scale(uint32_t byte) { return __uint_as_float(byte << 23); }
GS3D_DEV float q8_inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// Only a block at the top scale has values that reach past +-127.
GS3D_DEV int q8_code(float v, float inverse) {
    return (int)__builtin_amdgcn_fmed3f(__builtin_rintf(v * inverse), -127.0f, 127.0f);
}

// Magnitudes compare as integers, where NaN is larger than every number and
// so reaches the scale byte (the hardware's float maximum drops it).
GS3D_DEV uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

struct Q8Rows {
    const int8_t* codes;    // rows x channels
    const uint8_t* scales;  // rows x blocks of 32 channels
    int channels;
};

// The VEC<T> values of one row from channel `at` on (a multiple of VEC<T>),
// zero past the row's end.
template <class T>
GS3D_DEV u32x4 load_row_q8(const Q8Rows& q, int64_t row, int at) {
    constexpr int E = VEC<T>;
    float v[E];
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = 0.0f;
    if (at < q.channels) {
        const int8_t* p = q.codes + row * q.channels + at;
        const float scale = q8_scale(q.scales[row * ((q.channels + 31) >> 5) + (at >> 5)]);
        uint32_t word[E / 4];
        if (at + E <= q.channels) {
            if constexpr (E == 8) {
                const u32x2 w = *reinterpret_cast<const u32x2_at1*>(p);
                word[0] = w[0];
                word[1] = w[1];
            } else {
                word[0] = *reinterpret_cast<const u32_at1*>(p);
            }
        } else {
#pragma unroll
            for (int i = 0; i < E / 4; ++i) word[i] = 0u;
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (at + i < q.channels) word[i / 4] |= (uint32_t)(uint8_t)p[i] << (8 * (i & 3));
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float value = (float)(int)(int8_t)(word[i / 4] >> (8 * (i & 3))) * scale;
            v[i] = at + i < q.channels ? value : 0.0f;  // a NaN block ends with its row
        }
    }
    return pack<T>(v);
}

// ---------------------------------------------------------------------------
// Matrix fragments.  A fragment is 16 bytes a lane: lane l holds row l % 16
// and, in the contracted dimension, the VEC<T> elements from VEC<T> * (l / 16)
// on; 64 lanes hold 16 rows x CHUNK<T> elements.  multiply() adds
// A (16 x CHUNK) B (16 x CHUNK)^T to a 16 x 16 tile whose lane l holds
// column l % 16 (B's row) and rows 4 (l / 16) + 0..3 (A's).
// 16-bit types take one 16x16x32 instruction; float takes four 16x16x4 ones,
// the i-th contracting element i of every lane's four.
// ---------------------------------------------------------------------------
template <class T>
constexpr int CHUNK = 4 * VEC<T>;

template <class T>
GS3D_DEV f32x4 multiply(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (__is_same(T, bf16_t)) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    } else if constexpr (__is_same(T, f16_t)) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
        return c;
    }
}

}  // namespace gs3d
