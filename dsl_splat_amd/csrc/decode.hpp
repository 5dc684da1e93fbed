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

// The VEC<T> elements of a row of `count` from element `at` on, in two steps
// so that a load may be in flight while other work is done: issue_row starts
// it, finish_row makes the elements past the row's end zero.  A vector that
// would reach past the end is read from the row's last VEC<T> elements and
// shifted down, so nothing beyond the row is read.  Rows shorter than a
// vector are read element by element.
template <int UNIT_BITS>
GS3D_DEV u32x4 shift_down(u32x4 raw, int units) {
    if (units * UNIT_BITS >= 128) return u32x4{0u, 0u, 0u, 0u};
    uint64_t lo = (uint64_t)raw[1] << 32 | raw[0], hi = (uint64_t)raw[3] << 32 | raw[2];
    int bits = units * UNIT_BITS;
    if (bits >= 64) lo = hi, hi = 0u, bits -= 64;
    lo = lo >> bits | (hi << 1) << (63 - bits);
    hi >>= bits;
    return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// WIDE promises rows of at least a vector: no branch at all then, so that the
// compiler can count the loads in flight exactly.
template <class T, bool WIDE = false>
GS3D_DEV u32x4 issue_row(const T* row, int at, int count) {
    constexpr int E = VEC<T>;
    if (WIDE || count >= E) return load16(row + (at < count - E ? at : count - E));
    u32x4 raw = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int k = at + i < count ? at + i : count - 1;
        if constexpr (sizeof(T) == 4) {
            const uint32_t v = reinterpret_cast<const uint32_t*>(row)[k];
            raw[i] = at + i < count ? v : 0u;
        } else {
            const uint32_t v = reinterpret_cast<const uint16_t*>(row)[k];
            raw[i / 2] |= at + i < count ? v << (16 * (i & 1)) : 0u;
        }
    }
    return raw;
}
template <class T, bool WIDE = false>
GS3D_DEV u32x4 finish_row(u32x4 raw, int at, int count) {
    constexpr int E = VEC<T>;
    const int over = at + E - count;
    if ((WIDE || count >= E) && over > 0) return shift_down<8 * (int)sizeof(T)>(raw, over);
    return raw;
}
// finish_row for the wavefront's vectors of one chunk, from `first` on: looked
// at only where the chunk (a scalar) reaches past the row.
template <class T, bool WIDE>
GS3D_DEV u32x4 finish_chunk(u32x4 raw, int first, int at, int count) {
    if (first + 4 * VEC<T> <= count) return raw;
    return finish_row<T, WIDE>(raw, at, count);
}
template <class T>
GS3D_DEV u32x4 load_row(const T* row, int at, int count) {
    return finish_row<T>(issue_row(row, at, count), at, count);
}

// Its counterpart.  store_elements writes one by one, for an LDS row with the
// element's alignment only; `inside`: no lane's vector reaches past the row
// (looked at as a scalar).
template <class T>
GS3D_DEV void store_elements(T* row, bool inside, int at, int count, u32x4 raw) {
    constexpr int E = VEC<T>;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        if (!inside && at + i >= count) continue;
        if constexpr (E == 4) reinterpret_cast<uint32_t*>(row)[at + i] = raw[i];
        else reinterpret_cast<uint16_t*>(row)[at + i] = (uint16_t)(raw[i / 2] >> (16 * (i & 1)));
    }
}
template <class T>
GS3D_DEV void store_row(T* row, int at, int count, u32x4 raw) {
    if (at + VEC<T> <= count) store16(row + at, raw);
    else if (at < count) store_elements(row, false, at, count, raw);
}

// ---------------------------------------------------------------------------
// Activations (GS3D_ACT_*).  The kind is uniform over a launch.
// ---------------------------------------------------------------------------
// exp2 on the hardware's 1-ulp instruction; results below 2^-126 are zero.
GS3D_DEV float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }
GS3D_DEV float rcp_fast(float v) { return __builtin_amdgcn_rcpf(v); }

GS3D_DEV float sigmoid(float z) { return rcp_fast(1.0f + exp2_fast(z * -1.44269504f)); }

// Half the normal distribution's weight within |z|, Phi(|z|) - 1/2, and
// e^(-z^2/2) on the way: Abramowitz and Stegun, Handbook of Mathematical
// Functions, 7.1.26 (erfc by a polynomial in 1 / (1 + p x) times e^(-x^2),
// x = |z| / sqrt 2, absolute error 1.5e-7), with the half and the sqrt 2 folded
// into the constants.  With what follows it gelu takes 11 full-rate and two
// quarter-rate instructions, its slope 13 and two; the library's erf takes over
// 40, and the vector units bound the products that end in a gelu (1600 x 1200
// pixels, 32 to 128 channels, forward: 324 us with erf).  For 16-bit types,
// whose results round far more off.
GS3D_DEV float normal_half(float z, float& bell) {
    const float t = rcp_fast(__builtin_fmaf(__builtin_fabsf(z), 0.23164188f, 1.0f));
    bell = exp2_fast(z * z * -0.72134752f);
    float p = 0.53070271f;
    p = __builtin_fmaf(p, t, -0.72657601f);
    p = __builtin_fmaf(p, t, 0.71070687f);
    p = __builtin_fmaf(p, t, -0.14224837f);
    p = __builtin_fmaf(p, t, 0.12741480f);
    return __builtin_fmaf(p * -t, bell, 0.5f);
}

// z Phi(z) = z / 2 + |z| (Phi(|z|) - 1/2).
GS3D_DEV float gelu(float z) {
    float bell;
    const float half = normal_half(z, bell);
    return __builtin_fmaf(__builtin_fabsf(z), half, 0.5f * z);
}

// Float's: Phi(z), as exact as 32 bits hold it, and e^(-z^2/2).  Within 1 it is
// 1/2 + z Q(z^2); beyond, Phi(-|z|) = e^(-z^2/2) P(t), t = 1 / (1 + 0.28 |z|), in
// the manner of the above with a Newton step after the hardware's reciprocal
// (|z| ends at 20 there, where Phi is 0 and 1, so that it sees no infinity).
// Q and P are least squares fits to the two sides, reweighted until their
// largest errors were level: 1e-8 of Phi.  The errors of gelu and its slope, in
// norm, are 0.9 to 1.0 of those of torch's elementary operations; the form above
// has 1.4 to 2.5 of them.  1 M rows, 64 to 128 channels (us): forward 255,
// backward 620; with the form above 232 and 594.
GS3D_DEV float normal_below(float z, float& bell) {
    const float s = z * z;
    const float a = __builtin_fabsf(z) < 20.0f ? __builtin_fabsf(z) : 20.0f;
    const float d = __builtin_fmaf(a, 0.28f, 1.0f), r = rcp_fast(d);
    const float t = __builtin_fmaf(r, __builtin_fmaf(-d, r, 1.0f), r);
    bell = exp2_fast(s * -0.72134752f);
    float p = -0.10580869f;
    p = __builtin_fmaf(p, t, 0.3898759f);
    p = __builtin_fmaf(p, t, -0.23699655f);
    p = __builtin_fmaf(p, t, 0.26891267f);
    p = __builtin_fmaf(p, t, 0.06749573f);
    p = __builtin_fmaf(p, t, 0.11652094f);
    const float tail = p * t * bell;
    float q = 9.246849e-05f;
    q = __builtin_fmaf(q, s, -0.001165351f);
    q = __builtin_fmaf(q, s, 0.009964167f);
    q = __builtin_fmaf(q, s, -0.06648873f);
    q = __builtin_fmaf(q, s, 0.3989422f);
    if (a < 1.0f) return __builtin_fmaf(z, q, 0.5f);
    return z > 0.0f ? 1.0f - tail : tail;
}

template <class T, int KIND>
GS3D_DEV float activate_as(float z) {
    if constexpr (KIND == GS3D_ACT_SILU) return z * sigmoid(z);
    if constexpr (KIND == GS3D_ACT_GELU) {
        float bell;
        return sizeof(T) == 4 ? z * normal_below(z, bell) : gelu(z);
    }
    if constexpr (KIND == GS3D_ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN stays
    return z;
}

// Derivative of activate_as at z.
template <class T, int KIND>
GS3D_DEV float slope_as(float z) {
    if constexpr (KIND == GS3D_ACT_SILU) {
        const float s = sigmoid(z);
        return s * __builtin_fmaf(z, 1.0f - s, 1.0f);
    }
    if constexpr (KIND == GS3D_ACT_GELU) {
        float bell;
        if constexpr (sizeof(T) == 4) {
            const float below = normal_below(z, bell);
            return __builtin_fmaf(z * 0.39894228f, bell, below);
        }
        const float half = normal_half(z, bell);
        return __builtin_fmaf(z * 0.39894228f, bell, 0.5f) + __builtin_copysignf(half, z);
    }
    if constexpr (KIND == GS3D_ACT_RELU) return z > 0.0f ? 1.0f : (z == z ? 0.0f : z);
    return 1.0f;
}

// A vector at a time, the (uniform) kind looked at once.
template <class T, int E>
GS3D_DEV void activate(float (&z)[E], int kind) {
    if (kind == GS3D_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < E; ++i) z[i] = activate_as<T, GS3D_ACT_SILU>(z[i]);
    } else if (kind == GS3D_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < E; ++i) z[i] = activate_as<T, GS3D_ACT_GELU>(z[i]);
    } else if (kind == GS3D_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < E; ++i) z[i] = activate_as<T, GS3D_ACT_RELU>(z[i]);
    }
}
// g[i] *= slope at z[i].
template <class T, int E>
GS3D_DEV void pull_back(float (&g)[E], const float (&z)[E], int kind) {
    if (kind == GS3D_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < E; ++i) g[i] *= slope_as<T, GS3D_ACT_SILU>(z[i]);
    } else if (kind == GS3D_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < E; ++i) g[i] *= slope_as<T, GS3D_ACT_GELU>(z[i]);
    } else if (kind == GS3D_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < E; ++i) g[i] *= slope_as<T, GS3D_ACT_RELU>(z[i]);
    }
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

// Largest of the magnitudes in the lanes that share a block: a quad, or with
// LANES = 8 two quads.  They all must be active.
template <int LANES>
GS3D_DEV uint32_t q8_block_max(uint32_t v) {
    uint32_t o = dpp_u<0xB1>(v);  // quad_perm [1,0,3,2]
    v = v > o ? v : o;
    o = dpp_u<0x4E>(v);  // quad_perm [2,3,0,1]
    v = v > o ? v : o;
    if constexpr (LANES == 8) {
        o = dpp_u<0x141>(v);  // row_half_mirror: the other quad of the eight
        v = v > o ? v : o;
    }
    return v;
}

// Four codes as a word.
GS3D_DEV uint32_t q8_word(const float* v, uint32_t byte) {
    uint32_t word = 0u;
    if (byte != 255u) {
        const float inverse = q8_inverse_scale(byte);
#pragma unroll
        for (int i = 0; i < 4; ++i) word |= ((uint32_t)q8_code(v[i], inverse) & 0xFFu) << (8 * i);
    }
    return word;
}

// Codes from `at` on of a row of `count`: N words of four.
template <int N>
GS3D_DEV void q8_store(int8_t* row, int at, int count, const uint32_t (&words)[N]) {
    if (at + 4 * N <= count) {
        if constexpr (N == 2) *reinterpret_cast<u32x2_at1*>(row + at) = u32x2{words[0], words[1]};
        else *reinterpret_cast<u32_at1*>(row + at) = words[0];
    } else {
#pragma unroll
        for (int i = 0; i < 4 * N; ++i)
            if (at + i < count) row[at + i] = (int8_t)(words[i / 4] >> (8 * (i & 3)));
    }
}

// One lane's vector of a row written in 8 bits, from channel `at` on; LANES
// neighbouring lanes, all active, hold a block (32 / VEC<T> with zeros past the
// row's end, or fewer that cover all of a row).  `live`: the row is there.
template <class T, int LANES = 32 / VEC<T>>
GS3D_DEV void q8_keep(const float (&v)[VEC<T>], int8_t* codes, uint8_t* scales, int64_t row, int at, int channels,
                      bool live) {
    constexpr int E = VEC<T>;
    uint32_t largest = 0u;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const uint32_t m = magnitude_bits(v[i]);
        largest = m > largest ? m : largest;
    }
    const uint32_t byte = q8_scale_byte<T>(q8_block_max<LANES>(largest));
    uint32_t words[E / 4];
#pragma unroll
    for (int i = 0; i < E / 4; ++i) words[i] = q8_word(v + 4 * i, byte);
    if (!live || at >= channels) return;
    q8_store(codes + row * channels, at, channels, words);
    if ((at & 31) == 0) scales[row * ((channels + 31) >> 5) + (at >> 5)] = (uint8_t)byte;
}

// Rows of a strided tensor in 8 bits, a launch of its own (quantize.hip).
void quantize_rows(const void* x, int64_t ldx, int64_t rows, int channels, int dtype, int8_t* codes, uint8_t* scales,
                   hipStream_t stream);

struct Q8Rows {
    const int8_t* codes;    // rows x channels
    const uint8_t* scales;  // rows x blocks of 32 channels
    int channels;
};

// The VEC<T> values of one row from channel `at` on (a multiple of VEC<T>),
// zero past the row's end, in the same two steps.
struct Q8Raw {
    uint64_t codes;
    uint32_t scale;
};

template <class T, bool WIDE = false>
GS3D_DEV Q8Raw issue_row_q8(const Q8Rows& q, int64_t row, int at) {
    constexpr int E = VEC<T>;
    const int8_t* p = q.codes + row * q.channels;
    Q8Raw raw = {0u, 0u};
    const int block = (at < q.channels ? at : q.channels - 1) >> 5;
    raw.scale = q.scales[row * ((q.channels + 31) >> 5) + block];
    if (WIDE || q.channels >= E) {
        p += at < q.channels - E ? at : q.channels - E;
        if constexpr (E == 8) {
            const u32x2 w = *reinterpret_cast<const u32x2_at1*>(p);
            raw.codes = (uint64_t)w[1] << 32 | w[0];
        } else {
            raw.codes = *reinterpret_cast<const u32_at1*>(p);
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const uint32_t v = (uint8_t)p[at + i < q.channels ? at + i : q.channels - 1];
            raw.codes |= (uint64_t)(at + i < q.channels ? v : 0u) << (8 * i);
        }
    }
    return raw;
}

// An element past the row's end is zero also where the row ends in a block
// that reads back as NaN.  `inside`: the caller knows that no lane reaches
// past the end.
template <class T, bool WIDE = false>
GS3D_DEV u32x4 finish_row_q8(Q8Raw raw, int at, int channels, bool inside = false) {
    constexpr int E = VEC<T>;
    const int over = at + E - channels;
    if (!inside && (WIDE || channels >= E) && over > 0) raw.codes = over >= E ? 0u : raw.codes >> (8 * over);
    const float scale = q8_scale(raw.scale);
    const uint32_t words[2] = {(uint32_t)raw.codes, (uint32_t)(raw.codes >> 32)};
    float v[E];
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = (float)(int)(int8_t)(words[i / 4] >> (8 * (i & 3))) * scale;
    if (!inside && over > 0) {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = at + i < channels ? v[i] : 0.0f;
    }
    return pack<T>(v);
}
template <class T>
GS3D_DEV u32x4 load_row_q8(const Q8Rows& q, int64_t row, int at) {
    return finish_row_q8<T>(issue_row_q8<T>(q, row, at), at, q.channels);
}

// Rows of activations, plain or in 8 bits, behind one pair of steps.
struct Rows {
    const void* x;
    int64_t ldx;
    Q8Rows q8;
    int channels;
};
template <class T, bool Q8, bool WIDE = false>
struct RowRaw {
    u32x4 raw;
    GS3D_DEV void issue(const Rows& a, int64_t row, int at) {
        raw = issue_row<T, WIDE>(static_cast<const T*>(a.x) + row * a.ldx, at, a.channels);
    }
    GS3D_DEV u32x4 finish(const Rows& a, int at) const { return finish_row<T, WIDE>(raw, at, a.channels); }
    // `inside`: no lane's vector reaches past the row (looked at as a scalar).
    GS3D_DEV u32x4 finish_in(const Rows& a, bool inside, int at) const {
        return inside ? raw : finish_row<T, WIDE>(raw, at, a.channels);
    }
};
template <class T, bool WIDE>
struct RowRaw<T, true, WIDE> {
    Q8Raw raw;
    GS3D_DEV void issue(const Rows& a, int64_t row, int at) { raw = issue_row_q8<T, WIDE>(a.q8, row, at); }
    GS3D_DEV u32x4 finish(const Rows& a, int at) const { return finish_row_q8<T, WIDE>(raw, at, a.channels); }
    GS3D_DEV u32x4 finish_in(const Rows& a, bool inside, int at) const {
        return finish_row_q8<T, WIDE>(raw, at, a.channels, inside);
    }
};

// store_row for the wavefront's vectors of one chunk from `first` on.
template <class T>
GS3D_DEV void store_chunk(T* row, int first, int at, int count, u32x4 raw) {
    if (first + 4 * VEC<T> <= count) store16(row + at, raw);
    else store_row(row, at, count, raw);
}

// The block's wavefront as a scalar: what hangs on it branches and addresses as
// scalars do.
GS3D_DEV int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// ---------------------------------------------------------------------------
// A gradient dz = dy act'(z) is computed in 32 bits and then an operand of two
// matrix products.  Rounded once to 16 bits it makes the error of dx 1.41
// times, that of dW and db 1.34 to 1.53 times what rounding the results alone
// gives.  Both products take dz as two 16-bit values, high and low, and are
// then as exact as their own rounding (float16's grid of 2^-24 ends both).  The
// backward of 1.92 M rows of bfloat16, 128 to 128 channels from 8 bits, takes 387
// us with one value, 498 with the low one in dW and 505 to 519 with it in both.
// Float, and dy itself where there is no activation, are one value.
// ---------------------------------------------------------------------------
template <class T>
constexpr bool SPLIT = sizeof(T) == 2;

// The vector's high halves; v keeps what they leave.  A slope (1.13 at most)
// can take a float16 gradient past the type's range: the high half then is its
// largest value and the low one has the rest, which of an infinity or a NaN is
// itself.  bfloat16's high half is infinite with its value, the low one zero.
template <class T>
GS3D_DEV u32x4 take_high(float (&v)[VEC<T>]) {
    if constexpr (__is_same(T, f16_t)) {
        float top[VEC<T>], h[VEC<T>];
#pragma unroll
        for (int i = 0; i < VEC<T>; ++i) top[i] = __builtin_amdgcn_fmed3f(v[i], -65504.0f, 65504.0f);
        const u32x4 high = pack<T>(top);
        unpack<T>(high, h);
#pragma unroll
        for (int i = 0; i < VEC<T>; ++i) v[i] -= h[i];
        return high;
    }
    const u32x4 high = pack<T>(v);
    float h[VEC<T>];
    unpack<T>(high, h);
#pragma unroll
    for (int i = 0; i < VEC<T>; ++i) v[i] = __builtin_isinf(h[i]) ? 0.0f : v[i] - h[i];
    return high;
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

// Results of matrix instructions are not interlocked: a read needs 8 wait
// states after a 16-bit instruction and 11 after a float one.  The compiler
// counts them, but over an `if` between the two it can take the longer way
// only (seen in the listing of a strip with a residual: its last element was
// read two states after).  settle() ends a run of matrix instructions in the
// block that they are in, before any branch on the way to their use.
template <int N>
GS3D_DEV void settle(f32x4 (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(v[i]));  // all of them before the wait
    asm volatile("s_nop 11" : "+v"(v[0]));
#pragma unroll
    for (int i = 1; i < N; ++i) asm volatile("" : "+v"(v[i]));  // and their uses after it
}

// multiply() for a chunk of which only the first `valid` elements count (the
// rest are zero), `valid` the same in the whole wavefront.  Float skips the
// instructions that would contract zeros only: matrix instructions bound its
// products, and 33 channels are then 36 and not 48.  It branches, so it
// settles (12 cycles after 32 to 128).
template <class T>
GS3D_DEV f32x4 multiply_chunk(u32x4 a, u32x4 b, f32x4 c, int valid) {
    if constexpr (sizeof(T) == 4) {
        f32x4 v[1] = {c};
        if (valid >= 4) {
            v[0] = multiply<T>(a, b, v[0]);
            settle(v);
        } else if (valid > 0) {
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                if (i < valid) {
                    v[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), v[0], 0,
                                                                0, 0);
                    settle(v);
                }
            }
        }
        return v[0];
    }
    return multiply<T>(a, b, c);
}

// Column of row r of tile t in an operand whose rows become an output's
// columns.  A lane ends up with rows 4q..4q+3 of every tile; for 16-bit types
// two tiles are dealt out so that their eight values are neighbours, 16 bytes
// of an output row.
template <class T>
GS3D_DEV int tile_column(int t, int r) {
    if constexpr (sizeof(T) == 4) return 16 * t + r;
    return 32 * (t >> 1) + 8 * (r >> 2) + 4 * (t & 1) + (r & 3);
}

// Fragment of the transpose of a row-major LDS tile (`pitch` 16-byte units a
// row): lane l gets one column of 16 and the VEC<T> rows from
// row0 + VEC<T> (l / 16) on.  DEALT columns are tile_column's, else 16 t + r.
// 16-bit types use the transposing LDS read, of which 16 lanes fetch four rows
// of 16 columns (lane s the four columns 4 (s % 4).. of row s / 4, from any
// address) and lane i receives column i of the four rows; float reads words.
typedef short i16x4 __attribute__((ext_vector_type(4)));
template <class T, bool DEALT>
GS3D_DEV u32x4 read_transposed(const u32x4* tile, int pitch, int row0, int t, int lane) {
    const int s = lane & 15, q = lane >> 4;
    if constexpr (sizeof(T) == 4) {
        const uint32_t* p = reinterpret_cast<const uint32_t*>(tile) + (row0 + 4 * q) * pitch * 4 + 16 * t + s;
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = p[i * pitch * 4];
        return v;
    } else {
        const int column = DEALT ? 32 * (t >> 1) + 4 * (t & 1) + 8 * (s & 3) : 16 * t + 4 * (s & 3);
        const uint16_t* p = reinterpret_cast<const uint16_t*>(tile) + (row0 + 8 * q + (s >> 2)) * pitch * 8 + column;
        typedef __attribute__((address_space(3))) i16x4* lds_ptr;
        const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p);
        const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 4 * pitch * 8));
        const u32x2 lo = __builtin_bit_cast(u32x2, a), hi = __builtin_bit_cast(u32x2, b);
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
}

}  // namespace gs3d
