// The backward pass of a product in one pass over its rows: z again, dz, dx
// and the weight's and bias's gradients, with dz never in memory.  Included by
// linear_fused_*.hip, one per element type.
#pragma once

#include "decode.hpp"

namespace gs3d {

struct LinearFused {
    Rows x;
    const void* w;     // N x K
    const void* bias;  // N or NULL
    const void* dy;
    int64_t ldy;
    void* dx;          // rows x K, or NULL
    float* part;       // blocks x (N K + N): the blocks' shares of dW and db, or NULL
    int64_t rows, rows_per_block;
    int K, N, act;
};

template <bool V>
struct Flag {
    static constexpr bool value = V;
};

// Wavefronts a SIMD: four where the registers do without scratch memory (128 x
// 128 of bfloat16 at four: 681 us for the case below).
template <class T, int KCH, int NCH>
constexpr int fused_waves() {
    return KCH == 8 || KCH * NCH >= (sizeof(T) == 4 ? 32 : 16) ? 2 : 4;
}

// A block of 8 wavefronts takes 64 rows at a time, KCH chunks of K and NCH of
// N wide, over a range of rows of its own.
//
// First dz.  Wavefronts s and s + 4 take rows 16 s..16 s + 15, every other
// chunk of N each: lane l holds row l % 16 and the elements from VEC (l / 16)
// on of a chunk, of x as of dy.  With W's rows as the first operand, z comes
// out with that row in that lane and, W's rows dealt out as tile_column says,
// with dy's elements beside it, so dz = dy act'(z) is whole vectors of a row.
// dz and x go to LDS, row by row.
//
// Then dx = dz W and dW = dz^T x.  dx takes dz from LDS as it lies and W
// transposed (W is in LDS once, row by row), every other chunk of K a
// wavefront.  dW contracts over rows: both operands are read transposed, and
// each wavefront's share of its tiles (4 x 2) stays in its registers over all
// the block's rows.
//
// Bytes bound it where K and N are small (x and dy in, dx out).  The next 64
// rows are loaded as soon as these are used; two blocks, 16 wavefronts, share a
// compute unit where their LDS fits, so one block's loads and slopes run under
// the other's products.  With 4 wavefronts a block, each with a quarter of dW
// and its rows' whole dz in registers, half as many fit (1600 x 1200 x 128 to
// 128 channels of bfloat16: 426 us; float 33 to 97, three such images of 801 x
// 601: 962 us with one wavefront a SIMD).
template <class T, bool Q8, int KCH, int NCH, bool WIDE>
__global__ __launch_bounds__(512, (fused_waves<T, KCH, NCH>())) void linear_bwd_fused_kernel(LinearFused a) {
    constexpr int E = VEC<T>;
    constexpr int KC = CHUNK<T>;
    constexpr int TG = KC / 16;  // tiles a chunk
    constexpr int KT = KCH * TG, NT = NCH * TG;
    constexpr int WN = 4, WK = 2;
    constexpr int TN = (NT + WN - 1) / WN, TK = KT / WK;
    constexpr int HN = (NCH + 1) / 2, HK = (KCH + 1) / 2;
    constexpr bool SKIP = sizeof(T) == 4;  // matrix instructions bound float: none for what lies past K or N
    constexpr int PK = KCH * 4 + 1, PN = NCH * 4 + 1;  // pitches: the odd unit spreads rows over the banks
    __shared__ u32x4 w_lds[NCH * KC * PK];
    __shared__ u32x4 x_lds[64 * PK];
    __shared__ u32x4 z_lds[64 * PN];
    __shared__ f32x4 bias_lds[NCH * KC / 4];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, q = lane >> 4;
    const int strip = (wave & 3) * 16, half = wave >> 2;
    const int wn = wave / WK, wk = wave % WK;
    const int64_t begin = blockIdx.x * a.rows_per_block;
    const int64_t end = begin + a.rows_per_block < a.rows ? begin + a.rows_per_block : a.rows;
    const T* w = static_cast<const T*>(a.w);
    const T* dy = static_cast<const T*>(a.dy);
    T* dx = static_cast<T*>(a.dx);

    for (int i = tid; i < NCH * KC * KCH * 4; i += 512) {
        const int n = i / (KCH * 4), u = i % (KCH * 4);
        w_lds[n * PK + u] = n < a.N ? load_row(w + (int64_t)n * a.K, u * E, a.K) : u32x4{0u, 0u, 0u, 0u};
    }
    for (int n = tid; n < NCH * KC; n += 512)
        reinterpret_cast<float*>(bias_lds)[n] =
            a.bias && n < a.N ? to_f32(static_cast<const T*>(a.bias)[n]) : 0.0f;

    f32x4 acc[TN][TK], acc_b[TN];
#pragma unroll
    for (int i = 0; i < TN; ++i) {
        acc_b[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < TK; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    float one[E];
#pragma unroll
    for (int i = 0; i < E; ++i) one[i] = 1.0f;
    const u32x4 ones = pack<T>(one);

    RowRaw<T, Q8, WIDE> xr[KCH];
    u32x4 yr[HN];
    auto row_of = [&](int64_t m0) {  // past the end: the last row again
        const int64_t m = m0 + strip + r;
        return m < end ? m : end - 1;
    };
    auto load_x = [&](int64_t m) {
#pragma unroll
        for (int c = 0; c < KCH; ++c) xr[c].issue(a.x, m, c * KC + q * E);
    };
    auto load_y = [&](int64_t m, int gi) {
        yr[gi] = issue_row<T, WIDE>(dy + m * a.ldy, (2 * gi + half) * KC + q * E, a.N);
    };
    if (begin < end) {
        const int64_t m = row_of(begin);
        load_x(m);
#pragma unroll
        for (int gi = 0; gi < HN; ++gi) load_y(m, gi);
    }
    __syncthreads();  // W is there

    auto step = [&](int64_t m0, auto whole) {
        const int64_t m = m0 + strip + r, next = row_of(m0 + 64);
        const bool valid = whole.value || m < end;
        const u32x4 zero = {0u, 0u, 0u, 0u};
        u32x4 xf[KCH];
#pragma unroll
        for (int c = 0; c < KCH; ++c) {
            xf[c] = xr[c].finish_in(a.x, c * KC, c * KC + q * E);
            if (!valid) xf[c] = zero;  // rows past the end add nothing, whatever the last row holds
            if (a.part && (KCH == 1 ? half == 0 : (c & 1) == half)) x_lds[(strip + r) * PK + c * 4 + q] = xf[c];
        }
#pragma unroll
        for (int gi = 0; gi < HN; ++gi) {
            const int g = 2 * gi + half;
            if ((NCH == 1 && half) || (SKIP && g * KC >= a.N)) break;
            u32x4 dz = finish_chunk<T, WIDE>(yr[gi], g * KC, g * KC + q * E, a.N);
            if constexpr (whole.value) load_y(next, gi);
            if (a.act != GS3D_ACT_NONE) {
                f32x4 z[TG];
#pragma unroll
                for (int t = 0; t < TG; ++t) z[t] = bias_lds[g * 4 * TG + q * TG + t];
#pragma unroll
                for (int c = 0; c < KCH; ++c)
#pragma unroll
                    for (int t = 0; t < TG; ++t)
                        z[t] = multiply_chunk<T>(w_lds[tile_column<T>(g * TG + t, r) * PK + c * 4 + q], xf[c], z[t],
                                                 a.K - c * KC);
                float arg[E], grad[E];
                unpack<T>(dz, grad);
#pragma unroll
                for (int i = 0; i < E; ++i) arg[i] = z[i / 4][i & 3];
                pull_back(grad, arg, a.act);
                dz = pack<T>(grad);
            }
            z_lds[(strip + r) * PN + g * 4 + q] = valid ? dz : zero;
        }
        if constexpr (whole.value) load_x(next);
        __syncthreads();
        if (dx) {
            u32x4 dz[NCH];
#pragma unroll
            for (int g = 0; g < NCH; ++g) dz[g] = z_lds[(strip + r) * PN + g * 4 + q];
#pragma unroll
            for (int ci = 0; ci < HK; ++ci) {
                const int c = 2 * ci + half;
                if ((KCH == 1 && half) || (SKIP && c * KC >= a.K)) break;
                f32x4 out[TG];
#pragma unroll
                for (int t = 0; t < TG; ++t) out[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int g = 0; g < NCH; ++g) {
                    if (SKIP && g * KC >= a.N) break;
#pragma unroll
                    for (int t = 0; t < TG; ++t)
                        out[t] = multiply_chunk<T>(read_transposed<T, true>(w_lds, PK, g * KC, c * TG + t, lane), dz[g],
                                                   out[t], a.N - g * KC);
                }
                float v[E];
#pragma unroll
                for (int i = 0; i < E; ++i) v[i] = out[i / 4][i & 3];
                if (valid) store_chunk(dx + m * a.K, c * KC, c * KC + q * E, a.K, pack<T>(v));
            }
        }
        if (a.part && wn < NT) {
#pragma unroll
            for (int c = 0; c < 64 / KC; ++c) {
                u32x4 fz[TN], fx[TK];
#pragma unroll
                for (int i = 0; i < TN; ++i) fz[i] = read_transposed<T, false>(z_lds, PN, c * KC, i * WN + wn, lane);
#pragma unroll
                for (int j = 0; j < TK; ++j) fx[j] = read_transposed<T, false>(x_lds, PK, c * KC, j * WK + wk, lane);
#pragma unroll
                for (int i = 0; i < TN; ++i) {
                    if (SKIP && (i * WN + wn) * 16 >= a.N) break;
#pragma unroll
                    for (int j = 0; j < TK; ++j) {
                        if (SKIP && (j * WK + wk) * 16 >= a.K) break;
                        acc[i][j] = multiply<T>(fz[i], fx[j], acc[i][j]);
                    }
                    if (wk == 0) acc_b[i] = multiply<T>(fz[i], ones, acc_b[i]);
                }
            }
        }
        __syncthreads();  // the tiles' readers are done
    };
    int64_t m0 = begin;
    for (; m0 + 64 <= end; m0 += 64) step(m0, Flag<true>{});
    if (m0 < end) step(m0, Flag<false>{});

    if (!a.part || wn >= NT) return;
    float* part = a.part + (int64_t)blockIdx.x * ((int64_t)a.N * a.K + a.N);
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int n = (i * WN + wn) * 16 + 4 * q + e;
            if (n >= a.N) continue;
#pragma unroll
            for (int j = 0; j < TK; ++j) {
                const int k = (j * WK + wk) * 16 + r;
                if (k < a.K) part[(int64_t)n * a.K + k] = acc[i][j][e];
            }
            if (wk == 0 && r == 0) part[(int64_t)a.N * a.K + n] = acc_b[i][e];
        }
}

// Widths are covered by 1, 2, 4 or 8 chunks (float: 2, 4 or 8, so that dW's
// tiles split over 2 x 2 wavefronts), as far as a wavefront's quarter of dW
// stays in 64 registers: 128 x 128, 64 x 256, 32 x 256 of 16-bit types and
// 128 x 128 of float.
template <class T>
static int fused_chunks(int channels) {
    const int least = sizeof(T) == 4 ? 2 : 1;
    int chunks = 8;
    while (chunks > least && channels <= chunks / 2 * CHUNK<T>) chunks /= 2;
    return chunks;
}
template <class T>
static bool fused_fits(int K, int N) {
    if (K > 8 * CHUNK<T> || N > 8 * CHUNK<T>) return false;
    return sizeof(T) == 4 || fused_chunks<T>(K) * fused_chunks<T>(N) <= 16;
}

template <class T, bool Q8, int KCH, int NCH>
static void launch_fused_as(const LinearFused& a, int blocks, hipStream_t stream) {
    constexpr int LEAST = sizeof(T) == 4 ? 2 : 1;
    if constexpr (KCH == LEAST || NCH == LEAST) {
        if (a.K < VEC<T> || a.N < VEC<T>) {  // rows shorter than a vector
            hipLaunchKernelGGL((linear_bwd_fused_kernel<T, Q8, KCH, NCH, false>), dim3((unsigned)blocks), dim3(512), 0,
                               stream, a);
            return;
        }
    }
    hipLaunchKernelGGL((linear_bwd_fused_kernel<T, Q8, KCH, NCH, true>), dim3((unsigned)blocks), dim3(512), 0, stream,
                       a);
}
template <class T, bool Q8, int KCH>
static void launch_fused_n(const LinearFused& a, int blocks, hipStream_t stream) {
    constexpr int MOST = sizeof(T) == 4 ? 64 : 16;
    switch (fused_chunks<T>(a.N)) {
        case 1:
            if constexpr (sizeof(T) == 2) launch_fused_as<T, Q8, KCH, 1>(a, blocks, stream);
            break;
        case 2: launch_fused_as<T, Q8, KCH, 2>(a, blocks, stream); break;
        case 4:
            if constexpr (KCH * 4 <= MOST) launch_fused_as<T, Q8, KCH, 4>(a, blocks, stream);
            break;
        default:
            if constexpr (KCH * 8 <= MOST) launch_fused_as<T, Q8, KCH, 8>(a, blocks, stream);
            break;
    }
}
template <class T, bool Q8>
static void launch_fused(const LinearFused& a, int blocks, hipStream_t stream) {
    switch (fused_chunks<T>(a.K)) {
        case 1:
            if constexpr (sizeof(T) == 2) launch_fused_n<T, Q8, 1>(a, blocks, stream);
            break;
        case 2: launch_fused_n<T, Q8, 2>(a, blocks, stream); break;
        case 4: launch_fused_n<T, Q8, 4>(a, blocks, stream); break;
        default: launch_fused_n<T, Q8, 8>(a, blocks, stream); break;
    }
}

// Specialised by linear_fused_f32.hip, linear_fused_bf16.hip, linear_fused_f16.hip.
template <class T>
void fused_launch(const LinearFused& a, bool q8, int blocks, hipStream_t stream);
template <>
void fused_launch<float>(const LinearFused& a, bool q8, int blocks, hipStream_t stream);
template <>
void fused_launch<bf16_t>(const LinearFused& a, bool q8, int blocks, hipStream_t stream);
template <>
void fused_launch<f16_t>(const LinearFused& a, bool q8, int blocks, hipStream_t stream);

}  // namespace gs3d
