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

// A block of 4 wavefronts takes 64 rows at a time, KCH chunks of K and NCH of
// N wide, over a range of rows of its own.
//
// A wavefront's 16 rows first: lane l holds row l % 16 and the elements from
// VEC (l / 16) on of every chunk, of x as of dy.  With W's rows as the first
// operand, z comes out with that row in that lane and, W's rows dealt out as
// tile_column says, with dy's elements beside it: dz = dy act'(z) is then a
// fragment as it stands, the second operand of dx = dz W.  W lies in LDS once,
// row by row; dx's first operand is read from it transposed.
//
// dW = dz^T x contracts over rows, which are spread over lanes: dz and x go to
// LDS row by row, and all wavefronts read them transposed, each for a quarter
// of dW (2 x 2), which stays in its registers over all the block's rows.
//
// Bytes bound it where K and N are small (x and dy in, dx out): the next 64
// rows are loaded while these are multiplied, and two blocks share a compute
// unit where their LDS fits.
template <class T, bool Q8, int KCH, int NCH>
__global__ __launch_bounds__(256, 2) void linear_bwd_fused_kernel(LinearFused a) {
    constexpr int E = VEC<T>;
    constexpr int KC = CHUNK<T>;
    constexpr int TG = KC / 16;              // tiles a chunk
    constexpr int KT = KCH * TG, NT = NCH * TG;
    // dW's tiles over the wavefronts: 2 x 2, or for float, whose matrix
    // instructions count most and skip what lies past K or N, N's dealt to all
    // four (33 x 97: at most 2 x 3 tiles a wavefront, not 4 x 2).
    constexpr int WN = sizeof(T) == 4 && NT >= 4 ? 4 : 2, WK = 4 / WN;
    constexpr int TN = NT / WN, TK = KT / WK;
    constexpr bool SKIP = sizeof(T) == 4;
    constexpr int PK = KCH * 4 + 1, PN = NCH * 4 + 1;  // pitches: the odd unit spreads rows over the banks
    __shared__ u32x4 w_lds[NCH * KC * PK];
    __shared__ u32x4 x_lds[64 * PK];
    __shared__ u32x4 z_lds[64 * PN];
    __shared__ float bias_lds[NCH * KC];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, q = lane >> 4;
    const int wn = wave / WK, wk = wave % WK;
    const int64_t begin = blockIdx.x * a.rows_per_block;
    const int64_t end = begin + a.rows_per_block < a.rows ? begin + a.rows_per_block : a.rows;
    const T* w = static_cast<const T*>(a.w);
    const T* dy = static_cast<const T*>(a.dy);
    T* dx = static_cast<T*>(a.dx);

    for (int i = tid; i < NCH * KC * KCH * 4; i += 256) {
        const int n = i / (KCH * 4), u = i % (KCH * 4);
        w_lds[n * PK + u] = n < a.N ? load_row(w + (int64_t)n * a.K, u * E, a.K) : u32x4{0u, 0u, 0u, 0u};
    }
    for (int n = tid; n < NCH * KC; n += 256)
        bias_lds[n] = a.bias && n < a.N ? to_f32(static_cast<const T*>(a.bias)[n]) : 0.0f;

    RowRaw<T, Q8> xr[KCH];
    u32x4 yr[NCH];
    auto row_of = [&](int64_t m0) {  // past the end: the last row again
        const int64_t m = m0 + wave * 16 + r;
        return m < end ? m : end - 1;
    };

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

    if (begin < end) {
        const int64_t m = row_of(begin);
#pragma unroll
        for (int c = 0; c < KCH; ++c) xr[c].issue(a.x, m, c * KC + q * E);
#pragma unroll
        for (int g = 0; g < NCH; ++g) yr[g] = issue_row(dy + m * a.ldy, g * KC + q * E, a.N);
    }
    for (int64_t m0 = begin; m0 < end; m0 += 64) {
        const int64_t m = m0 + wave * 16 + r, next = row_of(m0 + 64);
        const bool valid = m < end;
        u32x4 xf[KCH];
#pragma unroll
        for (int c = 0; c < KCH; ++c) xf[c] = xr[c].finish(a.x, c * KC + q * E);
        if (m0 + 64 > end) {  // rows past the end add nothing, whatever the last row holds
#pragma unroll
            for (int c = 0; c < KCH; ++c) xf[c] = valid ? xf[c] : u32x4{0u, 0u, 0u, 0u};
        } else {
#pragma unroll
            for (int c = 0; c < KCH; ++c) xr[c].issue(a.x, next, c * KC + q * E);
        }
        __syncthreads();  // the tiles' last readers are done (and W is there)
        if (a.part) {
#pragma unroll
            for (int c = 0; c < KCH; ++c) x_lds[(wave * 16 + r) * PK + c * 4 + q] = xf[c];
        }
        f32x4 out[KT];
#pragma unroll
        for (int t = 0; t < KT; ++t) out[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int g = 0; g < NCH; ++g) {
            if (SKIP && g * KC >= a.N) break;
            u32x4 dz = finish_row<T>(yr[g], g * KC + q * E, a.N);
            yr[g] = issue_row(dy + next * a.ldy, g * KC + q * E, a.N);
            if (a.act != GS3D_ACT_NONE) {
                f32x4 z[TG];
#pragma unroll
                for (int t = 0; t < TG; ++t) z[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < KCH; ++c)
#pragma unroll
                    for (int t = 0; t < TG; ++t)
                        z[t] = multiply_chunk<T>(w_lds[tile_column<T>(g * TG + t, r) * PK + c * 4 + q], xf[c], z[t],
                                                 a.K - c * KC);
                float arg[E], grad[E];
                unpack<T>(dz, grad);
#pragma unroll
                for (int i = 0; i < E; ++i) arg[i] = z[i / 4][i & 3] + bias_lds[g * KC + q * E + i];
                pull_back(grad, arg, a.act);
                dz = pack<T>(grad);
            }
            if (m0 + 64 > end) dz = valid ? dz : u32x4{0u, 0u, 0u, 0u};
            if (a.part) z_lds[(wave * 16 + r) * PN + g * 4 + q] = dz;
            if (dx) {
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    if (SKIP && t * 16 >= a.K) break;
                    out[t] = multiply_chunk<T>(read_transposed<T, true>(w_lds, PK, g * KC, t, lane), dz, out[t],
                                               a.N - g * KC);
                }
            }
        }
        if (dx && valid) {
#pragma unroll
            for (int c = 0; c < KCH; ++c) {
                float v[E];
#pragma unroll
                for (int i = 0; i < E; ++i) v[i] = out[c * TG + i / 4][i & 3];
                store_row(dx + m * a.K, c * KC + q * E, a.K, pack<T>(v));
            }
        }
        if (a.part) {
            __syncthreads();
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
    }

    if (!a.part) return;
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
    hipLaunchKernelGGL((linear_bwd_fused_kernel<T, Q8, KCH, NCH>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
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
