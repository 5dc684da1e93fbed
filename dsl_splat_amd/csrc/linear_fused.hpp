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
    int* blocks;       // host: receives how many blocks were launched
};

// How a backward kernel of KCH x NCH chunks lies on a compute unit: two blocks
// of 8 wavefronts where their LDS fits, of 128, 64 or 32 rows at a time, whose
// barriers leave each other's work alone; else one of 16, the weights once for
// all of them.  Four wavefronts a SIMD either way.  Two blocks of 32 rows and
// one of 128 (us, silu): 1.92 M rows of bfloat16, 128 to 128 channels, 525 and
// 548; 1 M rows, 64 to 256: 323 and 372; float, 64 to 128: 570 and 664.
template <class T, int KCH, int NCH, bool ACT>
struct FusedShape {
    static constexpr int PLANES = SPLIT<T> && ACT ? 2 : 1;
    static constexpr int PAD = sizeof(T) == 4 ? 1 : 2;
    static constexpr int FIXED = NCH * CHUNK<T> * ((KCH * 4 + PAD) * 16 + 4);
    static constexpr int ROW = (KCH * 4 + PAD + PLANES * (NCH * 4 + PAD)) * 16;
    static constexpr bool TWO = FIXED + 32 * ROW <= 81920;
    static constexpr int WAVES = TWO ? 8 : 16;
    static constexpr int ROOM = TWO ? 81920 : 163840;
    static constexpr int ROWS = FIXED + 128 * ROW <= ROOM ? 128 : FIXED + 64 * ROW <= ROOM ? 64 : 32;
    static constexpr int STRIPS = ROWS == 128 && WAVES == 16 ? 8 : ROWS == 32 ? 2 : 4;  // of 16 rows, taken at a time
    static constexpr int PARTS = WAVES / STRIPS;                       // wavefronts that share a strip
    static constexpr int RB = ROWS / (16 * STRIPS);
};

// A block takes ROWS rows at a time, KCH chunks of K and NCH of N wide, over a
// range of rows of its own.
//
// x and dy go to LDS as they lie in memory, row by row (whole lines an
// instruction), the next rows on their way while these are worked on.
//
// First dz.  PARTS wavefronts take a strip of 16 rows, every PARTS-th chunk of
// N each: lane l has row l % 16 and the elements from VEC (l / 16) on of a
// chunk, of x as of dy.  With W's rows as the first operand, z comes out with
// that row in that lane and, W's rows dealt out as tile_column says, with dy's
// elements beside it, so dz = dy act'(z) takes dy's place vector by vector,
// its low half in a second plane.
//
// Then dx = dz W and dW = dz^T x.  dx takes dz from LDS as it lies and W
// transposed (W is in LDS once, row by row), every PARTS-th chunk of K a
// wavefront.  dW contracts over rows: both operands are read transposed, and
// each wavefront's share of its tiles stays in its registers over all the
// block's rows.
//
// Bytes bound it where K and N are small (x and dy in, dx out), the vector
// units where the slope is dear; four wavefronts a SIMD let one's loads and
// slopes run under another's products.  1.92 M rows of bfloat16, 32 to 128
// channels: 165 us without an activation (4.5 TB/s), 297 with gelu, whose slope
// keeps the vector units busy 80% of the time; 128 to 128 with silu from 8 bits
// 505, vector units 55% and matrix units 31%; 1.44 M rows of float, 33 to 97: 667,
// matrix units 61%.  As separate products instead: 745, 920 and 1066.
template <class T, bool Q8, int KCH, int NCH, bool WIDE, bool ACT>
__global__ __launch_bounds__((FusedShape<T, KCH, NCH, ACT>::WAVES * 64), 4)
void linear_bwd_fused_kernel(LinearFused a) {
    using S = FusedShape<T, KCH, NCH, ACT>;
    constexpr int E = VEC<T>;
    constexpr int KC = CHUNK<T>;
    constexpr int TG = KC / 16;  // tiles a chunk
    constexpr int KT = KCH * TG, NT = NCH * TG;
    constexpr int THREADS = S::WAVES * 64, PLANES = S::PLANES, PARTS = S::PARTS;
    constexpr int WK_MOST = S::WAVES / (NT < 4 ? 2 : 4);  // wavefronts along K and N, none without a tile
    constexpr int WK = KT < WK_MOST ? KT : WK_MOST, WN = S::WAVES / WK;
    constexpr int TN = (NT + WN - 1) / WN, TK = (KT + WK - 1) / WK;
    constexpr int HN = (NCH + PARTS - 1) / PARTS, HK = (KCH + PARTS - 1) / PARTS;
    constexpr bool SKIP = sizeof(T) == 4;  // matrix instructions bound float: none for what lies past K or N
    constexpr int VK = KCH * 4, VN = NCH * 4;          // vectors of a row
    constexpr int PK = VK + S::PAD, PN = VN + S::PAD;  // pitches that spread rows over the banks, read either way
    // Vectors are dealt to threads by powers of two a row; a row of 7 chunks
    // leaves some without.
    constexpr int DN = NCH > 4 ? 32 : VN;
    constexpr int RB = S::RB, ROWS = S::ROWS;
    constexpr int LK = (ROWS * VK + THREADS - 1) / THREADS, LN = (ROWS * DN + THREADS - 1) / THREADS;
    __shared__ u32x4 w_lds[NCH * KC * PK];
    __shared__ u32x4 x_lds[ROWS * PK];
    __shared__ u32x4 z_lds[PLANES][ROWS * PN];
    __shared__ f32x4 bias_lds[NCH * KC / 4];

    const int tid = threadIdx.x, wave = wave_id();
    const int part = wave / S::STRIPS;
    const int wn = wave / WK, wk = wave % WK;
    const int64_t begin = blockIdx.x * a.rows_per_block;
    const int64_t end = begin + a.rows_per_block < a.rows ? begin + a.rows_per_block : a.rows;
    const T* w = static_cast<const T*>(a.w);
    const T* dy = static_cast<const T*>(a.dy);
    T* dx = static_cast<T*>(a.dx);

    for (int i = tid; i < NCH * KC * VK; i += THREADS) {
        const int n = i / VK, u = i % VK;
        w_lds[n * PK + u] = n < a.N ? load_row(w + (int64_t)n * a.K, u * E, a.K) : u32x4{0u, 0u, 0u, 0u};
    }
    for (int n = tid; n < NCH * KC; n += THREADS)
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

    RowRaw<T, Q8, WIDE> xr[LK];
    u32x4 yr[LN];
    auto load = [&](int64_t m0) {  // rows past the end: the last row again
#pragma unroll
        for (int i = 0; i < LK; ++i) {
            const int u = i * THREADS + tid;
            const int64_t m = m0 + u / VK < end ? m0 + u / VK : end - 1;
            xr[i].issue(a.x, m, u % VK * E);
        }
#pragma unroll
        for (int i = 0; i < LN; ++i) {
            const int u = i * THREADS + tid;
            const int64_t m = m0 + u / DN < end ? m0 + u / DN : end - 1;
            yr[i] = issue_row<T, WIDE>(dy + m * a.ldy, u % DN * E, a.N);
        }
    };
    // Rows past the end add nothing, whatever the last row holds (dz is cleared
    // again after the slope, which an infinite weight makes NaN there).
    auto fill = [&](int64_t m0) {
        const u32x4 zero = {0u, 0u, 0u, 0u};
        const bool whole = m0 + ROWS <= end;
#pragma unroll
        for (int i = 0; i < LK; ++i) {
            const int u = i * THREADS + tid;
            if (ROWS * VK % THREADS != 0 && u >= ROWS * VK) break;
            u32x4 v = xr[i].finish_in(a.x, VK * E <= a.K, u % VK * E);
            x_lds[u / VK * PK + u % VK] = whole || m0 + u / VK < end ? v : zero;
        }
#pragma unroll
        for (int i = 0; i < LN; ++i) {
            const int u = i * THREADS + tid;
            if (ROWS * DN % THREADS != 0 && u >= ROWS * DN) break;
            u32x4 v = yr[i];
            if (VN * E > a.N) v = finish_row<T, WIDE>(v, u % DN * E, a.N);
            if (DN == VN || u % DN < VN) z_lds[0][u / DN * PN + u % DN] = whole || m0 + u / DN < end ? v : zero;
        }
    };

    if (begin < end) load(begin);
    for (int64_t m0 = begin; m0 < end; m0 += ROWS) {
        fill(m0);
        if (m0 + ROWS < end) load(m0 + ROWS);
        __syncthreads();
        // Opaque in every round: the tiles' addresses, all of them loop
        // invariant, would otherwise fill the registers.
        int lane = tid & 63;
        asm volatile("" : "+v"(lane));
        const int r = lane & 15, q = lane >> 4;
        if constexpr (ACT) {
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                const int strip = (b * S::STRIPS + wave % S::STRIPS) * 16;
                u32x4 xf[KCH];
#pragma unroll
                for (int c = 0; c < KCH; ++c) xf[c] = x_lds[(strip + r) * PK + c * 4 + q];
#pragma unroll
                for (int gi = 0; gi < HN; ++gi) {
                    const int g = NCH == 1 ? 0 : PARTS * gi + part;
                    if (NCH == 1 && part != (RB == 2 ? b : 0)) break;  // one chunk: a strip each
                    if (g >= NCH || (SKIP && g * KC >= a.N)) break;
                    f32x4 z[TG];
#pragma unroll
                    for (int t = 0; t < TG; ++t) z[t] = bias_lds[g * 4 * TG + q * TG + t];
#pragma unroll
                    for (int c = 0; c < KCH; ++c)
#pragma unroll
                        for (int t = 0; t < TG; ++t)
                            z[t] = multiply_chunk<T>(w_lds[tile_column<T>(g * TG + t, r) * PK + c * 4 + q], xf[c], z[t],
                                                     a.K - c * KC);
                    settle(z);
                    const int at = (strip + r) * PN + g * 4 + q;
                    float arg[E], grad[E];
                    unpack<T>(z_lds[0][at], grad);
#pragma unroll
                    for (int i = 0; i < E; ++i) arg[i] = z[i / 4][i & 3];
                    pull_back<T>(grad, arg, a.act);
                    // Past N and past the last row an infinity of x or of W
                    // meets a zero, and the slope there is NaN.
                    if (g * KC + KC > a.N || m0 + ROWS > end) {
                        const bool live = m0 + strip + r < end;
#pragma unroll
                        for (int i = 0; i < E; ++i)
                            grad[i] = live && g * KC + q * E + i < a.N ? grad[i] : 0.0f;
                    }
                    if constexpr (PLANES == 2) {
                        z_lds[0][at] = take_high<T>(grad);
                        z_lds[1][at] = pack<T>(grad);
                    } else {
                        z_lds[0][at] = pack<T>(grad);
                    }
                }
            }
            __syncthreads();
        }
        if (dx) {
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                const int strip = (b * S::STRIPS + wave % S::STRIPS) * 16;
                const int64_t m = m0 + strip + r;
#pragma unroll
                for (int ci = 0; ci < HK; ++ci) {
                    const int c = KCH == 1 ? 0 : PARTS * ci + part;
                    if (KCH == 1 && part != (RB == 2 ? b : 0)) break;
                    if (c >= KCH || (SKIP && c * KC >= a.K)) break;
                    f32x4 out[TG];
#pragma unroll
                    for (int t = 0; t < TG; ++t) out[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int g = 0; g < NCH; ++g) {
                        if (SKIP && g * KC >= a.N) break;
                        u32x4 dz[PLANES];
#pragma unroll
                        for (int p = 0; p < PLANES; ++p) dz[p] = z_lds[p][(strip + r) * PN + g * 4 + q];
#pragma unroll
                        for (int t = 0; t < TG; ++t) {
                            const u32x4 wf = read_transposed<T, true>(w_lds, PK, g * KC, c * TG + t, lane);
#pragma unroll
                            for (int p = 0; p < PLANES; ++p)
                                out[t] = multiply_chunk<T>(wf, dz[p], out[t], a.N - g * KC);
                        }
                    }
                    settle(out);
                    float v[E];
#pragma unroll
                    for (int i = 0; i < E; ++i) v[i] = out[i / 4][i & 3];
                    if (m < end) store_chunk(dx + m * a.K, c * KC, c * KC + q * E, a.K, pack<T>(v));
                }
            }
        }
        if (a.part) {
#pragma unroll
            for (int c = 0; c < ROWS / KC; ++c) {
                // Where the tiles do not share out evenly the last one is taken
                // again, and not stored.
                u32x4 fz[PLANES][TN], fx[TK];
#pragma unroll
                for (int i = 0; i < TN; ++i) {
                    const int t = i * WN + wn;
#pragma unroll
                    for (int p = 0; p < PLANES; ++p)
                        fz[p][i] = read_transposed<T, false>(z_lds[p], PN, c * KC, t < NT ? t : NT - 1, lane);
                }
#pragma unroll
                for (int j = 0; j < TK; ++j) {
                    const int t = j * WK + wk;
                    fx[j] = read_transposed<T, false>(x_lds, PK, c * KC, t < KT ? t : KT - 1, lane);
                }
#pragma unroll
                for (int p = 0; p < PLANES; ++p)
#pragma unroll
                    for (int i = 0; i < TN; ++i) {
#pragma unroll
                        for (int j = 0; j < TK; ++j) acc[i][j] = multiply<T>(fz[p][i], fx[j], acc[i][j]);
                        acc_b[i] = multiply<T>(fz[p][i], ones, acc_b[i]);
                    }
            }
        }
        __syncthreads();  // the tiles' readers are done
    }

    if (!a.part) return;
    const int r = tid & 15, q = (tid & 63) >> 4;
#pragma unroll
    for (int i = 0; i < TN; ++i) settle(acc[i]);
    settle(acc_b);
    float* out = a.part + (int64_t)blockIdx.x * ((int64_t)a.N * a.K + a.N);
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int n = (i * WN + wn) * 16 + 4 * q + e;
            if (n >= a.N) continue;
#pragma unroll
            for (int j = 0; j < TK; ++j) {
                const int k = (j * WK + wk) * 16 + r;
                if (k < a.K) out[(int64_t)n * a.K + k] = acc[i][j][e];
            }
            if (wk == 0 && r == 0) out[(int64_t)a.N * a.K + n] = acc_b[i][e];
        }
}

// Widths of 16-bit types are covered by 1, 2, 4 or 8 chunks, as far as a
// wavefront's share of dW leaves it registers: 128 x 128, 64 x 256, 256 x 64.
// Float's chunks are half as wide, 2, 4 or 8 of K, 2, 4, 7 or 8 of N: LDS
// decides how many rows a block of two on a compute unit takes at a time (us at
// 7 chunks of N and at 8: 1.44 M rows, 33 to 97 channels 672 and 757; 1 M, 64 to
// 112 529 and 550, 100 to 96 872 and 877, 64 to 90 498 and 505; at 6 the last
// two 915 and 498).
template <class T>
static int fused_chunks_k(int channels) {
    const int chunks = (channels + CHUNK<T> - 1) / CHUNK<T>;
    if (sizeof(T) == 4) return chunks <= 2 ? 2 : chunks <= 4 ? 4 : 8;
    return chunks <= 2 ? chunks : chunks <= 4 ? 4 : 8;
}
template <class T>
static int fused_chunks_n(int channels) {
    const int chunks = (channels + CHUNK<T> - 1) / CHUNK<T>;
    if (sizeof(T) == 4) return chunks <= 2 ? 2 : chunks <= 4 ? 4 : chunks <= 7 ? 7 : 8;
    return chunks <= 2 ? chunks : chunks <= 4 ? 4 : 8;
}
template <class T>
static bool fused_fits(int K, int N) {
    if (K > 8 * CHUNK<T> || N > 8 * CHUNK<T>) return false;
    return sizeof(T) == 4 || fused_chunks_k<T>(K) * fused_chunks_n<T>(N) <= 16;
}

template <class T, bool Q8, int KCH, int NCH, bool WIDE, bool ACT>
static void launch_fused_act(LinearFused a, int blocks, hipStream_t stream) {
    using S = FusedShape<T, KCH, NCH, ACT>;
    // Half as many blocks where one fills a compute unit (the scratch was
    // sized for two).
    if (!S::TWO && blocks > 256) {
        a.rows_per_block = (a.rows_per_block * blocks / 256 + 63) / 64 * 64;
        blocks = (int)((a.rows + a.rows_per_block - 1) / a.rows_per_block);
    }
    *a.blocks = blocks;
    hipLaunchKernelGGL((linear_bwd_fused_kernel<T, Q8, KCH, NCH, WIDE, ACT>), dim3((unsigned)blocks),
                       dim3(S::WAVES * 64), 0, stream, a);
}
template <class T, bool Q8, int KCH, int NCH>
static void launch_fused_as(const LinearFused& a, int blocks, hipStream_t stream) {
    constexpr int LEAST = sizeof(T) == 4 ? 2 : 1;
    const bool act = a.act != GS3D_ACT_NONE;
    if constexpr (KCH == LEAST || NCH == LEAST) {
        if (a.K < VEC<T> || a.N < VEC<T>) {  // rows shorter than a vector
            if (act) launch_fused_act<T, Q8, KCH, NCH, false, true>(a, blocks, stream);
            else launch_fused_act<T, Q8, KCH, NCH, false, false>(a, blocks, stream);
            return;
        }
    }
    if (act) launch_fused_act<T, Q8, KCH, NCH, true, true>(a, blocks, stream);
    else launch_fused_act<T, Q8, KCH, NCH, true, false>(a, blocks, stream);
}
template <class T, bool Q8, int KCH>
static void launch_fused_n(const LinearFused& a, int blocks, hipStream_t stream) {
    constexpr bool F = sizeof(T) == 4;
    switch (fused_chunks_n<T>(a.N)) {
        case 1:
            if constexpr (!F) launch_fused_as<T, Q8, KCH, 1>(a, blocks, stream);
            break;
        case 2: launch_fused_as<T, Q8, KCH, 2>(a, blocks, stream); break;
        case 4:
            if constexpr (F || KCH <= 4) launch_fused_as<T, Q8, KCH, 4>(a, blocks, stream);
            break;
        case 7:
            if constexpr (F) launch_fused_as<T, Q8, KCH, 7>(a, blocks, stream);
            break;
        case 8:
            if constexpr (F || KCH <= 2) launch_fused_as<T, Q8, KCH, 8>(a, blocks, stream);
            break;
    }
}
template <class T, bool Q8>
static void launch_fused(const LinearFused& a, int blocks, hipStream_t stream) {
    constexpr bool F = sizeof(T) == 4;
    switch (fused_chunks_k<T>(a.K)) {
        case 1:
            if constexpr (!F) launch_fused_n<T, Q8, 1>(a, blocks, stream);
            break;
        case 2: launch_fused_n<T, Q8, 2>(a, blocks, stream); break;
        case 4: launch_fused_n<T, Q8, 4>(a, blocks, stream); break;
        case 8: launch_fused_n<T, Q8, 8>(a, blocks, stream); break;
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
