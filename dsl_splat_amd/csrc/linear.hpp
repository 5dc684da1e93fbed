// Per-pixel products of the feature decoder: y = act(x W^T + b) + r and its
// gradients, over rows x (pixels) that are many and channels that are few.
// Included by linear_f32.hip, linear_bf16.hip and linear_f16.hip.
//
//   linear_stream_kernel     rows times weights that lie in LDS whole, while the
//                            rows stream past: every product whose contracted
//                            dimension has at most 4 chunks
//   linear_tile_kernel       longer ones of 16-bit types, of many rows into many
//                            columns: 64 whole rows in LDS against weights that
//                            pack_weights_kernel laid out
//   linear_rows_kernel       the other longer ones: rows and weights in steps
//   linear_bwd_fused_kernel  the whole backward pass in one (linear_fused.hpp),
//                            where its weights and their gradient fit a block
//   linear_gradw_kernel      otherwise: dW = dz^T x and db = sum dz, split over
//                            the rows, after dz and dx from the kernels above
//   sum_splits_kernel        the blocks' partial sums in a fixed order
//
// The products of the forward end in act (EPI 0), or in act and + r (EPI 2);
// those of the backward (EPI 1) in dz = dy act'(x W^T + b), z computed again
// rather than kept.
// Products of 16-bit types go through matrix instructions with sums in 32
// bits.  dz enters the products after it as decode.hpp says at SPLIT: a row of
// its N high halves and then its N low ones, so that dx = dz W is the product
// of that row, twice as long, with W^T beside itself.
#pragma once

#include "linear_fused.hpp"
#include "xcd.hpp"

namespace gs3d {

struct LinearRows {
    Rows x;              // rows x K
    const void* w;       // N x K
    const void* bias;    // N or NULL
    const void* other;   // EPI 1: dy; EPI 2: residual
    int64_t ldo;
    void* y;             // rows x N; EPI 1 of 16-bit types: x 2 N, the second half what the first leaves of dz
    int64_t ldy;
    int64_t rows;
    int K, N, act, n_tiles, row_blocks, strips;
    int8_t* keep_codes;  // where the rows of x are kept in 8 bits, or NULL
    uint8_t* keep_scales;
};

template <class T, int EPI>
constexpr bool KEEPS_LOW = EPI == 1 && SPLIT<T>;

// The end of a product for one lane's vector of E neighbouring outputs.
template <class T, int EPI, int E>
GS3D_DEV u32x4 linear_end(const LinearRows& a, float (&z)[E], u32x4 raw_other, u32x4& low) {
    float o[E];
    if constexpr (EPI != 0) unpack<T>(raw_other, o);
    if constexpr (EPI == 1) {
        pull_back<T>(o, z, a.act);
        if constexpr (!SPLIT<T>) return pack<T>(o);
        const u32x4 high = take_high<T>(o);
        low = pack<T>(o);
        return high;
    } else {
        activate<T>(z, a.act);
        if constexpr (EPI == 2) {
#pragma unroll
            for (int i = 0; i < E; ++i) z[i] += o[i];
        }
        return pack<T>(z);
    }
}

template <bool V>
struct Flag {
    static constexpr bool value = V;
};

// Orders a wavefront's own LDS accesses (the LDS takes them in order; this is
// for the compiler).
GS3D_DEV void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A wavefront's strip of 16 rows x VP vectors, in LDS at pitch PO, to rows of N
// columns from `first` on and columns from n0 on, whole row segments an
// instruction.
template <class T, int VP, int PO, class Whole>
GS3D_DEV void store_strip(const u32x4* strip, T* y, int64_t ldy, int64_t first, int64_t end, int n0, int N, int lane,
                          Whole) {
    constexpr int E = VEC<T>;
    wave_fence();
    const int vec = lane % VP, at = n0 + vec * E;
#pragma unroll
    for (int i = 0; i < 16 * VP / 64; ++i) {
        const int row = i * (64 / VP) + lane / VP;
        const u32x4 raw = strip[row * PO + vec];
        const int64_t to = first + row;
        if (Whole::value && n0 + VP * E <= N) store16(y + to * ldy + at, raw);
        else if (to < end) store_row(y + to * ldy, at, N, raw);
    }
    wave_fence();
}

// What the stream kernel keeps in LDS: 16-byte vectors of an input row and of an
// output row, their pitches, and the vectors of a strip, of all.
template <class T, int KCH, int NT>
struct StreamShape {
    static constexpr int PAD = sizeof(T) == 4 ? 1 : 2;
    static constexpr int VK = KCH * 4, PK = VK + PAD;
    static constexpr int VP = 16 * NT / VEC<T>, PO = VP + PAD;
    static constexpr int STRIP = 16 * (PK > PO ? PK : PO);
    static constexpr int LDS = KCH * NT * 64 + 4 * STRIP + 4 * NT;
};

// Wavefronts a SIMD that the stream kernel's registers and LDS leave room for (a
// block puts one on each).
template <class T, bool Q8, int EPI, int KCH, int NT, bool WIDE>
constexpr int stream_waves() {
    const int wide = sizeof(T) == 4 ? 2 : 1;  // float holds twice the vectors
    const int vectors =
        wide * (2 * KCH + (EPI != 0 ? NT / 2 : 0)) + (KEEPS_LOW<T, EPI> ? NT / 2 + 1 : 0) + (WIDE ? 0 : 5);
    const int waves = vectors <= 4 ? 6 : vectors <= 8 ? 5 : vectors <= 12 ? 4 : vectors <= 16 ? 3 : 2;
    const int blocks = 163840 / (16 * StreamShape<T, KCH, NT>::LDS);
    return waves < blocks ? waves : blocks;
}

// A block of 4 wavefronts holds the weights of 16 NT columns in LDS, in
// fragment order (one 1 KB run per chunk and tile, read without conflicts),
// and takes strips of 16 rows from a range of a.strips of them; the
// wavefronts never wait for one another.  W's rows are the first operand, so
// a lane ends with 16 bytes of one output row; the sums start at the bias.
// HBM bounds it while K and N are small, the vector units where it ends in a gelu
// (1.92 M rows of bfloat16, 32 to 128 channels: 145 us, 4.2 TB/s, busy 95%).
//
// A fragment has one row in every lane of 16, and the memory pipeline joins
// neighbouring lanes only: read as fragments, 1 KB takes 64 accesses of 16
// bytes.  So a strip's rows, of x, of dy or the residual and of y, move in
// whole row segments, neighbouring lanes on neighbouring vectors, and change
// their layout in LDS that is the wavefront's own (1920 x 1080 pixels, 64 to
// 512 channels of float16: 754 us with fragments written as they come).
//
// Loads wait for the stores issued before them, so the next strip's are issued
// first, and whole strips store without a branch: the wait for a load then
// leaves the stores after it in flight.
template <class T, bool Q8, int EPI, int KCH, int NT, bool WIDE>
__global__ __launch_bounds__(256, (stream_waves<T, Q8, EPI, KCH, NT, WIDE>())) void linear_stream_kernel(LinearRows a) {
    constexpr int E = VEC<T>;
    constexpr int KC = CHUNK<T>;
    constexpr int TG = KC / 16;  // tiles of a lane's 16-byte output vector
    constexpr int G = NT / TG;
    using S = StreamShape<T, KCH, NT>;
    constexpr int VK = S::VK, PK = S::PK, VP = S::VP, PO = S::PO;
    constexpr int LK = 16 * VK / 64, LP = 16 * VP / 64;
    __shared__ u32x4 w_lds[KCH * NT * 64];
    __shared__ u32x4 strip_lds[4][S::STRIP];
    __shared__ f32x4 bias_lds[4 * NT];

    const Dealt at_tile = deal_block(blockIdx.x, a.row_blocks, a.n_tiles);  // the column tiles of a range of rows
    const int n_tile = at_tile.tile, n0 = n_tile * 16 * NT;
    const int64_t first = (int64_t)at_tile.group * a.strips * 16;
    const int64_t end = first + a.strips * 16 < a.rows ? first + a.strips * 16 : a.rows;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int r = lane & 15, q = lane >> 4;
    const T* w = static_cast<const T*>(a.w);
    const T* other = static_cast<const T*>(a.other);
    T* y = static_cast<T*>(a.y);
    u32x4* mine = strip_lds[wave];

    RowRaw<T, Q8, WIDE> xr[LK];
    auto load = [&](int64_t m0) {  // rows past the end repeat the last one and are not stored
#pragma unroll
        for (int i = 0; i < LK; ++i) {
            const int64_t m = m0 + i * (64 / VK) + lane / VK;
            xr[i].issue(a.x, m < end ? m : end - 1, lane % VK * E);
        }
    };
    int64_t m0 = first + wave * 16;
    load(m0);

#pragma unroll
    for (int i = 0; i < (KCH * NT + 3) / 4; ++i) {
        const int slot = i * 256 + tid;
        if (KCH * NT % 4 != 0 && slot >= KCH * NT * 64) break;
        const int c = slot / (NT * 64), t = (slot / 64) % NT, l = slot & 63;
        const int n = n0 + tile_column<T>(t, l & 15), k = c * KC + (l >> 4) * E;
        w_lds[slot] = n < a.N ? load_row(w + (int64_t)n * a.K, k, a.K) : u32x4{0u, 0u, 0u, 0u};
    }
    if (tid < 16 * NT)
        reinterpret_cast<float*>(bias_lds)[tid] =
            a.bias && n0 + tid < a.N ? to_f32(static_cast<const T*>(a.bias)[n0 + tid]) : 0.0f;
    __syncthreads();

    const bool staged = a.N % E == 0;  // else segments start anywhere, and vectors leave as they come
    const bool keep = a.keep_codes && n_tile == 0;
    auto strip = [&](int64_t m0, auto whole) {
        u32x4 xf[KCH];
#pragma unroll
        for (int i = 0; i < LK; ++i) {
            const u32x4 v = xr[i].finish_in(a.x, VK * E <= a.K, lane % VK * E);
            mine[(i * (64 / VK) + lane / VK) * PK + lane % VK] = v;
            if constexpr (EPI != 1 && !Q8) {
                if (keep) {
                    const int64_t m = m0 + i * (64 / VK) + lane / VK;
                    float f[E];
                    unpack<T>(v, f);
                    q8_keep<T, (VK < 32 / E ? VK : 32 / E)>(f, a.keep_codes, a.keep_scales, m, lane % VK * E, a.K,
                                                            whole.value || m < end);
                }
            }
        }
        u32x4 o[LP];
        if constexpr (EPI != 0) {
#pragma unroll
            for (int i = 0; i < LP; ++i) {
                const int64_t m = m0 + i * (64 / VP) + lane / VP;
                o[i] = issue_row<T, WIDE>(other + (whole.value || m < end ? m : end - 1) * a.ldo, n0 + lane % VP * E,
                                          a.N);
            }
        }
        if constexpr (whole.value) load(m0 + 64);
        wave_fence();
#pragma unroll
        for (int c = 0; c < KCH; ++c) xf[c] = mine[r * PK + c * 4 + q];
        wave_fence();
        if constexpr (EPI != 0) {
#pragma unroll
            for (int i = 0; i < LP; ++i) {
                u32x4 v = o[i];
                if (n0 + VP * E > a.N) v = finish_row<T, WIDE>(v, n0 + lane % VP * E, a.N);
                mine[(i * (64 / VP) + lane / VP) * PO + lane % VP] = v;
            }
            wave_fence();
        }
        u32x4 low[G];
        // The weights stay in LDS: hoisted out of the loop they would take
        // every register (128 at 4 chunks x 8 tiles).
        int at_w = lane;
        asm volatile("" : "+v"(at_w));
#pragma unroll
        for (int g = 0; g < G; ++g) {
            if (sizeof(T) == 4 && n0 + g * KC >= a.N) break;
            f32x4 acc[TG];
#pragma unroll
            for (int t = 0; t < TG; ++t) acc[t] = bias_lds[g * 4 * TG + (at_w >> 4) * TG + t];
#pragma unroll
            for (int c = 0; c < KCH; ++c)
#pragma unroll
                for (int t = 0; t < TG; ++t)
                    acc[t] = multiply_chunk<T>(w_lds[(c * NT + g * TG + t) * 64 + at_w], xf[c], acc[t], a.K - c * KC);
            settle(acc);
            float z[E];
#pragma unroll
            for (int i = 0; i < E; ++i) z[i] = acc[i / 4][i & 3];
            u32x4& slot = mine[r * PO + g * 4 + q];
            u32x4 raw = {0u, 0u, 0u, 0u};
            if constexpr (EPI != 0) raw = slot;
            raw = linear_end<T, EPI, E>(a, z, raw, low[g]);
            const int64_t m = m0 + r;
            if (staged) slot = raw;
            else if (whole.value || m < end) {
                store_chunk(y + m * a.ldy, n0 + g * KC, n0 + g * KC + q * E, a.N, raw);
                if constexpr (KEEPS_LOW<T, EPI>)
                    store_chunk(y + a.N + m * a.ldy, n0 + g * KC, n0 + g * KC + q * E, a.N, low[g]);
            }
        }
        if (staged) store_strip<T, VP, PO>(mine, y, a.ldy, m0, end, n0, a.N, lane, whole);
        else wave_fence();
        if constexpr (KEEPS_LOW<T, EPI>) {
            if (staged) {
#pragma unroll
                for (int g = 0; g < G; ++g) mine[r * PO + g * 4 + q] = low[g];
                store_strip<T, VP, PO>(mine, y + a.N, a.ldy, m0, end, n0, a.N, lane, whole);
            }
        }
    };
    for (; m0 + 16 <= end; m0 += 64) strip(m0, Flag<true>{});
    if (m0 < end) strip(m0, Flag<false>{});
}

// Longer contracted dimensions, where the products count more than the bytes,
// of float, of a few rows, beyond 512 channels or into a few columns: a block
// of 4 wavefronts computes 64 RS rows x 16 NT columns.  CH chunks of the
// weights at a time go through LDS, twice buffered, so a step has one barrier;
// a fragment read from there serves the RS strips of a wavefront (the LDS port,
// 128 bytes a clock, would bound RS = 1: 8 clocks a fragment and wavefront, 16
// clocks a matrix instruction).  The next step's operands are loaded while this
// one's are multiplied.  1.44 M rows of float, 128 to 64 channels: 360 us, 66
// TFLOP/s of the 152 that a large product reaches, 3.1 TB/s.
template <class T, bool Q8, int EPI, int RS, int NT, bool WIDE>
__global__ __launch_bounds__(256, 2) void linear_rows_kernel(LinearRows a) {
    constexpr int E = VEC<T>;
    constexpr int KC = CHUNK<T>;
    constexpr int CH = 2;                  // chunks of the contracted dimension a step
    constexpr int WL = (CH * NT + 3) / 4;  // fragment vectors of W a thread brings in
    constexpr int TG = KC / 16;
    constexpr int G = NT / TG;
    constexpr int VP = 16 * NT / E, PO = VP + 1;  // an output row's vectors, and its pitch in LDS
    constexpr int STEP = CH * NT * 64;            // fragment vectors of a step's weights
    constexpr int OUT = 4 * 16 * PO;
    __shared__ u32x4 lds[2 * STEP > OUT ? 2 * STEP : OUT];  // the weights' two buffers, then the outputs
    __shared__ float bias_lds[16 * NT];

    const Dealt at_tile = deal_block(blockIdx.x, a.row_blocks, a.n_tiles);
    const int n0 = at_tile.tile * 16 * NT;
    const int64_t first = (int64_t)at_tile.group * (64 * RS);
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int r = lane & 15, q = lane >> 4;
    const T* w = static_cast<const T*>(a.w);

    int64_t row[RS];
#pragma unroll
    for (int s = 0; s < RS; ++s) {
        const int64_t m = first + wave * (16 * RS) + 16 * s + r;
        row[s] = m < a.rows ? m : a.rows - 1;  // rows past the end repeat the last one and are not stored
    }
    if (tid < 16 * NT) {
        const int n = n0 + tid;
        bias_lds[tid] = a.bias && n < a.N ? to_f32(static_cast<const T*>(a.bias)[n]) : 0.0f;
    }

    u32x4 wr[WL];
    RowRaw<T, Q8, WIDE> xr[RS][CH];
    auto load = [&](int k0) {
#pragma unroll
        for (int i = 0; i < WL; ++i) {
            const int slot = i * 256 + tid;
            const int c = slot / (NT * 64), t = (slot / 64) % NT, l = slot & 63;
            const int n = n0 + tile_column<T>(t, l & 15);
            wr[i] = issue_row<T, WIDE>(w + (int64_t)(n < a.N ? n : a.N - 1) * a.K, k0 + c * KC + (l >> 4) * E, a.K);
        }
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int s = 0; s < RS; ++s) xr[s][c].issue(a.x, row[s], k0 + c * KC + q * E);
    };
    auto store = [&](int k0, int buffer) {
#pragma unroll
        for (int i = 0; i < WL; ++i) {
            const int slot = i * 256 + tid;
            if (CH * NT % 4 != 0 && slot >= CH * NT * 64) break;
            const int c = slot / (NT * 64), t = (slot / 64) % NT, l = slot & 63;
            const u32x4 v = finish_chunk<T, WIDE>(wr[i], k0 + c * KC, k0 + c * KC + (l >> 4) * E, a.K);
            lds[buffer * STEP + slot] = n0 + tile_column<T>(t, l & 15) < a.N ? v : u32x4{0u, 0u, 0u, 0u};
        }
    };

    f32x4 acc[RS][NT];
#pragma unroll
    for (int s = 0; s < RS; ++s)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[s][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    load(0);
    store(0, 0);
    int buffer = 0;
    for (int k0 = 0; k0 < a.K; k0 += CH * KC) {
        u32x4 xc[RS][CH];
#pragma unroll
        for (int s = 0; s < RS; ++s)
#pragma unroll
            for (int c = 0; c < CH; ++c)
                xc[s][c] = xr[s][c].finish_in(a.x, k0 + c * KC + KC <= a.K, k0 + c * KC + q * E);
        __syncthreads();
        const bool more = k0 + CH * KC < a.K;
        if (more) load(k0 + CH * KC);
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const u32x4 wf = lds[buffer * STEP + (c * NT + t) * 64 + lane];
#pragma unroll
                for (int s = 0; s < RS; ++s) acc[s][t] = multiply<T>(wf, xc[s][c], acc[s][t]);
            }
        buffer ^= 1;
        if (more) store(k0 + CH * KC, buffer);
    }

#pragma unroll
    for (int s = 0; s < RS; ++s) settle(acc[s]);
    T* y = static_cast<T*>(a.y);
    const T* other = static_cast<const T*>(a.other);
    const bool staged = a.N % E == 0;
    u32x4* strip = lds + wave * 16 * PO;
    __syncthreads();  // the weights' last readers are done
#pragma unroll
    for (int s = 0; s < RS; ++s) {
        const int64_t m = first + wave * (16 * RS) + 16 * s + r;
        const int64_t at_row = m < a.rows ? m : a.rows - 1;
        u32x4 o[G], low[G];
        if constexpr (EPI != 0) {
#pragma unroll
            for (int g = 0; g < G; ++g) o[g] = issue_row<T, WIDE>(other + at_row * a.ldo, n0 + g * KC + q * E, a.N);
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int at = g * KC + q * E;  // column within the block's tile
            float z[E];
#pragma unroll
            for (int i = 0; i < E; ++i) z[i] = acc[s][g * TG + i / 4][i & 3] + bias_lds[at + i];
            u32x4 raw = {0u, 0u, 0u, 0u};
            if constexpr (EPI != 0) raw = finish_chunk<T, WIDE>(o[g], n0 + g * KC, n0 + at, a.N);
            raw = linear_end<T, EPI, E>(a, z, raw, low[g]);
            if (staged) strip[r * PO + g * 4 + q] = raw;
            else if (m < a.rows) {
                store_chunk(y + m * a.ldy, n0 + g * KC, n0 + at, a.N, raw);
                if constexpr (KEEPS_LOW<T, EPI>) store_chunk(y + a.N + m * a.ldy, n0 + g * KC, n0 + at, a.N, low[g]);
            }
        }
        auto put = [&](T* to) {
            const int64_t top = m - r;
            if (top + 16 <= a.rows) store_strip<T, VP, PO>(strip, to, a.ldy, top, a.rows, n0, a.N, lane, Flag<true>{});
            else store_strip<T, VP, PO>(strip, to, a.ldy, top, a.rows, n0, a.N, lane, Flag<false>{});
        };
        if (staged) {
            put(y);
            if constexpr (KEEPS_LOW<T, EPI>) {
#pragma unroll
                for (int g = 0; g < G; ++g) strip[r * PO + g * 4 + q] = low[g];
                put(y + a.N);
            }
        }
    }
}

// The weights as the tile kernel takes them: fragments of W, or of W^T as often
// beside itself as K holds its `inner` columns, 64 columns (4 tiles) after 64,
// within them chunk by chunk, zero past N and K, so that a wavefront reads a
// fragment as 1 KB in a row.
template <class T, bool TRANSPOSED>
__global__ __launch_bounds__(256) void pack_weights_kernel(const T* __restrict__ w, int N, int K, int inner, int chunks,
                                                           u32x4* __restrict__ out) {
    constexpr int E = VEC<T>;
    const int slot = blockIdx.x * 256 + threadIdx.x;
    const int l = slot & 63, t = (slot >> 6) & 3, rest = slot >> 8;
    const int c = rest % chunks, n = rest / chunks * 64 + tile_column<T>(t, l & 15);
    const int k = c * CHUNK<T> + (l >> 4) * E;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (n < N) {
        if constexpr (!TRANSPOSED) {
            v = load_row(w + (int64_t)n * K, k, K);
        } else {
            float f[E];
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] = k + i < K ? to_f32(w[(int64_t)((k + i) % inner) * N + n]) : 0.0f;
            v = pack<T>(f);
        }
    }
    out[slot] = v;
}
template <class T>
static int64_t packed_vectors(int N, int K) {
    return (int64_t)((N + 63) / 64) * ((K + CHUNK<T> - 1) / CHUNK<T>) * 256;
}

// Longer contracted dimensions with many rows: a block of 4 wavefronts brings
// 64 whole rows of x into LDS and goes over all N columns: a wavefront takes 64
// of them at a time against the 64 rows (4 x 4 tiles), its fragments of W,
// packed, from the L2, where they stay.  After the rows have come the
// wavefronts never wait for one another.  268177 rows, 256 to 512 channels of
// bfloat16: 138 us, 509 TFLOP/s and 3.0 TB/s, a third and a half of what either
// reaches alone: a block's loads, products and activations follow one another,
// and only the 2 or 3 blocks that its LDS leaves room for overlap them.
template <class T, bool Q8, int EPI, int KCH>
__global__ __launch_bounds__(256, KCH > 8 || EPI != 0 ? 2 : 3)
void linear_tile_kernel(LinearRows a) {
    constexpr int E = VEC<T>;
    constexpr int KC = CHUNK<T>;
    constexpr int TG = KC / 16;
    constexpr int NT = 4, G = NT / TG;
    constexpr int PAD = sizeof(T) == 4 ? 1 : 2;
    constexpr int VK = KCH * 4, PK = VK + PAD;
    constexpr int VP = 16 * NT / E, PO = VP + PAD;
    constexpr int LP = 16 * VP / 64;
    constexpr int LK = 64 * VK / 256;    // vectors of x a thread brings in
    constexpr int LB = LK < 8 ? LK : 8;  // of which this many at a time
    __shared__ u32x4 x_lds[64 * PK];
    __shared__ u32x4 strip_lds[4][16 * PO];

    const int64_t first = (int64_t)blockIdx.x * 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int r = lane & 15, q = lane >> 4;
    const u32x4* w = static_cast<const u32x4*>(a.w);
    const T* bias = static_cast<const T*>(a.bias);
    const T* other = static_cast<const T*>(a.other);
    T* y = static_cast<T*>(a.y);
    u32x4* mine = strip_lds[wave];

#pragma unroll
    for (int b = 0; b < LK; b += LB) {
        RowRaw<T, Q8, true> xr[LB];
#pragma unroll
        for (int i = 0; i < LB; ++i) {
            const int u = (b + i) * 256 + tid;
            const int64_t m = first + u / VK < a.rows ? first + u / VK : a.rows - 1;
            xr[i].issue(a.x, m, u % VK * E);
        }
#pragma unroll
        for (int i = 0; i < LB; ++i) {
            const int u = (b + i) * 256 + tid;
            x_lds[u / VK * PK + u % VK] = xr[i].finish_in(a.x, VK * E <= a.K, u % VK * E);
        }
    }
    __syncthreads();

    const bool staged = a.N % E == 0;
    const int chunks = (a.K + KC - 1) / KC;
    for (int n0 = wave * 64; n0 < a.N; n0 += 256) {
        f32x4 acc[4][NT];
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[s][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const u32x4* from = w + (int64_t)(n0 / 64) * chunks * 256 + lane;
        u32x4 wa[NT], wb[NT];  // one chunk of W on its way while the other is multiplied
        auto fetch = [&](int c, u32x4 (&wf)[NT]) {
            const u32x4* p = from + (c < chunks ? c : chunks - 1) * 256;
#pragma unroll
            for (int t = 0; t < NT; ++t) wf[t] = p[t * 64];
        };
        auto step = [&](int c, const u32x4 (&wf)[NT]) {
            u32x4 xf[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) xf[s] = x_lds[(16 * s + r) * PK + c * 4 + q];
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[s][t] = multiply<T>(wf[t], xf[s], acc[s][t]);
        };
        fetch(0, wa);
        for (int c = 0; c < chunks; c += 2) {
            fetch(c + 1, wb);
            step(c, wa);
            fetch(c + 2, wa);
            if (c + 1 < chunks) step(c + 1, wb);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) settle(acc[s]);
        float add[G][E];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            if (bias) {
                unpack<T>(load_row(bias, n0 + g * KC + q * E, a.N), add[g]);
            } else {
#pragma unroll
                for (int i = 0; i < E; ++i) add[g][i] = 0.0f;
            }
        }
        u32x4 ahead[4][EPI != 0 ? LP : 1];  // all four strips' rows of dy or the residual at once
        if constexpr (EPI != 0) {
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int i = 0; i < LP; ++i) {
                    const int64_t at = first + 16 * s + i * (64 / VP) + lane / VP;
                    ahead[s][i] = issue_row<T, true>(other + (at < a.rows ? at : a.rows - 1) * a.ldo,
                                                     n0 + lane % VP * E, a.N);
                }
        }
        auto finish = [&](int s, auto whole) {
            const int64_t m0 = first + 16 * s, m = m0 + r;
            if constexpr (EPI != 0) {
                const u32x4 (&o)[LP] = ahead[s];
#pragma unroll
                for (int i = 0; i < LP; ++i) {
                    u32x4 v = o[i];
                    if (n0 + VP * E > a.N) v = finish_row<T, true>(v, n0 + lane % VP * E, a.N);
                    mine[(i * (64 / VP) + lane / VP) * PO + lane % VP] = v;
                }
                wave_fence();
            }
            u32x4 low[G];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float z[E];
#pragma unroll
                for (int i = 0; i < E; ++i) z[i] = acc[s][g * TG + i / 4][i & 3] + add[g][i];
                u32x4& slot = mine[r * PO + g * 4 + q];
                u32x4 raw = {0u, 0u, 0u, 0u};
                if constexpr (EPI != 0) raw = slot;
                raw = linear_end<T, EPI, E>(a, z, raw, low[g]);
                if (staged) slot = raw;
                else if (whole.value || m < a.rows) {
                    store_chunk(y + m * a.ldy, n0 + g * KC, n0 + g * KC + q * E, a.N, raw);
                    if constexpr (KEEPS_LOW<T, EPI>)
                        store_chunk(y + a.N + m * a.ldy, n0 + g * KC, n0 + g * KC + q * E, a.N, low[g]);
                }
            }
            if (staged) store_strip<T, VP, PO>(mine, y, a.ldy, m0, a.rows, n0, a.N, lane, whole);
            else wave_fence();
            if constexpr (KEEPS_LOW<T, EPI>) {
                if (staged) {
#pragma unroll
                    for (int g = 0; g < G; ++g) mine[r * PO + g * 4 + q] = low[g];
                    store_strip<T, VP, PO>(mine, y + a.N, a.ldy, m0, a.rows, n0, a.N, lane, whole);
                }
            }
        };
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            if (first + 16 * s + 16 <= a.rows) finish(s, Flag<true>{});
            else if (first + 16 * s < a.rows) finish(s, Flag<false>{});
        }
    }
}

// W^T, `times` beside itself.
template <class T>
__global__ __launch_bounds__(256) void transpose_kernel(const T* __restrict__ w, int n, int k, int times,
                                                        T* __restrict__ out) {
    __shared__ T tile[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    for (int i = ty; i < 32; i += 8) {
        const int row = blockIdx.y * 32 + i, col = blockIdx.x * 32 + tx;
        if (row < n && col < k) tile[i][tx] = w[(int64_t)row * k + col];
    }
    __syncthreads();
    for (int i = ty; i < 32; i += 8) {
        const int row = blockIdx.x * 32 + i, col = blockIdx.y * 32 + tx;
        if (row < k && col < n)
            for (int j = 0; j < times; ++j) out[((int64_t)row * times + j) * n + col] = tile[tx][i];
    }
}

struct LinearGradW {
    Rows x;
    const void* dz;
    bool split;       // a row of dz is N high halves, then N low ones
    int64_t ldz;
    int64_t rows, rows_per_split;
    int N, n_tiles, k_tiles, splits;
    float* part;     // splits x (N K + N)
    int K;
};

// dW tile of 32 A columns of dz x 32 B columns of x over one split's rows.
// The contracted dimension is the row, the slow one of both operands: they go
// to LDS as they are, row by row, and are read transposed.  2 x 2 wavefronts
// multiply 16 A x 16 B columns each.
template <class T, bool Q8, int A, int B, int PLANES>
__global__ __launch_bounds__(256, 2) void linear_gradw_kernel(LinearGradW a) {
    constexpr int E = VEC<T>;
    constexpr int KC = CHUNK<T>;
    constexpr int MR = 2 * KC;                       // rows a step
    constexpr int CZ = 32 * A / E, CX = 32 * B / E;  // vectors across dz's and x's tile
    constexpr int PAD = sizeof(T) == 4 ? 1 : 2;      // spreads rows over the banks
    constexpr int PZ = CZ + PAD, PX = CX + PAD;
    constexpr int LZ = (MR * CZ + 255) / 256, LX = (MR * CX + 255) / 256;
    __shared__ u32x4 z_lds[PLANES][MR * PZ];
    __shared__ u32x4 x_lds[MR * PX];

    const Dealt at_tile = deal_block(blockIdx.x, a.splits, a.n_tiles * a.k_tiles);
    const int split = at_tile.group, kt = at_tile.tile % a.k_tiles, nt = at_tile.tile / a.k_tiles;
    const int n0 = nt * 32 * A, k0 = kt * 32 * B;
    const int64_t begin = split * a.rows_per_split;
    const int64_t end = begin + a.rows_per_split < a.rows ? begin + a.rows_per_split : a.rows;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int r = lane & 15, q = lane >> 4;
    const int wn = wave >> 1, wk = wave & 1;
    const bool sum_bias = kt == 0 && wk == 0;
    const T* dz = static_cast<const T*>(a.dz);

    u32x4 zr[PLANES][LZ];
    RowRaw<T, Q8> xr[LX];
    auto load = [&](int64_t m0) {
#pragma unroll
        for (int i = 0; i < LZ; ++i) {
            const int u = i * 256 + tid;
            const int64_t m = m0 + u / CZ < end ? m0 + u / CZ : end - 1;
#pragma unroll
            for (int p = 0; p < PLANES; ++p) zr[p][i] = issue_row(dz + m * a.ldz + p * a.N, n0 + u % CZ * E, a.N);
        }
#pragma unroll
        for (int i = 0; i < LX; ++i) {
            const int u = i * 256 + tid;
            const int64_t m = m0 + u / CX < end ? m0 + u / CX : end - 1;
            xr[i].issue(a.x, m, k0 + u % CX * E);
        }
    };
    auto store = [&](int64_t m0) {
#pragma unroll
        for (int i = 0; i < LZ; ++i) {
            const int u = i * 256 + tid;
#pragma unroll
            for (int p = 0; p < PLANES; ++p) {
                const u32x4 v = finish_row<T>(zr[p][i], n0 + u % CZ * E, a.N);
                if (MR * CZ % 256 == 0 || u < MR * CZ)
                    z_lds[p][u / CZ * PZ + u % CZ] = m0 + u / CZ < end ? v : u32x4{0u, 0u, 0u, 0u};
            }
        }
#pragma unroll
        for (int i = 0; i < LX; ++i) {
            const int u = i * 256 + tid;
            const u32x4 v = xr[i].finish(a.x, k0 + u % CX * E);
            if (MR * CX % 256 == 0 || u < MR * CX)
                x_lds[u / CX * PX + u % CX] = m0 + u / CX < end ? v : u32x4{0u, 0u, 0u, 0u};
        }
    };

    f32x4 acc[A][B], acc_b[A];
#pragma unroll
    for (int i = 0; i < A; ++i) {
        acc_b[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < B; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    float one[E];
#pragma unroll
    for (int i = 0; i < E; ++i) one[i] = 1.0f;
    const u32x4 ones = pack<T>(one);

    if (begin < end) load(begin);
    for (int64_t m0 = begin; m0 < end; m0 += MR) {
        __syncthreads();
        store(m0);
        __syncthreads();
        if (m0 + MR < end) load(m0 + MR);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            u32x4 fx[B];
#pragma unroll
            for (int j = 0; j < B; ++j) fx[j] = read_transposed<T, false>(x_lds, PX, c * KC, wk * B + j, lane);
#pragma unroll
            for (int p = 0; p < PLANES; ++p) {
                u32x4 fz[A];
#pragma unroll
                for (int i = 0; i < A; ++i) fz[i] = read_transposed<T, false>(z_lds[p], PZ, c * KC, wn * A + i, lane);
#pragma unroll
                for (int i = 0; i < A; ++i)
#pragma unroll
                    for (int j = 0; j < B; ++j) acc[i][j] = multiply<T>(fz[i], fx[j], acc[i][j]);
                if (sum_bias) {
#pragma unroll
                    for (int i = 0; i < A; ++i) acc_b[i] = multiply<T>(fz[i], ones, acc_b[i]);
                    settle(acc_b);
                }
            }
        }
    }

#pragma unroll
    for (int i = 0; i < A; ++i) settle(acc[i]);
    settle(acc_b);
    float* part = a.part + split * ((int64_t)a.N * a.K + a.N);
#pragma unroll
    for (int i = 0; i < A; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int n = n0 + (wn * A + i) * 16 + 4 * q + e;
            if (n >= a.N) continue;
#pragma unroll
            for (int j = 0; j < B; ++j) {
                const int k = k0 + (wk * B + j) * 16 + r;
                if (k < a.K) part[(int64_t)n * a.K + k] = acc[i][j][e];
            }
            if (sum_bias && r == 0) part[(int64_t)a.N * a.K + n] = acc_b[i][e];
        }
}

// Sums over the splits, in a fixed order: a block takes 32 outputs, 8 lanes
// each for every eighth split.  The first `weights` outputs are dW's, the rest db's.
template <class T>
__global__ __launch_bounds__(256) void sum_splits_kernel(const float* __restrict__ part, int splits, int64_t weights,
                                                         int64_t count, T* __restrict__ dw, T* __restrict__ db) {
    __shared__ float lds[8][32];
    const int col = threadIdx.x & 31, lane = threadIdx.x >> 5;
    const int64_t i = (int64_t)blockIdx.x * 32 + col;
    float total = 0.0f;
    if (i < count) {
#pragma unroll 8
        for (int s = lane; s < splits; s += 8) total += part[(int64_t)s * count + i];
    }
    lds[lane][col] = total;
    __syncthreads();
    if (lane == 0 && i < count) {
#pragma unroll
        for (int k = 1; k < 8; ++k) total += lds[k][col];
        if (i < weights) {
            if (dw) dw[i] = (T)total;
        } else if (db) {
            db[i - weights] = (T)total;
        }
    }
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
// Widths in powers of two: chunks of the contracted dimension, 16-column tiles.
template <class T>
static int chunks_of(int channels) {
    const int chunks = (channels + CHUNK<T> - 1) / CHUNK<T>;
    return chunks <= 1 ? 1 : chunks <= 2 ? 2 : chunks <= 4 ? 4 : 8;
}

template <class T, bool Q8, int EPI, int KCH, int NT, bool WIDE>
static void launch_stream_as(LinearRows a, hipStream_t stream) {
    a.n_tiles = (a.N + 16 * NT - 1) / (16 * NT);
    // 512 rows a block at most, fewer where that would leave less than eight
    // blocks a compute unit: a block reads its weights once.
    int64_t strips = a.rows * a.n_tiles / (16 * 2048) / 4 * 4;
    a.strips = (int)(strips < 4 ? 4 : strips > 32 ? 32 : strips);
    a.row_blocks = (int)((a.rows + 16 * a.strips - 1) / (16 * a.strips));
    hipLaunchKernelGGL((linear_stream_kernel<T, Q8, EPI, KCH, NT, WIDE>), dim3((unsigned)a.row_blocks * a.n_tiles),
                       dim3(256), 0, stream, a);
}
template <class T, bool Q8, int EPI, int RS, int NT, bool WIDE>
static void launch_long_as(LinearRows a, hipStream_t stream) {
    a.n_tiles = (a.N + 16 * NT - 1) / (16 * NT);
    a.row_blocks = (int)((a.rows + 64 * RS - 1) / (64 * RS));
    hipLaunchKernelGGL((linear_rows_kernel<T, Q8, EPI, RS, NT, WIDE>), dim3((unsigned)a.row_blocks * a.n_tiles),
                       dim3(256), 0, stream, a);
}

// Few rows: narrow column tiles, so that many compute units read the weights
// at once.  Narrow and wide (us, bfloat16): 300 rows, 512 to 512 channels 6.2
// and 18.2; 4096 rows 13.3 and 19.2, 32 to 512 3.8 and 4.3, 256 to 64 4.1 and
// 8.3, float 512 to 512 25.7 and 43.0; 8192 rows 24.3 and 19.5, 5.5 and 5.3, 4.3
// and 8.5, 48.0 and 44.9.
static bool few_rows(const LinearRows& a) { return a.rows <= 4096; }

// The tile's width: 128 columns read a row once, 64 leave a float tile's LDS
// room for twice the wavefronts (1.44 M rows of float, 32 to 128 channels: 224
// us at 64 columns, 260 at 128; 33 to 97: 242 and 308; 32 to 97: 268 and 256).
template <class T, bool Q8, int EPI, int KCH>
static void launch_stream(const LinearRows& a, hipStream_t stream) {
    constexpr int E = VEC<T>, MOST = sizeof(T) == 4 ? 4 : 8;
    if (a.K < E || a.N < E) {  // rows shorter than a vector, in or out
        if (a.N <= 32 || few_rows(a)) return launch_stream_as<T, Q8, EPI, KCH, 2, false>(a, stream);
        if constexpr (KCH == 1) return launch_stream_as<T, Q8, EPI, 1, MOST, false>(a, stream);
    }
    if (a.N <= 32 || few_rows(a)) launch_stream_as<T, Q8, EPI, KCH, 2, true>(a, stream);
    else if (a.N <= 64) launch_stream_as<T, Q8, EPI, KCH, 4, true>(a, stream);
    else launch_stream_as<T, Q8, EPI, KCH, MOST, true>(a, stream);
}
// Products that the tile kernel takes: of 16-bit types, more than 4 chunks of K,
// as many as a block's rows find room for, enough rows to fill the blocks, and
// enough columns for all four wavefronts of one.  It and the rows kernel in its
// place (us, packing included, bfloat16): 268177 rows, 256 to 512 channels 127
// and 167; 200000 rows, 512 to 512 171 and 216, 512 to 129 93 and 135, 512 to 256
// 104 and 119, 256 to 256 61 and 63, 160 to 300 66 and 59; 32768 rows 37 and 44,
// 25 and 30, 27 and 27, 22 and 20, 23 and 19; 16384 rows 21 and 20, 13 and 15,
// 14 and 15, 10 and 9, 12 and 9; narrower outputs, 500000 rows, 512 to 128 206
// and 158, 1.92 M rows, 512 to 64 686 and 457.  Float's rows take twice the LDS:
// 1.44 M rows, 128 to 64: 529 and 365.
template <class T>
static bool tile_rows(int64_t rows, int K) {
    return sizeof(T) == 2 && K > 4 * CHUNK<T> && K <= 512 && rows >= 32768;
}
template <class T>
static bool tiled(int64_t rows, int K, int N) {
    return tile_rows<T>(rows, K) && N > 128;
}
template <class T, bool Q8, int EPI, int KCH>
static void launch_tile(const LinearRows& a, hipStream_t stream) {
    hipLaunchKernelGGL((linear_tile_kernel<T, Q8, EPI, KCH>), dim3((unsigned)((a.rows + 63) / 64)), dim3(256), 0,
                       stream, a);
}
template <class T, bool Q8, int EPI>
static void launch_long(const LinearRows& a, hipStream_t stream) {
    if (a.N < VEC<T>) return launch_long_as<T, Q8, EPI, 1, 2, false>(a, stream);
    if (few_rows(a)) return launch_long_as<T, Q8, EPI, 1, 2, true>(a, stream);
    if (a.N <= 64) launch_long_as<T, Q8, EPI, 4, 4, true>(a, stream);
    else launch_long_as<T, Q8, EPI, 2, 8, true>(a, stream);
}
// `packed`: room for the packed weights where the tile kernel takes the
// product; TRANSPOSED: a.w is K / times x N.
template <class T, bool Q8, int EPI, bool TRANSPOSED>
static void launch_rows(LinearRows a, void* packed, hipStream_t stream, int times = 1) {
    if constexpr (sizeof(T) == 2) {
        if (tiled<T>(a.rows, a.K, a.N)) {
            const int64_t vectors = packed_vectors<T>(a.N, a.K);
            const int chunks = (a.K + CHUNK<T> - 1) / CHUNK<T>;
            hipLaunchKernelGGL((pack_weights_kernel<T, TRANSPOSED>), dim3((unsigned)(vectors / 256)), dim3(256), 0,
                               stream, static_cast<const T*>(a.w), a.N, a.K, a.K / times, chunks,
                               static_cast<u32x4*>(packed));
            a.w = packed;
            if (chunks <= 8) return launch_tile<T, Q8, EPI, 8>(a, stream);
            return launch_tile<T, Q8, EPI, 16>(a, stream);
        }
    }
    if constexpr (TRANSPOSED) {
        T* wt = static_cast<T*>(packed);
        const int inner = a.K / times;
        hipLaunchKernelGGL(transpose_kernel<T>, dim3((a.N + 31) / 32, (inner + 31) / 32), dim3(256), 0, stream,
                           static_cast<const T*>(a.w), inner, a.N, times, wt);
        a.w = wt;
    }
    switch (chunks_of<T>(a.K)) {
        case 1: return launch_stream<T, Q8, EPI, 1>(a, stream);
        case 2: return launch_stream<T, Q8, EPI, 2>(a, stream);
        case 4: return launch_stream<T, Q8, EPI, 4>(a, stream);
        default: return launch_long<T, Q8, EPI>(a, stream);
    }
}

template <class T, bool Q8, int A, int B>
static void launch_gradw_as(const LinearGradW& a, int splits, hipStream_t stream) {
    const dim3 grid((unsigned)(a.n_tiles * a.k_tiles * splits));
    if constexpr (SPLIT<T>) {
        if (a.split) {
            hipLaunchKernelGGL((linear_gradw_kernel<T, Q8, A, B, 2>), grid, dim3(256), 0, stream, a);
            return;
        }
    }
    hipLaunchKernelGGL((linear_gradw_kernel<T, Q8, A, B, 1>), grid, dim3(256), 0, stream, a);
}
template <class T, bool Q8, int A>
static void launch_gradw_b(const LinearGradW& a, int splits, hipStream_t stream) {
    if (a.K <= 32) launch_gradw_as<T, Q8, A, 1>(a, splits, stream);
    else if (a.K <= 64) launch_gradw_as<T, Q8, A, 2>(a, splits, stream);
    else launch_gradw_as<T, Q8, A, 4>(a, splits, stream);
}
template <class T, bool Q8>
static void launch_gradw(const LinearGradW& a, int splits, hipStream_t stream) {
    if (a.N <= 32) launch_gradw_b<T, Q8, 1>(a, splits, stream);
    else if (a.N <= 64) launch_gradw_b<T, Q8, 2>(a, splits, stream);
    else launch_gradw_b<T, Q8, 4>(a, splits, stream);
}

// How the rows of a backward pass are split: the fused kernel's blocks, or the
// weight gradient's splits.
struct BwdPlan {
    bool fused;
    int splits, n_tiles, k_tiles;
    int64_t rows_per_split;
};
static int gradw_tiles(int n) { return n <= 32 ? 1 : n <= 64 ? 1 : (n + 127) / 128; }
template <class T>
static BwdPlan bwd_plan(int64_t rows, int K, int N) {
    BwdPlan p;
    p.fused = fused_fits<T>(K, N);
    p.n_tiles = p.fused ? 1 : gradw_tiles(N);
    p.k_tiles = p.fused ? 1 : gradw_tiles(K);
    // Two blocks per compute unit in all, and 64 rows a block at least.
    int64_t splits = 512 / (p.n_tiles * p.k_tiles);
    const int64_t most = (rows + 63) / 64;
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    p.rows_per_split = ((rows + splits - 1) / splits + 63) / 64 * 64;
    if (p.rows_per_split < 64) p.rows_per_split = 64;
    p.splits = (int)((rows + p.rows_per_split - 1) / p.rows_per_split);
    if (p.splits < 1) p.splits = 1;
    return p;
}

static size_t aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }

// Scratch of the backward pass of a call that wants dW or db (params) and dx,
// of a product that ends in an activation or not: the splits' dW and db; unless
// it is fused also dz, its rows twice as long where it is split, and W^T, as
// often.  Without an activation dz is the upstream gradient itself.
struct BwdScratch {
    size_t part, dz, wt, total;
};
template <class T>
static BwdScratch bwd_scratch(int64_t rows, int K, int N, bool act, bool params, bool dx) {
    const BwdPlan p = bwd_plan<T>(rows, K, N);
    BwdScratch s;
    s.part = 0;
    s.dz = params ? aligned((size_t)p.splits * ((size_t)N * K + N) * 4) : 0;
    const int halves = SPLIT<T> && act ? 2 : 1;
    s.wt = s.dz + (act && !p.fused ? aligned((size_t)rows * N * halves * sizeof(T)) : 0);
    // W^T as it is, or packed; W packed in its place before.
    const int64_t forward = act ? packed_vectors<T>(N, K) : 0, back = dx ? packed_vectors<T>(K, N * halves) : 0;
    s.total = s.wt + (p.fused ? 0 : aligned((size_t)(forward > back ? forward : back) * 16));
    return s;
}

// The forward's scratch, asked for by rows and K alone.
template <class T>
static size_t fwd_bytes(int64_t rows, int K, int N) {
    return tile_rows<T>(rows, K) ? (size_t)packed_vectors<T>(N, K) * 16 : 0;
}

template <class T>
static int linear_fwd(const gs3d_linear_args& g, void* scratch, hipStream_t stream) {
    LinearRows a{};
    a.x = Rows{g.x, g.x_stride, {}, g.inner};
    a.w = g.weight, a.bias = g.bias, a.other = g.residual, a.ldo = g.residual_stride, a.y = g.y;
    a.rows = g.rows, a.K = g.inner, a.N = g.outer, a.ldy = g.outer, a.act = g.activation;
    // The stream kernel keeps the rows as it reads them.
    if (g.codes && chunks_of<T>(a.K) <= 4) a.keep_codes = g.codes, a.keep_scales = g.scales;
    else if (g.codes) quantize_rows(g.x, g.x_stride, g.rows, g.inner, g.dtype, g.codes, g.scales, stream);
    if (g.residual) launch_rows<T, false, 2, false>(a, scratch, stream);
    else launch_rows<T, false, 0, false>(a, scratch, stream);
    return launch_status("gs3d_linear_fwd");
}

template <class T, bool Q8>
static int linear_bwd(const gs3d_linear_bwd_args& g, char* scratch, hipStream_t stream) {
    const BwdPlan p = bwd_plan<T>(g.rows, g.inner, g.outer);
    const bool params = g.grad_weight || g.grad_bias;
    const BwdScratch at =
        bwd_scratch<T>(g.rows, g.inner, g.outer, g.activation != GS3D_ACT_NONE, params, g.grad_x != nullptr);
    // Without an activation only dW sees the input.  Where neither is wanted the
    // caller may not have it: a row of the weights then stands in for every
    // row, and the dW that comes of it is dropped.
    const bool seen = g.grad_weight || g.activation != GS3D_ACT_NONE;
    if (!seen && Q8) return linear_bwd<T, false>(g, scratch, stream);
    const Rows x{seen ? g.x : g.weight, seen ? g.x_stride : 0, {g.codes, g.scales, g.inner}, g.inner};
    float* part = reinterpret_cast<float*>(scratch + at.part);
    int splits = p.splits;
    if (g.rows == 0) {
        splits = 0;  // the parameters' gradients are sums of nothing, and no tensor has to be there
    } else if (p.fused) {
        LinearFused a{x, g.weight, g.bias, g.upstream, g.upstream_stride, g.grad_x, params ? part : nullptr,
                      g.rows, p.rows_per_split, g.inner, g.outer, g.activation, &splits};
        fused_launch<T>(a, Q8, p.splits, stream);
    } else {
        const void* dz = g.upstream;
        int64_t ldz = g.upstream_stride;
        const int halves = SPLIT<T> && g.activation != GS3D_ACT_NONE ? 2 : 1;  // of dz
        if (g.activation != GS3D_ACT_NONE) {
            LinearRows a{};
            a.x = x, a.w = g.weight, a.bias = g.bias, a.other = g.upstream, a.ldo = g.upstream_stride;
            a.y = scratch + at.dz, a.ldy = (int64_t)halves * g.outer;
            a.rows = g.rows, a.K = g.inner, a.N = g.outer, a.act = g.activation;
            launch_rows<T, Q8, 1, false>(a, scratch + at.wt, stream);
            dz = a.y, ldz = a.ldy;
        }
        if (g.grad_x) {
            LinearRows a{};
            a.x = Rows{dz, ldz, {}, halves * g.outer}, a.w = g.weight, a.y = g.grad_x, a.ldy = g.inner;
            a.rows = g.rows, a.K = halves * g.outer, a.N = g.inner, a.act = GS3D_ACT_NONE;
            launch_rows<T, false, 0, true>(a, scratch + at.wt, stream, halves);
        }
        if (params) {
            LinearGradW a{x, dz, halves == 2, ldz, g.rows, p.rows_per_split, g.outer, p.n_tiles, p.k_tiles, p.splits,
                          part, g.inner};
            launch_gradw<T, Q8>(a, p.splits, stream);
        }
    }
    if (params) {
        const int64_t weights = (int64_t)g.outer * g.inner, count = weights + g.outer;
        hipLaunchKernelGGL(sum_splits_kernel<T>, dim3(blocks_for(count, 32)), dim3(256), 0, stream, part, splits,
                           weights, count, static_cast<T*>(g.grad_weight), static_cast<T*>(g.grad_bias));
    }
    return launch_status("gs3d_linear_bwd");
}

}  // namespace gs3d
