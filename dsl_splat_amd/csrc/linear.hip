// Per-pixel products of the feature decoder: y = act(x W^T + b) + r and its
// gradients, over rows x (pixels) that are many and channels that are few.
//
//   linear_rows_kernel   rows times weights, for the forward (EPI 0), for
//                        dz = dy act'(x W^T + b) (EPI 1, z computed again
//                        rather than kept) and for dx = dz W (EPI 0 with W^T)
//   linear_gradw_kernel  dW = dz^T x and db = sum dz, split over the rows
//   sum_splits_kernel    the splits' partial sums in a fixed order
//
// Products of 16-bit types go through matrix instructions with sums in 32
// bits.  dz is rounded to the element type once, as the operand of the two
// products that follow it.
#include "decode.hpp"

namespace gs3d {

struct LinearRows {
    const void* x;       // rows x K, or NULL: q8
    int64_t ldx;
    Q8Rows q8;
    const void* w;       // N x K
    const void* bias;    // N or NULL
    const void* other;   // EPI 0: residual or NULL; EPI 1: dy
    int64_t ldo;
    void* y;
    int64_t ldy;
    int64_t rows;
    int K, N, act, n_tiles;
};

// Column of W's tile row r of tile t.  A lane ends up with rows 4q..4q+3 of
// every tile; for 16-bit types two tiles are dealt out so that their eight
// values are neighbours, 16 bytes of an output row.
template <class T>
GS3D_DEV int tile_column(int t, int r) {
    if constexpr (sizeof(T) == 4) return 16 * t + r;
    return 32 * (t >> 1) + 8 * (r >> 2) + 4 * (t & 1) + (r & 3);
}

// A block of 4 wavefronts computes 64 RS rows x 16 NT columns.  W's fragments
// go through LDS in fragment order (one 1 KB run per tile and chunk, read
// without conflicts) and serve the four wavefronts; a wavefront reads its own
// rows of x straight into fragments, 64 bytes of a row at a time.  The next
// step's operands are loaded while this step's are multiplied.
template <class T, bool Q8, int EPI, int RS, int NT>
__global__ __launch_bounds__(256) void linear_rows_kernel(LinearRows a) {
    constexpr int E = VEC<T>;
    constexpr int KC = CHUNK<T>;
    constexpr int CH = 2;               // chunks of the contracted dimension a step
    constexpr int WL = CH * NT / 4;     // fragments of W a thread brings in
    constexpr int TG = 4 * E / 16;      // tiles of a lane's 16-byte output vector
    __shared__ u32x4 w_lds[CH * NT * 64];
    __shared__ float bias_lds[16 * NT];

    // Blocks b, b + 8, b + 16, ... run on one XCD: the column tiles of a row
    // block are dealt to one of them, whose L2 then holds x once.
    const int64_t local = blockIdx.x >> 3;
    const int64_t row_block = (local / a.n_tiles) * 8 + (blockIdx.x & 7);
    const int n0 = (int)(local % a.n_tiles) * 16 * NT;
    const int64_t first = row_block * (64 * RS);
    if (first >= a.rows) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, q = lane >> 4;
    const T* w = static_cast<const T*>(a.w);
    const T* x = static_cast<const T*>(a.x);

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

    u32x4 wr[WL], xr[RS][CH];
    auto load = [&](int k0) {
#pragma unroll
        for (int i = 0; i < WL; ++i) {
            const int slot = i * 256 + tid;
            const int c = slot / (NT * 64), t = (slot / 64) % NT, l = slot & 63;
            const int n = n0 + tile_column<T>(t, l & 15);
            const int k = k0 + c * KC + (l >> 4) * E;
            wr[i] = n < a.N ? load_row(w + (int64_t)n * a.K, k, a.K) : u32x4{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int s = 0; s < RS; ++s) {
                const int k = k0 + c * KC + q * E;
                if constexpr (Q8) xr[s][c] = load_row_q8<T>(a.q8, row[s], k);
                else xr[s][c] = load_row(x + row[s] * a.ldx, k, a.K);
            }
    };

    f32x4 acc[RS][NT];
#pragma unroll
    for (int s = 0; s < RS; ++s)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[s][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    load(0);
    for (int k0 = 0; k0 < a.K; k0 += CH * KC) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WL; ++i) w_lds[i * 256 + tid] = wr[i];
        u32x4 xc[RS][CH];
#pragma unroll
        for (int s = 0; s < RS; ++s)
#pragma unroll
            for (int c = 0; c < CH; ++c) xc[s][c] = xr[s][c];
        __syncthreads();
        if (k0 + CH * KC < a.K) load(k0 + CH * KC);
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const u32x4 wf = w_lds[(c * NT + t) * 64 + lane];
#pragma unroll
                for (int s = 0; s < RS; ++s) acc[s][t] = multiply<T>(wf, xc[s][c], acc[s][t]);
            }
    }

    T* y = static_cast<T*>(a.y);
    const T* other = static_cast<const T*>(a.other);
#pragma unroll
    for (int s = 0; s < RS; ++s) {
        const int64_t m = first + wave * (16 * RS) + 16 * s + r;
        if (m >= a.rows) continue;
#pragma unroll
        for (int g = 0; g < NT / TG; ++g) {
            const int at = g * 16 * TG + q * E;  // column within the block's tile
            const int n = n0 + at;
            if (n >= a.N) continue;
            float z[E], o[E];
#pragma unroll
            for (int i = 0; i < E; ++i) z[i] = acc[s][g * TG + i / 4][i & 3] + bias_lds[at + i];
            if (EPI == 1 || other) unpack<T>(load_row(other + m * a.ldo, n, a.N), o);
            if constexpr (EPI == 1) {
#pragma unroll
                for (int i = 0; i < E; ++i) z[i] = o[i] * slope(z[i], a.act);
            } else {
#pragma unroll
                for (int i = 0; i < E; ++i) z[i] = activate(z[i], a.act);
                if (other) {
#pragma unroll
                    for (int i = 0; i < E; ++i) z[i] += o[i];
                }
            }
            store_row(y + m * a.ldy, n, a.N, pack<T>(z));
        }
    }
}

template <class T>
__global__ __launch_bounds__(256) void transpose_kernel(const T* __restrict__ w, int n, int k, T* __restrict__ out) {
    __shared__ T tile[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    for (int i = ty; i < 32; i += 8) {
        const int row = blockIdx.y * 32 + i, col = blockIdx.x * 32 + tx;
        if (row < n && col < k) tile[i][tx] = w[(int64_t)row * k + col];
    }
    __syncthreads();
    for (int i = ty; i < 32; i += 8) {
        const int row = blockIdx.x * 32 + i, col = blockIdx.y * 32 + tx;
        if (row < k && col < n) out[(int64_t)row * n + col] = tile[tx][i];
    }
}

struct LinearGradW {
    const void* x;
    int64_t ldx;
    Q8Rows q8;
    const void* dz;
    int64_t ldz;
    int64_t rows, rows_per_split;
    int K, N, n_tiles, k_tiles, splits;
    float* part_w;  // splits x N x K, or NULL
    float* part_b;  // splits x N, or NULL
};

// E x E elements in registers, row i in v[i], to their transpose (VEC<T>
// rows of one column each become one fragment vector).
GS3D_DEV void transpose_unit(u32x4 (&v)[4]) {
    const u32x4 a = v[0], b = v[1], c = v[2], d = v[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = u32x4{a[i], b[i], c[i], d[i]};
}
GS3D_DEV void transpose_unit(u32x4 (&v)[8]) {
    u32x4 o[8];
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            // Rows 2p, 2p+1 of columns 2w, 2w+1.
            o[2 * w][p] = __builtin_amdgcn_perm(v[2 * p + 1][w], v[2 * p][w], 0x05040100u);
            o[2 * w + 1][p] = __builtin_amdgcn_perm(v[2 * p + 1][w], v[2 * p][w], 0x07060302u);
        }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = o[i];
}

// dW tile of 32 A columns of dz x 32 B columns of x over one split's rows.
// The contracted dimension is the row, which both operands have as their slow
// one: a thread loads VEC rows of 16 bytes, transposes them in registers and
// writes fragment vectors to LDS, so the reads are whole fragments.  2 x 2
// wavefronts each multiply 16 A x 16 B columns.
template <class T, bool Q8, int A, int B>
__global__ __launch_bounds__(256) void linear_gradw_kernel(LinearGradW a) {
    constexpr int E = VEC<T>;
    constexpr int MR = 8 * E;                       // rows a step: two chunks
    constexpr int CZ = 32 * A / E, CX = 32 * B / E; // units across dz's and x's tile
    constexpr int UNITS = 8 * (CZ + CX);
    constexpr int PER = (UNITS + 255) / 256;
    __shared__ u32x4 lds[2 * (2 * A + 2 * B) * 64];
    u32x4* lds_z = lds;
    u32x4* lds_x = lds + 2 * 2 * A * 64;

    int64_t b = blockIdx.x;
    const int kt = (int)(b % a.k_tiles);
    b /= a.k_tiles;
    const int nt = (int)(b % a.n_tiles);
    const int split = (int)(b / a.n_tiles);
    const int n0 = nt * 32 * A, k0 = kt * 32 * B;
    const int64_t begin = split * a.rows_per_split;
    const int64_t end = begin + a.rows_per_split < a.rows ? begin + a.rows_per_split : a.rows;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, q = lane >> 4;
    const int wn = wave >> 1, wk = wave & 1;
    const bool sum_bias = a.part_b && kt == 0 && wk == 0;
    const T* x = static_cast<const T*>(a.x);
    const T* dz = static_cast<const T*>(a.dz);

    u32x4 v[PER][E];
    auto load = [&](int64_t m0) {
#pragma unroll
        for (int p = 0; p < PER; ++p) {
            const int u = p * 256 + tid;
            if (UNITS % 256 == 0 || u < UNITS) {
                const bool of_z = u < 8 * CZ;
                const int w = of_z ? u : u - 8 * CZ;
                const int across = of_z ? CZ : CX;
                const int group = w / across, cg = w % across;
                const int64_t m = m0 + group * E;
                const int col = (of_z ? n0 : k0) + cg * E;
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    if (m + i >= end) v[p][i] = u32x4{0u, 0u, 0u, 0u};
                    else if (of_z) v[p][i] = load_row(dz + (m + i) * a.ldz, col, a.N);
                    else if constexpr (Q8) v[p][i] = load_row_q8<T>(a.q8, m + i, col);
                    else v[p][i] = load_row(x + (m + i) * a.ldx, col, a.K);
                }
            }
        }
    };
    // Slot of column j of a tile row: chunk, tile, then lane.  The lane is
    // swizzled by the tile so that the lanes of a store, whose columns are a
    // whole vector apart, reach different banks.
    auto store = [&]() {
#pragma unroll
        for (int p = 0; p < PER; ++p) {
            const int u = p * 256 + tid;
            if (UNITS % 256 == 0 || u < UNITS) {
                transpose_unit(v[p]);
                const bool of_z = u < 8 * CZ;
                const int w = of_z ? u : u - 8 * CZ;
                const int across = of_z ? CZ : CX;
                const int tiles = of_z ? 2 * A : 2 * B;
                const int group = w / across, cg = w % across;
                u32x4* base = of_z ? lds_z : lds_x;
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    const int col = cg * E + j, t = col >> 4;
                    base[((group >> 2) * tiles + t) * 64 + (((group & 3) * 16 + (col & 15)) ^ (t & (E - 1)))] = v[p][j];
                }
            }
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
        store();
        __syncthreads();
        if (m0 + MR < end) load(m0 + MR);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            u32x4 fz[A], fx[B];
#pragma unroll
            for (int i = 0; i < A; ++i) {
                const int t = wn * A + i;
                fz[i] = lds_z[(c * 2 * A + t) * 64 + (lane ^ (t & (E - 1)))];
            }
#pragma unroll
            for (int j = 0; j < B; ++j) {
                const int t = wk * B + j;
                fx[j] = lds_x[(c * 2 * B + t) * 64 + (lane ^ (t & (E - 1)))];
            }
#pragma unroll
            for (int i = 0; i < A; ++i)
#pragma unroll
                for (int j = 0; j < B; ++j) acc[i][j] = multiply<T>(fz[i], fx[j], acc[i][j]);
            if (sum_bias) {
#pragma unroll
                for (int i = 0; i < A; ++i) acc_b[i] = multiply<T>(fz[i], ones, acc_b[i]);
            }
        }
    }

#pragma unroll
    for (int i = 0; i < A; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int n = n0 + (wn * A + i) * 16 + 4 * q + e;
            if (n >= a.N) continue;
            if (a.part_w) {
#pragma unroll
                for (int j = 0; j < B; ++j) {
                    const int k = k0 + (wk * B + j) * 16 + r;
                    if (k < a.K) a.part_w[((int64_t)split * a.N + n) * a.K + k] = acc[i][j][e];
                }
            }
            if (sum_bias && r == 0) a.part_b[(int64_t)split * a.N + n] = acc_b[i][e];
        }
}

// out[i] = sum over the splits of part[s][i], in order.
template <class T>
__global__ __launch_bounds__(256) void sum_splits_kernel(const float* __restrict__ part, int splits, int64_t count,
                                                         T* __restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= count) return;
    float total = 0.0f;
    for (int s = 0; s < splits; ++s) total += part[(int64_t)s * count + i];
    out[i] = (T)total;
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
template <class T, bool Q8, int EPI, int RS, int NT>
static void launch_rows_as(LinearRows a, hipStream_t stream) {
    a.n_tiles = (a.N + 16 * NT - 1) / (16 * NT);
    const int64_t row_blocks = (a.rows + 64 * RS - 1) / (64 * RS);
    const int64_t blocks = (row_blocks + 7) / 8 * 8 * a.n_tiles;
    hipLaunchKernelGGL((linear_rows_kernel<T, Q8, EPI, RS, NT>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
}

template <class T, bool Q8, int EPI>
static void launch_rows(const LinearRows& a, hipStream_t stream) {
    // Few rows: narrow column tiles, so that the weights are read by many
    // compute units at once.
    const bool few = a.rows <= 1024;
    if (a.N <= 32 || few) launch_rows_as<T, Q8, EPI, 1, 2>(a, stream);
    else if (a.N <= 64) launch_rows_as<T, Q8, EPI, 2, 4>(a, stream);
    else launch_rows_as<T, Q8, EPI, 2, 8>(a, stream);
}

template <class T, bool Q8, int A, int B>
static void launch_gradw_as(LinearGradW a, hipStream_t stream) {
    hipLaunchKernelGGL((linear_gradw_kernel<T, Q8, A, B>), dim3((unsigned)(a.n_tiles * a.k_tiles * a.splits)),
                       dim3(256), 0, stream, a);
}

static int gradw_width(int n) { return n <= 32 ? 1 : n <= 64 ? 2 : 4; }

struct GradWPlan {
    int n_tiles, k_tiles, splits;
    int64_t rows_per_split;
};
static GradWPlan gradw_plan(int64_t rows, int K, int N) {
    GradWPlan p;
    const int A = gradw_width(N), B = gradw_width(K);
    p.n_tiles = (N + 32 * A - 1) / (32 * A);
    p.k_tiles = (K + 32 * B - 1) / (32 * B);
    // About two blocks per compute unit in all, and 256 rows a split at least.
    int64_t splits = 512 / (p.n_tiles * p.k_tiles);
    const int64_t most = (rows + 255) / 256;
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    p.rows_per_split = ((rows + splits - 1) / splits + 63) / 64 * 64;
    if (p.rows_per_split < 64) p.rows_per_split = 64;
    p.splits = (int)((rows + p.rows_per_split - 1) / p.rows_per_split);
    if (p.splits < 1) p.splits = 1;
    return p;
}

template <class T, bool Q8, int A>
static void launch_gradw_b(const LinearGradW& a, hipStream_t stream) {
    switch (gradw_width(a.K)) {
        case 1: launch_gradw_as<T, Q8, A, 1>(a, stream); break;
        case 2: launch_gradw_as<T, Q8, A, 2>(a, stream); break;
        default: launch_gradw_as<T, Q8, A, 4>(a, stream); break;
    }
}
template <class T, bool Q8>
static void launch_gradw(const LinearGradW& a, hipStream_t stream) {
    switch (gradw_width(a.N)) {
        case 1: launch_gradw_b<T, Q8, 1>(a, stream); break;
        case 2: launch_gradw_b<T, Q8, 2>(a, stream); break;
        default: launch_gradw_b<T, Q8, 4>(a, stream); break;
    }
}

static size_t aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }

// Scratch of the backward pass: dz, W^T, the splits' dW and db.
struct BwdScratch {
    size_t dz, wt, part_w, part_b, total;
};
static BwdScratch bwd_scratch(int64_t rows, int K, int N, int dtype) {
    const size_t size = dtype == GS3D_F32 ? 4 : 2;
    const GradWPlan p = gradw_plan(rows, K, N), bias_only = gradw_plan(rows, 1, N);
    BwdScratch s;
    s.dz = 0;
    s.wt = aligned((size_t)rows * N * size);
    s.part_w = s.wt + aligned((size_t)N * K * size);
    s.part_b = s.part_w + aligned((size_t)p.splits * N * K * 4);
    const int splits = p.splits > bias_only.splits ? p.splits : bias_only.splits;
    s.total = s.part_b + aligned((size_t)splits * N * 4);
    return s;
}

template <class T>
static int linear_fwd(const gs3d_linear_args& g, hipStream_t stream) {
    LinearRows a{};
    a.x = g.x, a.ldx = g.x_stride, a.w = g.weight, a.bias = g.bias, a.other = g.residual, a.ldo = g.residual_stride;
    a.y = g.y, a.ldy = g.outer, a.rows = g.rows, a.K = g.inner, a.N = g.outer, a.act = g.activation;
    launch_rows<T, false, 0>(a, stream);
    return launch_status("gs3d_linear_fwd");
}

template <class T, bool Q8>
static int linear_bwd(const gs3d_linear_bwd_args& g, char* scratch, hipStream_t stream) {
    const BwdScratch at = bwd_scratch(g.rows, g.inner, g.outer, g.dtype);
    const Q8Rows q8{g.codes, g.scales, g.inner};
    const void* dz = g.upstream;
    int64_t ldz = g.upstream_stride;
    if (g.activation != GS3D_ACT_NONE && g.rows > 0) {
        LinearRows a{};
        a.x = g.x, a.ldx = g.x_stride, a.q8 = q8, a.w = g.weight, a.bias = g.bias;
        a.other = g.upstream, a.ldo = g.upstream_stride, a.y = scratch + at.dz, a.ldy = g.outer;
        a.rows = g.rows, a.K = g.inner, a.N = g.outer, a.act = g.activation;
        launch_rows<T, Q8, 1>(a, stream);
        dz = scratch + at.dz;
        ldz = g.outer;
    }
    if (g.grad_x && g.rows > 0) {
        T* wt = reinterpret_cast<T*>(scratch + at.wt);
        hipLaunchKernelGGL(transpose_kernel<T>, dim3((g.inner + 31) / 32, (g.outer + 31) / 32), dim3(256), 0, stream,
                           static_cast<const T*>(g.weight), g.outer, g.inner, wt);
        LinearRows a{};
        a.x = dz, a.ldx = ldz, a.w = wt, a.y = g.grad_x, a.ldy = g.inner;
        a.rows = g.rows, a.K = g.outer, a.N = g.inner, a.act = GS3D_ACT_NONE;
        launch_rows<T, false, 0>(a, stream);
    }
    if (g.grad_weight || g.grad_bias) {
        // Without the weight's gradient the input has no columns to read.
        const int K = g.grad_weight ? g.inner : 0;
        const GradWPlan p = gradw_plan(g.rows, K ? K : 1, g.outer);
        LinearGradW a{};
        a.x = g.x, a.ldx = g.x_stride, a.q8 = Q8Rows{g.codes, g.scales, K}, a.dz = dz, a.ldz = ldz, a.rows = g.rows;
        a.rows_per_split = p.rows_per_split, a.K = K, a.N = g.outer;
        a.n_tiles = p.n_tiles, a.k_tiles = p.k_tiles, a.splits = p.splits;
        a.part_w = g.grad_weight ? reinterpret_cast<float*>(scratch + at.part_w) : nullptr;
        a.part_b = g.grad_bias ? reinterpret_cast<float*>(scratch + at.part_b) : nullptr;
        launch_gradw<T, Q8>(a, stream);
        if (g.grad_weight) {
            const int64_t count = (int64_t)g.outer * g.inner;
            hipLaunchKernelGGL(sum_splits_kernel<T>, dim3(blocks_for(count, 256)), dim3(256), 0, stream, a.part_w,
                               p.splits, count, static_cast<T*>(g.grad_weight));
        }
        if (g.grad_bias)
            hipLaunchKernelGGL(sum_splits_kernel<T>, dim3(blocks_for(g.outer, 256)), dim3(256), 0, stream, a.part_b,
                               p.splits, (int64_t)g.outer, static_cast<T*>(g.grad_bias));
    }
    return launch_status("gs3d_linear_bwd");
}

static bool linear_sizes_ok(int64_t rows, int K, int N, int dtype, int activation) {
    return rows >= 0 && rows <= GS3D_MAX_ROWS && K >= 1 && N >= 1 && K <= GS3D_MAX_CHANNELS &&
           N <= GS3D_MAX_CHANNELS && dtype >= 0 && dtype <= 2 && activation >= 0 && activation <= 3;
}

}  // namespace gs3d

extern "C" int gs3d_linear_fwd(const gs3d_linear_args* g, void* stream) {
    if (!g || !gs3d::linear_sizes_ok(g->rows, g->inner, g->outer, g->dtype, g->activation)) return GS3D_ERR_ARGUMENT;
    if (g->x_stride < g->inner || (g->residual && g->residual_stride < g->outer)) return GS3D_ERR_ARGUMENT;
    if (g->rows == 0) return GS3D_OK;
    if (!g->x || !g->weight || !g->y) return GS3D_ERR_ARGUMENT;
    const hipStream_t s = gs3d::as_stream(stream);
    if (g->dtype == GS3D_F32) return gs3d::linear_fwd<float>(*g, s);
    if (g->dtype == GS3D_BF16) return gs3d::linear_fwd<gs3d::bf16_t>(*g, s);
    return gs3d::linear_fwd<gs3d::f16_t>(*g, s);
}

extern "C" size_t gs3d_linear_bwd_scratch_bytes(int64_t rows, int32_t inner, int32_t outer, int32_t dtype) {
    if (!gs3d::linear_sizes_ok(rows, inner, outer, dtype, 0)) return 0;
    return gs3d::bwd_scratch(rows, inner, outer, dtype).total;
}

extern "C" int gs3d_linear_bwd(const gs3d_linear_bwd_args* g, void* scratch, size_t scratch_bytes, void* stream) {
    if (!g || !gs3d::linear_sizes_ok(g->rows, g->inner, g->outer, g->dtype, g->activation)) return GS3D_ERR_ARGUMENT;
    const bool q8 = g->codes != nullptr;
    if (q8 != (g->scales != nullptr) || (q8 && g->x)) return GS3D_ERR_ARGUMENT;
    const bool sees_input = g->grad_weight || g->activation != GS3D_ACT_NONE;
    if (g->rows > 0 && (!g->weight || !g->upstream || g->upstream_stride < g->outer ||
                        (sees_input && !q8 && (!g->x || g->x_stride < g->inner))))
        return GS3D_ERR_ARGUMENT;
    if (scratch_bytes < gs3d_linear_bwd_scratch_bytes(g->rows, g->inner, g->outer, g->dtype) || !scratch)
        return GS3D_ERR_SCRATCH;
    const hipStream_t s = gs3d::as_stream(stream);
    char* p = static_cast<char*>(scratch);
    if (g->dtype == GS3D_F32) return q8 ? gs3d::linear_bwd<float, true>(*g, p, s) : gs3d::linear_bwd<float, false>(*g, p, s);
    if (g->dtype == GS3D_BF16)
        return q8 ? gs3d::linear_bwd<gs3d::bf16_t, true>(*g, p, s) : gs3d::linear_bwd<gs3d::bf16_t, false>(*g, p, s);
    return q8 ? gs3d::linear_bwd<gs3d::f16_t, true>(*g, p, s) : gs3d::linear_bwd<gs3d::f16_t, false>(*g, p, s);
}
