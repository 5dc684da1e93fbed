// Group normalisation of channel-last images, then an activation:
//   u = (x - mean) rstd gamma + beta,  y = act(u)
// with one mean and variance per image and group of neighbouring channels,
// over all the image's pixels, and its gradients.
//
// Both directions read their images twice: once for the sums, once for the
// result.  A thread keeps one 16-byte vector of channels and walks down the
// pixels, so everything that belongs to a channel stays in its registers.
//
//   norm_statistics_kernel  per strip of pixels and channel: mean and summed
//                           squared deviation (Welford's update)
//   norm_merge_kernel       per image and group: mean and 1/sqrt(var + eps)
//   norm_apply_kernel       y from x
//   norm_sums_kernel        per strip and channel: sum dz, sum dz (x - mean)
//   norm_totals_kernel      per image and group: the strips' sums in order
//   norm_params_kernel      dgamma, dbeta: the images' sums in order
//   norm_grad_kernel        dx from dy and x
//
// Moments are merged as (count, mean, M2) throughout: an image whose mean is
// far from zero loses no digits to a difference of squares.
//
// HBM bounds all of it: 4 x 1920 x 1080 x 64 floats, statistics 384 us (5.5
// TB/s), apply 827 and sums 736 (5.1, 5.8), gradient 1232 (5.2).  The second
// passes walk backwards over each strip, whose end the first one left in the
// cache (1 to 2%).  One pass would need an image to stay on the chip: a launch
// per image, so that the last-level cache held it, cost more than it saved.
#include "decode.hpp"

namespace gs3d {

struct NormShape {
    int64_t pixels;      // of an image
    int64_t strip_rows;  // pixels of a strip
    int images, channels, groups, strips, act;
    float eps;
};

struct NormParams {
    const void* gamma;  // channels, or NULL: 1
    const void* beta;   // channels, or NULL: 0
    const float2* stats;  // images x groups: mean, rstd
};

// A block covers up to 256 vectors of channels (blockIdx.z the further ones)
// and 256 / width pixels at a time.
struct NormThread {
    int width, slots, slot, at;  // at: first channel
    bool live;
};
template <int E>
GS3D_DEV NormThread norm_thread(int channels) {
    const int vectors = (channels + E - 1) / E, first = blockIdx.z * 256;
    NormThread t;
    t.width = vectors - first < 256 ? vectors - first : 256;
    t.slots = 256 / t.width;
    t.slot = threadIdx.x / t.width;
    t.at = (first + threadIdx.x % t.width) * E;
    t.live = t.slot < t.slots;
    return t;
}

// Per-channel constants of a thread: u = (x - mean) scale + beta.
template <class T, int E>
GS3D_DEV void norm_constants(const NormShape& s, const NormParams& p, int image, int at, float (&mean)[E],
                             float (&rstd)[E], float (&scale)[E], float (&beta)[E]) {
    const int per_group = s.channels / s.groups;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int c = at + i < s.channels ? at + i : s.channels - 1;
        const float2 m = p.stats[(int64_t)image * s.groups + c / per_group];
        mean[i] = m.x;
        rstd[i] = m.y;
        scale[i] = p.gamma ? m.y * to_f32(static_cast<const T*>(p.gamma)[c]) : m.y;
        beta[i] = p.beta ? to_f32(static_cast<const T*>(p.beta)[c]) : 0.0f;
    }
}

// (n, mean, M2) of two sets together (Chan, Golub and LeVeque's update).
GS3D_DEV void merge_moments(float& n, float& mean, float& m2, float nb, float mb, float m2b) {
    if (nb == 0.0f) return;
    const float total = n + nb, d = mb - mean, share = nb / total;
    mean = __builtin_fmaf(d, share, mean);
    m2 += __builtin_fmaf(d * d, n * share, m2b);
    n = total;
}

template <class T, bool WIDE>
__global__ __launch_bounds__(256) void norm_statistics_kernel(NormShape s, Rows a, float2* __restrict__ part) {
    constexpr int E = VEC<T>;
    constexpr int U = 4;  // pixels whose loads are in flight together
    const NormThread t = norm_thread<E>(s.channels);
    const bool inside = s.channels % E == 0;  // every vector is whole
    const int64_t begin = blockIdx.x * s.strip_rows, base = blockIdx.y * s.pixels;
    const int64_t end = begin + s.strip_rows < s.pixels ? begin + s.strip_rows : s.pixels;
    float mean[E], m2[E], n = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) mean[i] = m2[i] = 0.0f;
    if (t.live) {
        for (int64_t p = begin + t.slot; p < end; p += U * t.slots) {
            RowRaw<T, false, WIDE> raw[U];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int64_t row = p + k * t.slots;
                raw[k].issue(a, base + (row < end ? row : p), t.at);
            }
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (p + k * t.slots >= end) break;
                float v[E];
                unpack<T>(raw[k].finish_in(a, inside, t.at), v);
                n += 1.0f;
                const float share = __builtin_amdgcn_rcpf(n);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const float d = v[i] - mean[i];
                    mean[i] = __builtin_fmaf(d, share, mean[i]);
                    m2[i] = __builtin_fmaf(d, v[i] - mean[i], m2[i]);
                }
            }
        }
    }
    // The block's pixels of a channel together, halving the slots.
    __shared__ float lds[2 * E + 1][256];
    for (int live = t.slots; live > 1; live = (live + 1) / 2) {
        const int half = (live + 1) / 2;
        __syncthreads();
        if (t.slot >= half && t.slot < live) {
            lds[2 * E][threadIdx.x] = n;
#pragma unroll
            for (int i = 0; i < E; ++i) lds[i][threadIdx.x] = mean[i], lds[E + i][threadIdx.x] = m2[i];
        }
        __syncthreads();
        if (t.slot + half < live) {
            const int j = threadIdx.x + half * t.width;
            const float nb = lds[2 * E][j], total = n + nb;
            if (nb > 0.0f) {
                const float share = nb / total, weight = n * share;
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const float d = lds[i][j] - mean[i];
                    mean[i] = __builtin_fmaf(d, share, mean[i]);
                    m2[i] += __builtin_fmaf(d * d, weight, lds[E + i][j]);
                }
                n = total;
            }
        }
    }
    if (t.slot == 0) {
        float2* out = part + ((int64_t)blockIdx.y * s.strips + blockIdx.x) * s.channels + t.at;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (t.at + i < s.channels) out[i] = float2{mean[i], m2[i]};
    }
}

// One block per (group, image): every thread merges its share of the strips'
// moments in order, then a tree over the threads.
__global__ __launch_bounds__(1024) void norm_merge_kernel(NormShape s, const float2* __restrict__ part,
                                                          float2* __restrict__ stats) {
    const int per_group = s.channels / s.groups, group = blockIdx.x, image = blockIdx.y;
    const int items = s.strips * per_group;
    float n = 0.0f, mean = 0.0f, m2 = 0.0f;
    for (int i = threadIdx.x; i < items; i += 1024) {
        const int strip = i / per_group, c = i - strip * per_group;
        const int64_t begin = strip * s.strip_rows;
        const int64_t rows = s.pixels - begin < s.strip_rows ? s.pixels - begin : s.strip_rows;
        const float2 m = part[((int64_t)image * s.strips + strip) * s.channels + group * per_group + c];
        merge_moments(n, mean, m2, (float)rows, m.x, m.y);
    }
    __shared__ float lds[3][1024];
    for (int half = 512; half > 0; half >>= 1) {
        if ((int)threadIdx.x < 2 * half) {
            lds[0][threadIdx.x] = n;
            lds[1][threadIdx.x] = mean;
            lds[2][threadIdx.x] = m2;
        }
        __syncthreads();
        if ((int)threadIdx.x < half) {
            const int j = threadIdx.x + half;
            merge_moments(n, mean, m2, lds[0][j], lds[1][j], lds[2][j]);
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const float count = (float)((double)s.pixels * per_group);
        stats[(int64_t)image * s.groups + group] = float2{mean, 1.0f / __builtin_sqrtf(m2 / count + s.eps)};
    }
}

// KEEP: x is also written in 8 bits as it is read; whole blocks of 32 channels
// then, so that a block lies in neighbouring lanes.
template <class T, bool KEEP, bool WIDE>
__global__ __launch_bounds__(256) void norm_apply_kernel(NormShape s, Rows a, NormParams p, T* __restrict__ y,
                                                         int8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    constexpr int E = VEC<T>;
    constexpr int U = 4;
    const NormThread t = norm_thread<E>(s.channels);
    const bool inside = s.channels % E == 0;  // every vector is whole
    if (!t.live) return;
    const int64_t begin = blockIdx.x * s.strip_rows, base = blockIdx.y * s.pixels;
    const int64_t end = begin + s.strip_rows < s.pixels ? begin + s.strip_rows : s.pixels;
    float mean[E], rstd[E], scale[E], beta[E];
    norm_constants<T, E>(s, p, blockIdx.y, t.at, mean, rstd, scale, beta);
    // Backwards: what the first pass read last is still in the cache.
    for (int64_t row = end - 1 - t.slot; row >= begin; row -= U * t.slots) {
        RowRaw<T, false, WIDE> raw[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int64_t at = row - k * t.slots;
            raw[k].issue(a, base + (at >= begin ? at : row), t.at);
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int64_t at = row - k * t.slots;
            if (at < begin) break;
            float v[E];
            unpack<T>(raw[k].finish_in(a, inside, t.at), v);
            if constexpr (KEEP) q8_keep<T>(v, codes, scales, base + at, t.at, s.channels, true);
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = __builtin_fmaf(v[i] - mean[i], scale[i], beta[i]);
            activate<T>(v, s.act);
            store_row(y + (base + at) * s.channels, t.at, s.channels, pack<T>(v));
        }
    }
}

template <class T, bool Q8, bool WIDE>
__global__ __launch_bounds__(256, 4) void norm_sums_kernel(NormShape s, Rows a, NormParams p, const T* __restrict__ dy,
                                                        int64_t ldy, float2* __restrict__ part) {
    constexpr int E = VEC<T>;
    constexpr int U = 2;
    const NormThread t = norm_thread<E>(s.channels);
    const bool inside = s.channels % E == 0;  // every vector is whole
    const int64_t begin = blockIdx.x * s.strip_rows, base = blockIdx.y * s.pixels;
    const int64_t end = begin + s.strip_rows < s.pixels ? begin + s.strip_rows : s.pixels;
    float s1[E], s2[E];
#pragma unroll
    for (int i = 0; i < E; ++i) s1[i] = s2[i] = 0.0f;
    if (t.live) {
        float mean[E], rstd[E], scale[E], beta[E];
        norm_constants<T, E>(s, p, blockIdx.y, t.at, mean, rstd, scale, beta);
        for (int64_t row = begin + t.slot; row < end; row += U * t.slots) {
            RowRaw<T, Q8, WIDE> raw[U];
            u32x4 up[U];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int64_t r = row + k * t.slots, at = base + (r < end ? r : row);
                raw[k].issue(a, at, t.at);
                up[k] = issue_row<T, WIDE>(dy + at * ldy, t.at, s.channels);
            }
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (row + k * t.slots >= end) break;
                float v[E], u[E], g[E];
                unpack<T>(raw[k].finish_in(a, inside, t.at), v);
                unpack<T>(inside ? up[k] : finish_row<T, WIDE>(up[k], t.at, s.channels), g);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    v[i] -= mean[i];
                    u[i] = __builtin_fmaf(v[i], scale[i], beta[i]);
                }
                pull_back<T>(g, u, s.act);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    s1[i] += g[i];
                    s2[i] = __builtin_fmaf(g[i], v[i], s2[i]);
                }
            }
        }
    }
    __shared__ float lds[2 * E][256];
    for (int live = t.slots; live > 1; live = (live + 1) / 2) {
        const int half = (live + 1) / 2;
        __syncthreads();
        if (t.slot >= half && t.slot < live) {
#pragma unroll
            for (int i = 0; i < E; ++i) lds[i][threadIdx.x] = s1[i], lds[E + i][threadIdx.x] = s2[i];
        }
        __syncthreads();
        if (t.slot + half < live) {
            const int j = threadIdx.x + half * t.width;
#pragma unroll
            for (int i = 0; i < E; ++i) s1[i] += lds[i][j], s2[i] += lds[E + i][j];
        }
    }
    if (t.slot == 0) {
        float2* out = part + ((int64_t)blockIdx.y * s.strips + blockIdx.x) * s.channels + t.at;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (t.at + i < s.channels) {
                const int group = (t.at + i) / (s.channels / s.groups);
                out[i] = float2{s1[i], s2[i] * p.stats[(int64_t)blockIdx.y * s.groups + group].y};
            }
    }
}

// One block per (group, image).  sums[image][channel] = (sum dz, sum dz xhat);
// pulls[image][group] = the means of gamma dz and of gamma dz xhat.
template <class T>
__global__ __launch_bounds__(1024) void norm_totals_kernel(NormShape s, const T* __restrict__ gamma,
                                                           const float2* __restrict__ part, float2* __restrict__ sums,
                                                           float2* __restrict__ pulls) {
    const int per_group = s.channels / s.groups, group = blockIdx.x, image = blockIdx.y;
    __shared__ float lds[2][1024];
    float p1 = 0.0f, p2 = 0.0f;  // thread 0..width-1: its channels' share of the pulls
    for (int first = 0; first < per_group; first += 1024) {
        const int width = per_group - first < 1024 ? per_group - first : 1024;
        const int lanes = 1024 / width, lane = threadIdx.x / width;
        const int c = group * per_group + first + threadIdx.x % width;
        float a1 = 0.0f, a2 = 0.0f;
        if (lane < lanes) {
            for (int strip = lane; strip < s.strips; strip += lanes) {
                const float2 v = part[((int64_t)image * s.strips + strip) * s.channels + c];
                a1 += v.x;
                a2 += v.y;
            }
        }
        __syncthreads();
        lds[0][threadIdx.x] = a1;
        lds[1][threadIdx.x] = a2;
        __syncthreads();
        if (lane == 0) {
            for (int k = 1; k < lanes; ++k) {
                a1 += lds[0][threadIdx.x + k * width];
                a2 += lds[1][threadIdx.x + k * width];
            }
            sums[(int64_t)image * s.channels + c] = float2{a1, a2};
            const float w = gamma ? to_f32(gamma[c]) : 1.0f;
            p1 = __builtin_fmaf(w, a1, p1);
            p2 = __builtin_fmaf(w, a2, p2);
        }
    }
    for (int half = 512; half > 0; half >>= 1) {
        __syncthreads();
        lds[0][threadIdx.x] = p1;
        lds[1][threadIdx.x] = p2;
        __syncthreads();
        if ((int)threadIdx.x < half) {
            p1 += lds[0][threadIdx.x + half];
            p2 += lds[1][threadIdx.x + half];
        }
    }
    if (threadIdx.x == 0) {
        const float count = (float)((double)s.pixels * per_group);
        pulls[(int64_t)image * s.groups + group] = float2{p1 / count, p2 / count};
    }
}

template <class T>
__global__ __launch_bounds__(256) void norm_params_kernel(int images, int channels, const float2* __restrict__ sums,
                                                          T* __restrict__ dgamma, T* __restrict__ dbeta) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= channels) return;
    float a1 = 0.0f, a2 = 0.0f;
    for (int b = 0; b < images; ++b) {
        const float2 v = sums[(int64_t)b * channels + c];
        a1 += v.x;
        a2 += v.y;
    }
    if (dbeta) dbeta[c] = (T)a1;
    if (dgamma) dgamma[c] = (T)a2;
}

template <class T, bool Q8, bool WIDE>
__global__ __launch_bounds__(256, 4) void norm_grad_kernel(NormShape s, Rows a, NormParams p, const T* __restrict__ dy,
                                                        int64_t ldy, const float2* __restrict__ pulls,
                                                        T* __restrict__ dx) {
    constexpr int E = VEC<T>;
    constexpr int U = 2;
    const NormThread t = norm_thread<E>(s.channels);
    const bool inside = s.channels % E == 0;  // every vector is whole
    if (!t.live) return;
    const int64_t begin = blockIdx.x * s.strip_rows, base = blockIdx.y * s.pixels;
    const int64_t end = begin + s.strip_rows < s.pixels ? begin + s.strip_rows : s.pixels;
    const int per_group = s.channels / s.groups;
    // dx = scale dz - level - (x - mean) along
    float mean[E], level[E], along[E], scale[E], beta[E];
    norm_constants<T, E>(s, p, blockIdx.y, t.at, mean, level, scale, beta);
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int c = t.at + i < s.channels ? t.at + i : s.channels - 1;
        const float2 pull = pulls[(int64_t)blockIdx.y * s.groups + c / per_group];
        const float rstd = level[i];
        level[i] = rstd * pull.x;
        along[i] = rstd * rstd * pull.y;
    }
    for (int64_t row = end - 1 - t.slot; row >= begin; row -= U * t.slots) {  // backwards, as in norm_apply_kernel
        RowRaw<T, Q8, WIDE> raw[U];
        u32x4 up[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int64_t r = row - k * t.slots, at = base + (r >= begin ? r : row);
            raw[k].issue(a, at, t.at);
            up[k] = issue_row<T, WIDE>(dy + at * ldy, t.at, s.channels);
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int64_t at = row - k * t.slots;
            if (at < begin) break;
            float v[E], u[E], g[E];
            unpack<T>(raw[k].finish_in(a, inside, t.at), v);
            unpack<T>(inside ? up[k] : finish_row<T, WIDE>(up[k], t.at, s.channels), g);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                v[i] -= mean[i];
                u[i] = __builtin_fmaf(v[i], scale[i], beta[i]);
            }
            pull_back<T>(g, u, s.act);
#pragma unroll
            for (int i = 0; i < E; ++i)
                v[i] = __builtin_fmaf(-v[i], along[i], __builtin_fmaf(scale[i], g[i], -level[i]));
            store_row(dx + (base + at) * s.channels, t.at, s.channels, pack<T>(v));
        }
    }
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
// Strips: about 1024 blocks in all (four a compute unit), and no strip
// shorter than eight steps of a block.
static NormShape norm_shape(int images, int64_t pixels, int channels, int groups, int dtype) {
    NormShape s{};
    s.images = images, s.pixels = pixels, s.channels = channels, s.groups = groups;
    const int E = dtype == GS3D_F32 ? 4 : 8;
    const int vectors = (channels + E - 1) / E;
    const int width = vectors < 256 ? vectors : 256;
    const int64_t shortest = 8 * (256 / width);
    int64_t strips = 1024 / ((int64_t)images * ((vectors + 255) / 256));
    const int64_t most = (pixels + shortest - 1) / shortest;
    if (strips > most) strips = most;
    if (strips < 1) strips = 1;
    s.strip_rows = (pixels + strips - 1) / strips;
    s.strips = (int)((pixels + s.strip_rows - 1) / s.strip_rows);
    return s;
}

static dim3 norm_grid(const NormShape& s, int dtype) {
    const int E = dtype == GS3D_F32 ? 4 : 8;
    return dim3((unsigned)s.strips, (unsigned)s.images, (unsigned)(((s.channels + E - 1) / E + 255) / 256));
}

static size_t norm_aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }

static size_t norm_part_bytes(const NormShape& s) {
    return norm_aligned((size_t)s.images * s.strips * s.channels * sizeof(float2));
}

template <class T>
static int norm_fwd(const gs3d_group_norm_args& g, void* scratch, hipStream_t stream) {
    NormShape s = norm_shape(g.images, g.pixels, g.channels, g.groups, g.dtype);
    s.act = g.activation, s.eps = g.eps;
    const Rows a{g.x, g.x_stride, {}, g.channels};
    float2* part = static_cast<float2*>(scratch);
    float2* stats = reinterpret_cast<float2*>(g.statistics);
    const dim3 grid = norm_grid(s, g.dtype);
    const bool wide = g.channels >= VEC<T>;
    if (wide) hipLaunchKernelGGL((norm_statistics_kernel<T, true>), grid, dim3(256), 0, stream, s, a, part);
    else hipLaunchKernelGGL((norm_statistics_kernel<T, false>), grid, dim3(256), 0, stream, s, a, part);
    hipLaunchKernelGGL(norm_merge_kernel, dim3(s.groups, s.images), dim3(1024), 0, stream, s, part, stats);
    const NormParams p{g.weight, g.bias, stats};
    T* y = static_cast<T*>(g.y);
    if (g.codes && g.channels % Q8_BLOCK == 0) {
        hipLaunchKernelGGL((norm_apply_kernel<T, true, true>), grid, dim3(256), 0, stream, s, a, p, y, g.codes,
                           g.scales);
    } else {
        if (g.codes)
            quantize_rows(g.x, g.x_stride, g.images * g.pixels, g.channels, g.dtype, g.codes, g.scales, stream);
        if (wide)
            hipLaunchKernelGGL((norm_apply_kernel<T, false, true>), grid, dim3(256), 0, stream, s, a, p, y, nullptr,
                               nullptr);
        else
            hipLaunchKernelGGL((norm_apply_kernel<T, false, false>), grid, dim3(256), 0, stream, s, a, p, y, nullptr,
                               nullptr);
    }
    return launch_status("gs3d_group_norm_fwd");
}

// The images' sums to dgamma and dbeta (zero without images).
template <class T>
static void launch_params(const gs3d_group_norm_bwd_args& g, int images, const float2* sums, hipStream_t stream) {
    if (g.grad_weight || g.grad_bias)
        hipLaunchKernelGGL(norm_params_kernel<T>, dim3(blocks_for(g.channels, 256)), dim3(256), 0, stream, images,
                           g.channels, sums, static_cast<T*>(g.grad_weight), static_cast<T*>(g.grad_bias));
}

template <class T, bool Q8, bool WIDE>
static int norm_bwd_as(const gs3d_group_norm_bwd_args& g, char* scratch, hipStream_t stream) {
    NormShape s = norm_shape(g.images, g.pixels, g.channels, g.groups, g.dtype);
    s.act = g.activation;
    const Rows a{g.x, g.x_stride, {g.codes, g.scales, g.channels}, g.channels};
    const NormParams p{g.weight, g.bias, reinterpret_cast<const float2*>(g.statistics)};
    float2* part = reinterpret_cast<float2*>(scratch);
    float2* sums = reinterpret_cast<float2*>(scratch + norm_part_bytes(s));
    float2* pulls = sums + norm_aligned((size_t)s.images * s.channels * sizeof(float2)) / sizeof(float2);
    const T* dy = static_cast<const T*>(g.upstream);
    const T* gamma = static_cast<const T*>(g.weight);
    const dim3 grid = norm_grid(s, g.dtype);
    hipLaunchKernelGGL((norm_sums_kernel<T, Q8, WIDE>), grid, dim3(256), 0, stream, s, a, p, dy, g.upstream_stride,
                       part);
    hipLaunchKernelGGL(norm_totals_kernel<T>, dim3(s.groups, s.images), dim3(1024), 0, stream, s, gamma, part, sums,
                       pulls);
    if (g.grad_x)
        hipLaunchKernelGGL((norm_grad_kernel<T, Q8, WIDE>), grid, dim3(256), 0, stream, s, a, p, dy, g.upstream_stride,
                           pulls, static_cast<T*>(g.grad_x));
    launch_params<T>(g, g.images, sums, stream);
    return launch_status("gs3d_group_norm_bwd");
}
template <class T, bool Q8>
static int norm_bwd(const gs3d_group_norm_bwd_args& g, char* scratch, hipStream_t stream) {
    if (g.images == 0 || g.pixels == 0) {  // the parameters' gradients are sums of nothing
        launch_params<T>(g, 0, nullptr, stream);
        return launch_status("gs3d_group_norm_bwd");
    }
    return g.channels >= VEC<T> ? norm_bwd_as<T, Q8, true>(g, scratch, stream)
                                : norm_bwd_as<T, Q8, false>(g, scratch, stream);
}

static bool norm_sizes_ok(int32_t images, int64_t pixels, int32_t channels, int32_t groups, int dtype, int activation) {
    return images >= 0 && images <= GS3D_MAX_IMAGES && pixels >= 0 && pixels <= GS3D_MAX_ROWS && channels >= 1 &&
           channels <= GS3D_MAX_CHANNELS && groups >= 1 && channels % groups == 0 && dtype >= 0 && dtype <= 2 &&
           activation >= 0 && activation <= 3;
}

}  // namespace gs3d

extern "C" size_t gs3d_group_norm_scratch_bytes(int32_t images, int64_t pixels, int32_t channels, int32_t groups,
                                                int32_t dtype) {
    if (!gs3d::norm_sizes_ok(images, pixels, channels, groups, dtype, 0) || images == 0 || pixels == 0) return 0;
    const gs3d::NormShape s = gs3d::norm_shape(images, pixels, channels, groups, dtype);
    return gs3d::norm_part_bytes(s) + gs3d::norm_aligned((size_t)images * channels * sizeof(float2)) +
           gs3d::norm_aligned((size_t)images * groups * sizeof(float2));
}

extern "C" int gs3d_group_norm_fwd(const gs3d_group_norm_args* g, void* scratch, size_t scratch_bytes, void* stream) {
    if (!g || !gs3d::norm_sizes_ok(g->images, g->pixels, g->channels, g->groups, g->dtype, g->activation) ||
        !(g->eps > 0.0f) || g->x_stride < g->channels)
        return GS3D_ERR_ARGUMENT;
    if (g->images == 0 || g->pixels == 0) return GS3D_OK;
    if (!g->x || !g->y || !g->statistics || !g->codes != !g->scales) return GS3D_ERR_ARGUMENT;
    if (!scratch ||
        scratch_bytes < gs3d_group_norm_scratch_bytes(g->images, g->pixels, g->channels, g->groups, g->dtype))
        return GS3D_ERR_SCRATCH;
    const hipStream_t s = gs3d::as_stream(stream);
    if (g->dtype == GS3D_F32) return gs3d::norm_fwd<float>(*g, scratch, s);
    if (g->dtype == GS3D_BF16) return gs3d::norm_fwd<gs3d::bf16_t>(*g, scratch, s);
    return gs3d::norm_fwd<gs3d::f16_t>(*g, scratch, s);
}

extern "C" int gs3d_group_norm_bwd(const gs3d_group_norm_bwd_args* g, void* scratch, size_t scratch_bytes,
                                   void* stream) {
    if (!g || !gs3d::norm_sizes_ok(g->images, g->pixels, g->channels, g->groups, g->dtype, g->activation))
        return GS3D_ERR_ARGUMENT;
    const bool q8 = g->codes != nullptr;
    if (q8 != (g->scales != nullptr) || (q8 && g->x)) return GS3D_ERR_ARGUMENT;
    const size_t needed = gs3d_group_norm_scratch_bytes(g->images, g->pixels, g->channels, g->groups, g->dtype);
    if (needed > 0) {  // there are pixels
        if (!g->statistics || !g->upstream || g->upstream_stride < g->channels ||
            (!q8 && (!g->x || g->x_stride < g->channels)))
            return GS3D_ERR_ARGUMENT;
        if (!scratch || scratch_bytes < needed) return GS3D_ERR_SCRATCH;
    }
    const hipStream_t s = gs3d::as_stream(stream);
    char* p = static_cast<char*>(scratch);
    if (g->dtype == GS3D_F32) return q8 ? gs3d::norm_bwd<float, true>(*g, p, s) : gs3d::norm_bwd<float, false>(*g, p, s);
    if (g->dtype == GS3D_BF16)
        return q8 ? gs3d::norm_bwd<gs3d::bf16_t, true>(*g, p, s) : gs3d::norm_bwd<gs3d::bf16_t, false>(*g, p, s);
    return q8 ? gs3d::norm_bwd<gs3d::f16_t, true>(*g, p, s) : gs3d::norm_bwd<gs3d::f16_t, false>(*g, p, s);
}
