// groupnorm.hpp — group norm with an activation and optional dropout over channels-last feature maps, forward and backward.
//
//   xhat = (x - mean) / sqrt(var + eps)   mean, var (biased) over the pixels of one image and the channels of one group
//   z = xhat * weight + bias,  y = activation(z),  then dropout (elements.hpp)
//   backward: dz = dy * activation'(z);  dbias = sum dz, dweight = sum dz * xhat over images and pixels;
//   dx = (weight * dz - A - xhat * B) / sqrt(var + eps), A and B the group's means of weight * dz and weight * dz * xhat
//
// A block takes a run of pixels (a slab) of one image and a tile of channels: a thread keeps one vector of channels (16 bytes
// where the channel count, the strides and the pointers allow) and steps over the slab's pixels, so that a block reads whole
// runs of memory. Statistics are held per channel until a slab is done, so any number of channels per group works. Sums are
// in fp32 in an order that depends on the sizes alone.
#pragma once

#include <algorithm>

#include "elements.hpp"

namespace inpc {
namespace norm {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;            // pixels a thread has in flight
constexpr uint32_t kFillBlocks = 2048;   // blocks that fill the chip: eight per compute unit

struct Shape {
    uint64_t x_image, x_pixel;   // strides of x in elements (channels are adjacent); y and dx are dense
    uint64_t g_image, g_pixel;   // of the gradient of y
    uint32_t n, pixels, channels, groups, per_group;
    uint32_t columns, tiles;     // vectors of a channel tile; channel tiles
    uint32_t rows;               // pixels a block covers at once
    uint32_t slabs, slab_pixels; // per image
    int32_t activation, param_dtype;
    float eps;
};

// The part of the feature maps that a block works on, and the part of that which is the calling thread's.
struct Place {
    uint32_t image, slab, channel, row, begin, end;
    bool active;
};

template <int V>
__device__ __forceinline__ Place place_of(const Shape& s) {
    Place p;
    p.slab = blockIdx.x % s.slabs;
    const uint32_t rest = blockIdx.x / s.slabs;
    const uint32_t tile = rest % s.tiles;
    p.image = rest / s.tiles;
    p.row = threadIdx.x / s.columns;
    p.channel = (tile * s.columns + threadIdx.x % s.columns) * V;
    p.active = p.row < s.rows && p.channel < s.channels;
    p.begin = p.slab * s.slab_pixels;
    p.end = min(p.begin + s.slab_pixels, s.pixels);
    return p;
}

// Two sets of values merged: counts na and nb, means, sums of squared deviations (Chan, Golub, LeVeque 1979). Nothing
// cancels, however far the mean is from zero.
__device__ __forceinline__ void merge_moments(float& na, float& mean, float& m2, float nb, float mean_b, float m2_b) {
    if (nb == 0.0f) return;
    const float n = na + nb, d = mean_b - mean, share = nb / n;
    mean = fmaf(d, share, mean);
    m2 += fmaf(d * d, na * share, m2_b);
    na = n;
}

// ---- forward: moments of every (image, slab, channel) -------------------------------------------------------------
template <int D, int V>
__global__ void __launch_bounds__(kThreads) k_moments(const void* __restrict__ x, float2* __restrict__ partial, Shape s) {
    __shared__ float2 merged[kThreads * V];
    __shared__ float counts[kThreads];
    const Place p = place_of<V>(s);
    float mean[V], m2[V], count = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) mean[j] = m2[j] = 0.0f;
    if (p.active) {
        const size_t base = (size_t)p.image * s.x_image + p.channel;
        uint32_t r = p.begin + p.row;
        for (; r + (kUnroll - 1) * s.rows < p.end; r += kUnroll * s.rows) {
            PackedVector<D, V> packed[kUnroll];
            float v[kUnroll][V];
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) packed[k] = load_packed<D, V>(x, base + (size_t)(r + k * s.rows) * s.x_pixel);
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) unpack<D, V>(packed[k], v[k]);
            // the moments of these few pixels first, then merged: two passes over registers
            const float n = count + kUnroll, share = kUnroll / n, weight = count * share;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float sum = v[0][j], squares = 0.0f;
#pragma unroll
                for (int k = 1; k < kUnroll; ++k) sum += v[k][j];
                const float m = sum * (1.0f / kUnroll), d = m - mean[j];
#pragma unroll
                for (int k = 0; k < kUnroll; ++k) squares = fmaf(v[k][j] - m, v[k][j] - m, squares);
                mean[j] = fmaf(d, share, mean[j]);
                m2[j] += fmaf(d * d, weight, squares);
            }
            count = n;
        }
        for (; r < p.end; r += s.rows) {
            float v[V];
            load_vector<D, V>(x, base + (size_t)r * s.x_pixel, v);
            const float n = count + 1.0f, share = 1.0f / n, weight = count * share;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = v[j] - mean[j];
                mean[j] = fmaf(d, share, mean[j]);
                m2[j] = fmaf(d * d, weight, m2[j]);
            }
            count = n;
        }
    }
    // merge the block's rows, halving
#pragma unroll
    for (int j = 0; j < V; ++j) merged[threadIdx.x * V + j] = make_float2(mean[j], m2[j]);
    counts[threadIdx.x] = count;
    uint32_t half = 1;
    while (half < s.rows) half <<= 1;
    for (half >>= 1; half > 0; half >>= 1) {
        __syncthreads();
        const uint32_t other = threadIdx.x + half * s.columns;
        const bool mine = p.row < half && p.row + half < s.rows;
        float n = 0.0f;
        if (mine) {
            for (int j = 0; j < V; ++j) {
                n = counts[threadIdx.x];
                float2 a = merged[threadIdx.x * V + j];
                const float2 b = merged[other * V + j];
                merge_moments(n, a.x, a.y, counts[other], b.x, b.y);
                merged[threadIdx.x * V + j] = a;
            }
            counts[threadIdx.x] = n;
        }
    }
    if (p.active && p.row == 0) {
        const size_t at = ((size_t)p.image * s.slabs + p.slab) * s.channels + p.channel;
        for (int j = 0; j < V; ++j) partial[at + j] = merged[threadIdx.x * V + j];
    }
}

// ... and of every (image, group): {mean, 1 / sqrt(var + eps)}, a block each
__global__ void __launch_bounds__(kThreads) k_group_moments(const float2* __restrict__ partial, float2* __restrict__ moments, Shape s) {
    __shared__ float4 merged[kThreads];
    const uint32_t image = blockIdx.x / s.groups, group = blockIdx.x % s.groups;
    float n = 0.0f, mean = 0.0f, m2 = 0.0f;
    const uint64_t items = (uint64_t)s.slabs * s.per_group;
    for (uint64_t i = threadIdx.x; i < items; i += kThreads) {
        const uint32_t slab = (uint32_t)(i / s.per_group), channel = group * s.per_group + (uint32_t)(i % s.per_group);
        const uint32_t begin = slab * s.slab_pixels;
        const float2 b = partial[((size_t)image * s.slabs + slab) * s.channels + channel];
        merge_moments(n, mean, m2, (float)(min(begin + s.slab_pixels, s.pixels) - begin), b.x, b.y);
    }
    merged[threadIdx.x] = make_float4(n, mean, m2, 0.0f);
    for (uint32_t half = kThreads / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (threadIdx.x < half) {
            float4 a = merged[threadIdx.x];
            const float4 b = merged[threadIdx.x + half];
            merge_moments(a.x, a.y, a.z, b.x, b.y, b.z);
            merged[threadIdx.x] = a;
        }
    }
    if (threadIdx.x == 0) moments[blockIdx.x] = make_float2(merged[0].y, 1.0f / sqrtf(merged[0].z / merged[0].x + s.eps));
}

// ---- the activations -----------------------------------------------------------------------------------------------
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

template <int V>
__device__ __forceinline__ void activate(int32_t activation, float (&z)[V]) {
    if (activation == INPC_ACTIVATION_RELU) {
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] = z[j] < 0.0f ? 0.0f : z[j];
    } else if (activation == INPC_ACTIVATION_SILU) {
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] *= sigmoid(z[j]);
    } else if (activation == INPC_ACTIVATION_GELU) {
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] = 0.5f * z[j] * (1.0f + erff(z[j] * 0.70710678f));
    }
}

// g *= activation'(z)
template <int V>
__device__ __forceinline__ void activate_backward(int32_t activation, const float (&z)[V], float (&g)[V]) {
    if (activation == INPC_ACTIVATION_RELU) {
#pragma unroll
        for (int j = 0; j < V; ++j) g[j] = z[j] > 0.0f ? g[j] : 0.0f;
    } else if (activation == INPC_ACTIVATION_SILU) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float p = sigmoid(z[j]);
            g[j] *= fmaf(z[j] * p, 1.0f - p, p);
        }
    } else if (activation == INPC_ACTIVATION_GELU) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            g[j] *= fmaf(z[j] * 0.39894228f, __expf(-0.5f * z[j] * z[j]), 0.5f * (1.0f + erff(z[j] * 0.70710678f)));
    }
}

// What a thread's channels are normalised with.
template <int V>
struct Channels {
    float mean[V], rstd[V], weight[V], bias[V];
};

template <int V>
__device__ __forceinline__ Channels<V> load_channels(const Shape& s, const Place& p, const float2* moments, const void* weight,
                                                     const void* bias) {
    Channels<V> c;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float2 m = moments[(size_t)p.image * s.groups + (p.channel + j) / s.per_group];
        c.mean[j] = m.x;
        c.rstd[j] = m.y;
        c.weight[j] = weight ? load_element(weight, s.param_dtype, p.channel + j) : 1.0f;
        c.bias[j] = bias ? load_element(bias, s.param_dtype, p.channel + j) : 0.0f;
    }
    return c;
}

template <int D, int V>
__global__ void __launch_bounds__(kThreads) k_apply(const void* __restrict__ x, const float2* __restrict__ moments,
                                                    const void* __restrict__ weight, const void* __restrict__ bias,
                                                    void* __restrict__ y, Shape s, Dropout d) {
    const Place p = place_of<V>(s);
    if (!p.active) return;
    const Channels<V> c = load_channels<V>(s, p, moments, weight, bias);
    const uint64_t seed = dropout_seed(d);
    const size_t base = (size_t)p.image * s.x_image + p.channel;
    const size_t out = (size_t)p.image * s.pixels * s.channels + p.channel;
    const auto one = [&](uint32_t r, const PackedVector<D, V>& packed) {
        float v[V];
        unpack<D, V>(packed, v);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = fmaf((v[j] - c.mean[j]) * c.rstd[j], c.weight[j], c.bias[j]);
        activate<V>(s.activation, v);
        const size_t at = out + (size_t)r * s.channels;
        if (d.on) dropout_apply<V>(d, seed, at, v);
        store_vector<D, V>(y, at, v);
    };
    uint32_t r = p.begin + p.row;
    for (; r + (kUnroll - 1) * s.rows < p.end; r += kUnroll * s.rows) {
        PackedVector<D, V> packed[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) packed[k] = load_packed<D, V>(x, base + (size_t)(r + k * s.rows) * s.x_pixel);
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) one(r + k * s.rows, packed[k]);
    }
    for (; r < p.end; r += s.rows) one(r, load_packed<D, V>(x, base + (size_t)r * s.x_pixel));
}

// ---- backward: {sum dz, sum dz * xhat} of every (image, slab, channel) -----------------------------------------------
// dz of one vector; xhat is left in v
template <int V>
__device__ __forceinline__ void gradient_of_z(const Shape& s, const Channels<V>& c, const Dropout& d, uint64_t seed, uint64_t at,
                                              float (&v)[V], float (&g)[V]) {
    float z[V];
    if (d.on) dropout_apply<V>(d, seed, at, g);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        v[j] = (v[j] - c.mean[j]) * c.rstd[j];
        z[j] = fmaf(v[j], c.weight[j], c.bias[j]);
    }
    activate_backward<V>(s.activation, z, g);
}

template <int D, int V>
__global__ void __launch_bounds__(kThreads) k_gradient_sums(const void* __restrict__ x, const void* __restrict__ dy,
                                                            const float2* __restrict__ moments, const void* __restrict__ weight,
                                                            const void* __restrict__ bias, float2* __restrict__ partial, Shape s,
                                                            Dropout d) {
    __shared__ float2 merged[kThreads * V];
    const Place p = place_of<V>(s);
    float sum[V], product[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = product[j] = 0.0f;
    if (p.active) {
        const Channels<V> c = load_channels<V>(s, p, moments, weight, bias);
        const uint64_t seed = dropout_seed(d);
        const size_t base = (size_t)p.image * s.x_image + p.channel, gbase = (size_t)p.image * s.g_image + p.channel;
        const size_t out = (size_t)p.image * s.pixels * s.channels + p.channel;
        const auto one = [&](uint32_t r, const PackedVector<D, V>& px, const PackedVector<D, V>& pg) {
            float v[V], g[V];
            unpack<D, V>(px, v);
            unpack<D, V>(pg, g);
            gradient_of_z<V>(s, c, d, seed, out + (size_t)r * s.channels, v, g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                sum[j] += g[j];
                product[j] = fmaf(g[j], v[j], product[j]);
            }
        };
        uint32_t r = p.begin + p.row;
        for (; r + (kUnroll - 1) * s.rows < p.end; r += kUnroll * s.rows) {
            PackedVector<D, V> px[kUnroll], pg[kUnroll];
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                px[k] = load_packed<D, V>(x, base + (size_t)(r + k * s.rows) * s.x_pixel);
                pg[k] = load_packed<D, V>(dy, gbase + (size_t)(r + k * s.rows) * s.g_pixel);
            }
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) one(r + k * s.rows, px[k], pg[k]);
        }
        for (; r < p.end; r += s.rows)
            one(r, load_packed<D, V>(x, base + (size_t)r * s.x_pixel), load_packed<D, V>(dy, gbase + (size_t)r * s.g_pixel));
    }
#pragma unroll
    for (int j = 0; j < V; ++j) merged[threadIdx.x * V + j] = make_float2(sum[j], product[j]);
    uint32_t half = 1;
    while (half < s.rows) half <<= 1;
    for (half >>= 1; half > 0; half >>= 1) {
        __syncthreads();
        if (p.row < half && p.row + half < s.rows) {
            const uint32_t other = threadIdx.x + half * s.columns;
            for (int j = 0; j < V; ++j) {
                float2 a = merged[threadIdx.x * V + j];
                const float2 b = merged[other * V + j];
                a.x += b.x;
                a.y += b.y;
                merged[threadIdx.x * V + j] = a;
            }
        }
    }
    if (p.active && p.row == 0) {
        const size_t at = ((size_t)p.image * s.slabs + p.slab) * s.channels + p.channel;
        for (int j = 0; j < V; ++j) partial[at + j] = merged[threadIdx.x * V + j];
    }
}

// ... summed over the slabs: per (image, channel) into `sums`, and per (image, group) the means A and B. A block per (image,
// group); `lanes` threads share a channel's slabs, per_group channels at a time.
__global__ void __launch_bounds__(kThreads) k_group_gradients(const float2* __restrict__ partial, const void* __restrict__ weight,
                                                              float2* __restrict__ sums, float2* __restrict__ means, Shape s) {
    __shared__ float2 merged[kThreads];
    const uint32_t image = blockIdx.x / s.groups, group = blockIdx.x % s.groups;
    const uint32_t width = min(s.per_group, (uint32_t)kThreads), lanes = kThreads / width;
    const uint32_t lane = threadIdx.x / width;
    float a = 0.0f, b = 0.0f;
    for (uint32_t first = 0; first < s.per_group; first += width) {
        const uint32_t in_group = first + threadIdx.x % width, channel = group * s.per_group + in_group;
        const bool mine = lane < lanes && in_group < s.per_group;
        float2 t = make_float2(0.0f, 0.0f);
        if (mine)
            for (uint32_t slab = lane; slab < s.slabs; slab += lanes) {
                const float2 v = partial[((size_t)image * s.slabs + slab) * s.channels + channel];
                t.x += v.x;
                t.y += v.y;
            }
        __syncthreads();
        merged[threadIdx.x] = t;
        __syncthreads();
        if (mine && lane == 0) {
            for (uint32_t l = 1; l < lanes; ++l) {
                t.x += merged[threadIdx.x + l * width].x;
                t.y += merged[threadIdx.x + l * width].y;
            }
            sums[(size_t)image * s.channels + channel] = t;
            const float w = weight ? load_element(weight, s.param_dtype, channel) : 1.0f;
            a = fmaf(w, t.x, a);
            b = fmaf(w, t.y, b);
        }
    }
    __syncthreads();
    merged[threadIdx.x] = make_float2(a, b);
    for (uint32_t half = kThreads / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (threadIdx.x < half) {
            merged[threadIdx.x].x += merged[threadIdx.x + half].x;
            merged[threadIdx.x].y += merged[threadIdx.x + half].y;
        }
    }
    if (threadIdx.x == 0) {
        const float count = (float)s.pixels * (float)s.per_group;
        means[blockIdx.x] = make_float2(merged[0].x / count, merged[0].y / count);
    }
}

// dbias and dweight: the sums of all images, a block per channel
__global__ void __launch_bounds__(kThreads) k_parameter_gradients(const float2* __restrict__ sums, void* __restrict__ dweight,
                                                                  void* __restrict__ dbias, Shape s) {
    __shared__ float2 merged[kThreads];
    float2 t = make_float2(0.0f, 0.0f);
    for (uint32_t image = threadIdx.x; image < s.n; image += kThreads) {
        const float2 v = sums[(size_t)image * s.channels + blockIdx.x];
        t.x += v.x;
        t.y += v.y;
    }
    merged[threadIdx.x] = t;
    for (uint32_t half = kThreads / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (threadIdx.x < half) {
            merged[threadIdx.x].x += merged[threadIdx.x + half].x;
            merged[threadIdx.x].y += merged[threadIdx.x + half].y;
        }
    }
    if (threadIdx.x == 0) {
        if (dbias) store_element(dbias, s.param_dtype, blockIdx.x, merged[0].x);
        if (dweight) store_element(dweight, s.param_dtype, blockIdx.x, merged[0].y);
    }
}

template <int D, int V>
__global__ void __launch_bounds__(kThreads) k_input_gradient(const void* __restrict__ x, const void* __restrict__ dy,
                                                             const float2* __restrict__ moments, const float2* __restrict__ means,
                                                             const void* __restrict__ weight, const void* __restrict__ bias,
                                                             void* __restrict__ dx, Shape s, Dropout d) {
    const Place p = place_of<V>(s);
    if (!p.active) return;
    const Channels<V> c = load_channels<V>(s, p, moments, weight, bias);
    float mean_a[V], mean_b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float2 m = means[(size_t)p.image * s.groups + (p.channel + j) / s.per_group];
        mean_a[j] = m.x;
        mean_b[j] = m.y;
    }
    const uint64_t seed = dropout_seed(d);
    const size_t base = (size_t)p.image * s.x_image + p.channel, gbase = (size_t)p.image * s.g_image + p.channel;
    const size_t out = (size_t)p.image * s.pixels * s.channels + p.channel;
    const auto one = [&](uint32_t r, const PackedVector<D, V>& px, const PackedVector<D, V>& pg) {
        float v[V], g[V];
        unpack<D, V>(px, v);
        unpack<D, V>(pg, g);
        const size_t at = out + (size_t)r * s.channels;
        gradient_of_z<V>(s, c, d, seed, at, v, g);
#pragma unroll
        for (int j = 0; j < V; ++j) g[j] = (fmaf(g[j], c.weight[j], -mean_a[j]) - v[j] * mean_b[j]) * c.rstd[j];
        store_vector<D, V>(dx, at, g);
    };
    uint32_t r = p.begin + p.row;
    for (; r + (kUnroll - 1) * s.rows < p.end; r += kUnroll * s.rows) {
        PackedVector<D, V> px[kUnroll], pg[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            px[k] = load_packed<D, V>(x, base + (size_t)(r + k * s.rows) * s.x_pixel);
            pg[k] = load_packed<D, V>(dy, gbase + (size_t)(r + k * s.rows) * s.g_pixel);
        }
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) one(r + k * s.rows, px[k], pg[k]);
    }
    for (; r < p.end; r += s.rows)
        one(r, load_packed<D, V>(x, base + (size_t)r * s.x_pixel), load_packed<D, V>(dy, gbase + (size_t)r * s.g_pixel));
}

// ---- host side -----------------------------------------------------------------------------------------------------

// Elements of a vector: the largest power of two up to 16 bytes that divides the channels, every stride and every pointer.
// `divisible` and `pointers` are the bitwise or of these: a power of two divides all of them iff it divides that.
inline int vector_width(size_t bytes, uint64_t divisible, uintptr_t pointers) {
    int v = (int)(16 / bytes);
    while (v > 1 && (divisible % v != 0 || pointers % (v * bytes) != 0)) v /= 2;
    return v;
}

inline Shape make_shape(const inpc_group_norm_config& cfg, int v, uint32_t fill_blocks) {
    Shape s{};
    s.n = cfg.n_images;
    s.pixels = cfg.n_pixels;
    s.channels = cfg.channels;
    s.groups = cfg.groups;
    s.per_group = cfg.channels / cfg.groups;
    s.x_image = cfg.input_image_stride;
    s.x_pixel = cfg.input_pixel_stride;
    s.g_image = cfg.grad_image_stride;
    s.g_pixel = cfg.grad_pixel_stride;
    s.activation = cfg.activation;
    s.param_dtype = cfg.param_dtype;
    s.eps = cfg.eps;
    const uint32_t vectors = cfg.channels / (uint32_t)v;
    s.tiles = div_up(vectors, kThreads);
    s.columns = div_up(vectors, s.tiles);
    s.rows = kThreads / s.columns;
    const uint64_t per_image = std::max<uint64_t>(1, fill_blocks / ((uint64_t)s.n * s.tiles));
    const uint32_t step = s.rows * kUnroll;
    const uint64_t wanted = (s.pixels + per_image - 1) / per_image;
    s.slab_pixels = (uint32_t)std::min<uint64_t>((wanted + step - 1) / step * step, 0x7FFFFFFFu);
    s.slabs = div_up(s.pixels, s.slab_pixels);
    return s;
}

// The smallest vector the configuration can lead to gives the most slabs: what the workspace is sized for.
inline uint32_t most_slabs(const inpc_group_norm_config& cfg) {
    uint32_t most = 1;
    for (int v = (int)(16 / element_bytes(cfg.dtype)); v >= 1; v /= 2)
        if (cfg.channels % (uint32_t)v == 0) most = std::max(most, make_shape(cfg, v, kFillBlocks).slabs);
    return most;
}

// [moments or gradient sums per (image, slab, channel)] [gradient sums per (image, channel)] [means per (image, group)]
struct Workspace {
    size_t partial, sums, means, bytes;
};
inline Workspace workspace_of(const inpc_group_norm_config& cfg) {
    Workspace w;
    w.partial = 0;
    w.sums = align_up((size_t)cfg.n_images * most_slabs(cfg) * cfg.channels * sizeof(float2), 256);
    w.means = w.sums + align_up((size_t)cfg.n_images * cfg.channels * sizeof(float2), 256);
    w.bytes = w.means + align_up((size_t)cfg.n_images * cfg.groups * sizeof(float2), 256);
    return w;
}

inline int check_config(const inpc_group_norm_config* cfg, const char* what) {
    if (!cfg) return fail(INPC_E_INVALID_ARGUMENT, "%s: null configuration", what);
    if (!known_dtype(cfg->dtype) || !(cfg->param_dtype == INPC_DTYPE_F32 || cfg->param_dtype == cfg->dtype))
        return fail(INPC_E_UNSUPPORTED, "%s: values are fp32, fp16 or bf16, parameters fp32 or of the values' type", what);
    if (cfg->activation < INPC_ACTIVATION_NONE || cfg->activation > INPC_ACTIVATION_GELU)
        return fail(INPC_E_UNSUPPORTED, "%s: unknown activation %d", what, cfg->activation);
    if (cfg->channels == 0 || cfg->groups == 0 || cfg->channels % cfg->groups != 0)
        return fail(INPC_E_INVALID_ARGUMENT, "%s: %u channels cannot be split into %u groups", what, cfg->channels, cfg->groups);
    if (cfg->channels > INPC_GROUP_NORM_MAX_CHANNELS || cfg->n_pixels >= (1u << 30))
        return fail(INPC_E_UNSUPPORTED, "%s: at most %u channels and fewer than 2^30 pixels per image", what,
                    INPC_GROUP_NORM_MAX_CHANNELS);
    if (!(cfg->eps >= 0.0f)) return fail(INPC_E_INVALID_ARGUMENT, "%s: eps must not be negative", what);
    if (!valid_probability(cfg->dropout_p)) return fail(INPC_E_INVALID_ARGUMENT, "%s: the dropout probability is outside [0, 1]", what);
    return INPC_OK;
}

inline int check_workspace(const inpc_group_norm_config& cfg, const void* workspace, size_t bytes, const char* what) {
    const size_t needed = workspace_of(cfg).bytes;
    if (!workspace || bytes < needed || (uintptr_t)workspace % 16 != 0)
        return fail(INPC_E_WORKSPACE, "%s: the workspace holds %zu bytes, %zu are needed, 16-byte aligned", what, bytes, needed);
    return INPC_OK;
}

// Blocks of a launch over all slabs, channel tiles and images, or an error where they are too many.
inline int grid_blocks(const Shape& s, const char* what, uint32_t& blocks) {
    const uint64_t b = (uint64_t)s.slabs * s.tiles * s.n, per_group = (uint64_t)s.n * s.groups;
    if (b > 0x7FFFFFFFu || per_group > 0x7FFFFFFFu) return fail(INPC_E_UNSUPPORTED, "%s: too many images", what);
    blocks = (uint32_t)b;
    return INPC_OK;
}

template <int D, int V>
int forward(const inpc_group_norm_config& cfg, const void* x, const void* weight, const void* bias, void* y, float2* moments,
            char* ws, hipStream_t stream) {
    const Shape s = make_shape(cfg, V, kFillBlocks);
    const Dropout d = make_dropout(cfg.dropout_p, cfg.seed, cfg.seed_dev, cfg.offset);
    uint32_t blocks = 0;
    if (const int rc = grid_blocks(s, "group_norm_forward", blocks)) return rc;
    float2* partial = (float2*)(ws + workspace_of(cfg).partial);
    INPC_LAUNCH("group_norm_moments", (k_moments<D, V>), dim3(blocks), dim3(kThreads), stream, x, partial, s);
    INPC_LAUNCH("group_norm_group_moments", k_group_moments, dim3(s.n * s.groups), dim3(kThreads), stream, partial, moments, s);
    INPC_LAUNCH("group_norm_apply", (k_apply<D, V>), dim3(blocks), dim3(kThreads), stream, x, moments, weight, bias, y, s, d);
    return INPC_OK;
}

template <int D, int V>
int backward(const inpc_group_norm_config& cfg, const void* x, const void* dy, const float2* moments, const void* weight,
             const void* bias, void* dx, void* dweight, void* dbias, char* ws, hipStream_t stream) {
    const Shape s = make_shape(cfg, V, kFillBlocks);
    const Dropout d = make_dropout(cfg.dropout_p, cfg.seed, cfg.seed_dev, cfg.offset);
    uint32_t blocks = 0;
    if (const int rc = grid_blocks(s, "group_norm_backward", blocks)) return rc;
    const Workspace w = workspace_of(cfg);
    float2 *partial = (float2*)(ws + w.partial), *sums = (float2*)(ws + w.sums), *means = (float2*)(ws + w.means);
    INPC_LAUNCH("group_norm_gradient_sums", (k_gradient_sums<D, V>), dim3(blocks), dim3(kThreads), stream, x, dy, moments, weight,
                bias, partial, s, d);
    INPC_LAUNCH("group_norm_group_gradients", k_group_gradients, dim3(s.n * s.groups), dim3(kThreads), stream, partial, weight,
                sums, means, s);
    if (dweight || dbias)
        INPC_LAUNCH("group_norm_parameter_gradients", k_parameter_gradients, dim3(s.channels), dim3(kThreads), stream, sums,
                    dweight, dbias, s);
    if (dx)
        INPC_LAUNCH("group_norm_input_gradient", (k_input_gradient<D, V>), dim3(blocks), dim3(kThreads), stream, x, dy, moments,
                    means, weight, bias, dx, s, d);
    return INPC_OK;
}

// Calls f<dtype, vector width>(args...).
#define INPC_NORM_DISPATCH(f, dtype, v, ...)                                                              \
    ((dtype) == INPC_DTYPE_F32   ? ((v) == 4 ? f<INPC_DTYPE_F32, 4>(__VA_ARGS__)                           \
                                    : (v) == 2 ? f<INPC_DTYPE_F32, 2>(__VA_ARGS__)                         \
                                               : f<INPC_DTYPE_F32, 1>(__VA_ARGS__))                        \
     : (dtype) == INPC_DTYPE_F16 ? ((v) == 8   ? f<INPC_DTYPE_F16, 8>(__VA_ARGS__)                         \
                                    : (v) == 4 ? f<INPC_DTYPE_F16, 4>(__VA_ARGS__)                         \
                                    : (v) == 2 ? f<INPC_DTYPE_F16, 2>(__VA_ARGS__)                         \
                                               : f<INPC_DTYPE_F16, 1>(__VA_ARGS__))                        \
                                 : ((v) == 8   ? f<INPC_DTYPE_BF16, 8>(__VA_ARGS__)                        \
                                    : (v) == 4 ? f<INPC_DTYPE_BF16, 4>(__VA_ARGS__)                        \
                                    : (v) == 2 ? f<INPC_DTYPE_BF16, 2>(__VA_ARGS__)                        \
                                               : f<INPC_DTYPE_BF16, 1>(__VA_ARGS__)))

}  // namespace norm
}  // namespace inpc
