// groupnorm.hpp — group norm with an activation and optional dropout over channels-last feature maps, forward and backward.
//
//   xhat = (x - mean) / sqrt(var + eps)   mean, var (biased) over the pixels of one image and the channels of one group
//   z = xhat * weight + bias,  y = activation(z),  then dropout (elements.hpp)
//   backward: dz = dy * activation'(z);  dbias = sum dz, dweight = sum dz * xhat over images and pixels;
//   dx = (weight * dz - A - xhat * B) / sqrt(var + eps), A and B the group's means of weight * dz and weight * dz * xhat
//
// Two forms. "single": a block per (image, group) does everything in one launch, from registers where the group fits them;
// for maps whose launches cost more than their bytes. "split": a block per run of pixels (a slab) of an image and all
// of its channels, so that it reads whole runs of memory; one launch writes each slab's sums, the next adds
// them up at the start of every block and applies. In both a thread keeps one vector of channels (16 bytes where channel
// counts, strides and pointers allow). Sums are fp32 in an order that depends on sizes and alignments alone (no atomics);
// deviations are taken from a mean, never squares from squares, so that nothing cancels however far the values are from 0.
#pragma once

#include <algorithm>

#include "elements.hpp"

namespace inpc {
namespace norm {

constexpr int kMaxThreads = 1024;        // of the single form
constexpr int kMaxThreadsBackward = 512; // ... whose threads need more registers here
constexpr int kHeld = 8;                 // vectors of x, and in the backward pass of dy, a thread of it keeps in registers
constexpr int kThreads = 512;            // of the split form
constexpr int kUnroll = 4;               // pixels a thread of it has in flight
constexpr uint32_t kFillBlocks = 512;    // blocks that fill the chip: two per compute unit
constexpr uint32_t kFoldedSums = 8192;   // slab sums of an image up to which every block adds them up itself
constexpr uint32_t kParameterColumns = 32;

struct Shape {
    uint64_t x_image, x_pixel;   // strides of x in elements (channels are adjacent); y and dx are dense
    uint64_t g_image, g_pixel;   // of the gradient of y
    uint32_t n, pixels, channels, groups, per_group;
    uint32_t columns, rows;      // threads of a block: vectors side by side, pixels at once
    uint32_t slabs, slab_pixels; // split form, per image
    int32_t activation, param_dtype;
    float eps;
};

// ---- sums over a block -----------------------------------------------------------------------------------------------
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// The sum of all threads' values, in every thread. `lds`: one float per wave; free again when the next barrier has passed.
__device__ __forceinline__ float block_sum(float v, float* lds) {
    v = wave_sum(v);
    const uint32_t waves = blockDim.x / 64u;
    __syncthreads();
    if (lane_id() == 0) lds[threadIdx.x / 64u] = v;
    __syncthreads();
    float total = 0.0f;
    for (uint32_t w = 0; w < waves; ++w) total += lds[w];
    return total;
}

// Adds N values per thread over the threads of a column (thread = row * columns + column; threads beyond rows * columns
// bring zeros). Returns where the totals lie in LDS, [column][N], for every thread to read until the next call.
// `lds` holds blockDim.x * N + 32 * N floats.
template <int N>
__device__ __forceinline__ const float* column_sums(const float (&values)[N], uint32_t columns, uint32_t rows, float* lds) {
    const uint32_t t = threadIdx.x;
    __syncthreads();
    if (columns <= 32u && (columns & (columns - 1u)) == 0u) {
        // the lanes of a wave first, then the waves
        float v[N];
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = values[j];
        for (uint32_t o = columns; o < 64u; o <<= 1)
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] += __shfl_xor(v[j], (int)o, 64);
        const uint32_t waves = blockDim.x / 64u, width = columns * N;
        if (lane_id() < columns)
#pragma unroll
            for (int j = 0; j < N; ++j) lds[(t / 64u) * width + lane_id() * N + j] = v[j];
        __syncthreads();
        float* total = lds + blockDim.x * N;
        for (uint32_t i = t; i < width; i += blockDim.x) {
            float sum = 0.0f;
            for (uint32_t w = 0; w < waves; ++w) sum += lds[w * width + i];
            total[i] = sum;
        }
        __syncthreads();
        return total;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) lds[t * N + j] = values[j];
    const uint32_t row = t / columns;
    uint32_t half = 1;
    while (half < rows) half <<= 1;
    for (half >>= 1; half > 0; half >>= 1) {
        __syncthreads();
        if (row < half && row + half < rows)
#pragma unroll
            for (int j = 0; j < N; ++j) lds[t * N + j] += lds[(t + half * columns) * N + j];
    }
    __syncthreads();
    return lds;
}

// Two sets of values merged: counts na and nb, means, sums of squared deviations (Chan, Golub, LeVeque 1979).
__device__ __forceinline__ void merge_moments(float& na, float& mean, float& m2, float nb, float mean_b, float m2_b) {
    if (nb == 0.0f) return;
    const float n = na + nb, d = mean_b - mean, share = nb / n;
    mean = fmaf(d, share, mean);
    m2 += fmaf(d * d, na * share, m2_b);
    na = n;
}

// ---- activations -----------------------------------------------------------------------------------------------------
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

// ---- one vector ------------------------------------------------------------------------------------------------------
template <int V>
struct Parameters {
    float weight[V], bias[V];
};
template <int V>
__device__ __forceinline__ Parameters<V> load_parameters(const Shape& s, const void* weight, const void* bias, uint32_t channel) {
    Parameters<V> p;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        p.weight[j] = weight ? load_element(weight, s.param_dtype, channel + j) : 1.0f;
        p.bias[j] = bias ? load_element(bias, s.param_dtype, channel + j) : 0.0f;
    }
    return p;
}

// The moments of a vector's channels: one pair where all of them lie in one group (M = 1), else a pair each (M = V).
template <int M>
struct Moments {
    float mean[M], rstd[M];
};

template <int D, int V, int M>
__device__ __forceinline__ void apply_vector(const Shape& s, const Dropout& d, uint64_t seed, const Moments<M>& m,
                                             const Parameters<V>& p, const PackedVector<D, V>& packed, void* y, size_t at) {
    float v[V];
    unpack<D, V>(packed, v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = fmaf((v[j] - m.mean[j % M]) * m.rstd[j % M], p.weight[j], p.bias[j]);
    activate<V>(s.activation, v);
    if (d.on) dropout_apply<V>(d, seed, at, v);
    store_vector<D, V>(y, at, v);
}

// xhat in v and dz in g
template <int D, int V, int M>
__device__ __forceinline__ void gradient_vector(const Shape& s, const Dropout& d, uint64_t seed, const Moments<M>& m,
                                                const Parameters<V>& p, const PackedVector<D, V>& px, const PackedVector<D, V>& pg,
                                                size_t at, float (&v)[V], float (&g)[V]) {
    float z[V];
    unpack<D, V>(px, v);
    unpack<D, V>(pg, g);
    if (d.on) dropout_apply<V>(d, seed, at, g);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        v[j] = (v[j] - m.mean[j % M]) * m.rstd[j % M];
        z[j] = fmaf(v[j], p.weight[j], p.bias[j]);
    }
    activate_backward<V>(s.activation, z, g);
}

template <int D, int V, int M>
__device__ __forceinline__ void input_gradient_vector(const Shape& s, const Dropout& d, uint64_t seed, const Moments<M>& m,
                                                      const float (&mean_a)[M], const float (&mean_b)[M], const Parameters<V>& p,
                                                      const PackedVector<D, V>& px, const PackedVector<D, V>& pg, void* dx, size_t at) {
    float v[V], g[V];
    gradient_vector<D, V, M>(s, d, seed, m, p, px, pg, at, v, g);
#pragma unroll
    for (int j = 0; j < V; ++j) g[j] = (fmaf(g[j], p.weight[j], -mean_a[j % M]) - v[j] * mean_b[j % M]) * m.rstd[j % M];
    store_vector<D, V>(dx, at, g);
}

// ---- the single form -------------------------------------------------------------------------------------------------
// Blocks go to the eight dies in turn: neighbouring (image, group) pairs, which share cache lines, go to one die.
__device__ __forceinline__ uint32_t swizzled_block() {
    const uint32_t share = gridDim.x / 8u;
    return blockIdx.x < share * 8u ? (blockIdx.x % 8u) * share + blockIdx.x / 8u : blockIdx.x;
}

template <int D, int V>
__global__ void __launch_bounds__(kMaxThreads) k_single(const void* __restrict__ x, const void* __restrict__ weight,
                                                        const void* __restrict__ bias, void* __restrict__ y,
                                                        float2* __restrict__ moments, Shape s, Dropout d) {
    __shared__ float lds[kMaxThreads / 64];
    const uint32_t b = swizzled_block(), image = b / s.groups, first = b % s.groups * s.per_group;
    const uint32_t column = threadIdx.x % s.columns, row = threadIdx.x / s.columns, vectors = s.per_group / V;
    const size_t base = (size_t)image * s.x_image + first, out = (size_t)image * s.pixels * s.channels + first;
    const float count = (float)s.pixels * (float)s.per_group;
    const bool held = s.columns == vectors && s.pixels <= s.rows * kHeld, active = row < s.rows;
    PackedVector<D, V> px[kHeld];
    Moments<1> m;
    float variance;
    if (held) {
        // the whole group is in the block's registers: its mean, then the squares of the deviations from that
        float sum = 0.0f, squares = 0.0f;
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
            if (active && row + k * s.rows < s.pixels) px[k] = load_packed<D, V>(x, base + (size_t)(row + k * s.rows) * s.x_pixel + column * V);
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
            if (active && row + k * s.rows < s.pixels) {
                float v[V];
                unpack<D, V>(px[k], v);
#pragma unroll
                for (int j = 0; j < V; ++j) sum += v[j];
            }
        m.mean[0] = block_sum(sum, lds) / count;
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
            if (active && row + k * s.rows < s.pixels) {
                float v[V];
                unpack<D, V>(px[k], v);
#pragma unroll
                for (int j = 0; j < V; ++j) squares = fmaf(v[j] - m.mean[0], v[j] - m.mean[0], squares);
            }
        variance = block_sum(squares, lds) / count;
    } else {
        // a thread's values vector by vector, then the threads
        float n = 0.0f, mean = 0.0f, m2 = 0.0f;
        if (active)
            for (uint32_t c = column; c < vectors; c += s.columns)
                for (uint32_t r = row; r < s.pixels; r += s.rows) {
                    float v[V], vector_mean = 0.0f, vector_m2 = 0.0f;
                    load_vector<D, V>(x, base + (size_t)r * s.x_pixel + c * V, v);
#pragma unroll
                    for (int j = 0; j < V; ++j) vector_mean += v[j];
                    vector_mean *= 1.0f / V;
#pragma unroll
                    for (int j = 0; j < V; ++j) vector_m2 = fmaf(v[j] - vector_mean, v[j] - vector_mean, vector_m2);
                    merge_moments(n, mean, m2, (float)V, vector_mean, vector_m2);
                }
        m.mean[0] = block_sum(n * mean, lds) / count;
        variance = block_sum(fmaf(n * (mean - m.mean[0]), mean - m.mean[0], m2), lds) / count;
    }
    m.rstd[0] = 1.0f / sqrtf(variance + s.eps);
    if (threadIdx.x == 0) moments[b] = make_float2(m.mean[0], m.rstd[0]);
    if (!active) return;
    const uint64_t seed = dropout_seed(d);
    if (held) {
        const Parameters<V> p = load_parameters<V>(s, weight, bias, first + column * V);
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            const uint32_t r = row + k * s.rows;
            if (r < s.pixels) apply_vector<D, V, 1>(s, d, seed, m, p, px[k], y, out + (size_t)r * s.channels + column * V);
        }
        return;
    }
    for (uint32_t c = column; c < vectors; c += s.columns) {
        const Parameters<V> p = load_parameters<V>(s, weight, bias, first + c * V);
        for (uint32_t r = row; r < s.pixels; r += s.rows)
            apply_vector<D, V, 1>(s, d, seed, m, p, load_packed<D, V>(x, base + (size_t)r * s.x_pixel + c * V), y,
                                  out + (size_t)r * s.channels + c * V);
    }
}

// With one image dbias and dweight come from here, with more the sums of every (image, channel) do.
template <int D, int V>
__global__ void __launch_bounds__(kMaxThreadsBackward) k_single_backward(const void* __restrict__ x, const void* __restrict__ dy,
                                                                 const float2* __restrict__ moments,
                                                                 const void* __restrict__ weight, const void* __restrict__ bias,
                                                                 void* __restrict__ dx, void* __restrict__ dweight,
                                                                 void* __restrict__ dbias, float2* __restrict__ sums, Shape s,
                                                                 Dropout d) {
    INPC_DYNAMIC_LDS(float, lds);   // column_sums of 2 V values per thread
    __shared__ float waves[kMaxThreadsBackward / 64];
    const uint32_t b = swizzled_block(), image = b / s.groups, first = b % s.groups * s.per_group;
    const uint32_t column = threadIdx.x % s.columns, row = threadIdx.x / s.columns, vectors = s.per_group / V;
    const size_t base = (size_t)image * s.x_image + first, gbase = (size_t)image * s.g_image + first;
    const size_t out = (size_t)image * s.pixels * s.channels + first;
    const bool held = s.columns == vectors && s.pixels <= s.rows * kHeld, active = row < s.rows;
    const uint64_t seed = dropout_seed(d);
    const Moments<1> m{{moments[b].x}, {moments[b].y}};
    PackedVector<D, V> px[kHeld], pg[kHeld];
    float a = 0.0f, bb = 0.0f;
    for (uint32_t tile = 0; tile < vectors; tile += s.columns) {
        const uint32_t c = tile + column;
        const bool mine = active && c < vectors;
        float total[2 * V];
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) total[j] = 0.0f;
        const auto add = [&](const Parameters<V>& p, const PackedVector<D, V>& vx, const PackedVector<D, V>& vg, uint32_t r) {
            float v[V], g[V];
            gradient_vector<D, V, 1>(s, d, seed, m, p, vx, vg, out + (size_t)r * s.channels + c * V, v, g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                total[j] += g[j];
                total[V + j] = fmaf(g[j], v[j], total[V + j]);
            }
        };
        if (mine) {
            const Parameters<V> p = load_parameters<V>(s, weight, bias, first + c * V);
            if (held) {
#pragma unroll
                for (int k = 0; k < kHeld; ++k) {
                    const uint32_t r = row + k * s.rows;
                    if (r < s.pixels) {
                        px[k] = load_packed<D, V>(x, base + (size_t)r * s.x_pixel + c * V);
                        pg[k] = load_packed<D, V>(dy, gbase + (size_t)r * s.g_pixel + c * V);
                    }
                }
#pragma unroll
                for (int k = 0; k < kHeld; ++k)
                    if (row + k * s.rows < s.pixels) add(p, px[k], pg[k], row + k * s.rows);
            } else {
                for (uint32_t r = row; r < s.pixels; r += s.rows)
                    add(p, load_packed<D, V>(x, base + (size_t)r * s.x_pixel + c * V),
                        load_packed<D, V>(dy, gbase + (size_t)r * s.g_pixel + c * V), r);
            }
        }
        const float* columns = column_sums<2 * V>(total, s.columns, s.rows, lds);
        const uint32_t channels = min(s.columns, vectors - tile) * V;
        for (uint32_t i = threadIdx.x; i < channels; i += blockDim.x) {
            const float sum = columns[i / V * (2 * V) + i % V], product = columns[i / V * (2 * V) + V + i % V];
            const uint32_t channel = first + tile * V + i;
            const float w = weight ? load_element(weight, s.param_dtype, channel) : 1.0f;
            a = fmaf(w, sum, a);
            bb = fmaf(w, product, bb);
            if (sums) sums[(size_t)image * s.channels + channel] = make_float2(sum, product);
            if (dbias) store_element(dbias, s.param_dtype, channel, sum);
            if (dweight) store_element(dweight, s.param_dtype, channel, product);
        }
    }
    if (!dx) return;
    const float count = (float)s.pixels * (float)s.per_group;
    const float mean_a[1] = {block_sum(a, waves) / count}, mean_b[1] = {block_sum(bb, waves) / count};
    if (!active) return;
    for (uint32_t c = column; c < vectors; c += s.columns) {
        const Parameters<V> p = load_parameters<V>(s, weight, bias, first + c * V);
        const size_t at = out + c * V;
        if (held) {
#pragma unroll
            for (int k = 0; k < kHeld; ++k) {
                const uint32_t r = row + k * s.rows;
                if (r < s.pixels)
                    input_gradient_vector<D, V, 1>(s, d, seed, m, mean_a, mean_b, p, px[k], pg[k], dx, at + (size_t)r * s.channels);
            }
        } else {
            for (uint32_t r = row; r < s.pixels; r += s.rows)
                input_gradient_vector<D, V, 1>(s, d, seed, m, mean_a, mean_b, p,
                                               load_packed<D, V>(x, base + (size_t)r * s.x_pixel + c * V),
                                               load_packed<D, V>(dy, gbase + (size_t)r * s.g_pixel + c * V), dx,
                                               at + (size_t)r * s.channels);
        }
    }
}

// dbias and dweight from `rows` rows of sums, kParameterColumns channels to a block
__device__ __forceinline__ void add_parameter_gradients(const float2* sums, size_t rows, void* dweight, void* dbias, const Shape& s,
                                                        uint32_t block, float* lds) {
    const uint32_t channel = block * kParameterColumns + threadIdx.x % kParameterColumns;
    float total[2] = {0.0f, 0.0f};
    if (channel < s.channels)
        for (size_t r = threadIdx.x / kParameterColumns; r < rows; r += blockDim.x / kParameterColumns) {
            const float2 v = sums[r * s.channels + channel];
            total[0] += v.x;
            total[1] += v.y;
        }
    const float* all = column_sums<2>(total, kParameterColumns, blockDim.x / kParameterColumns, lds);
    if (threadIdx.x < kParameterColumns && channel < s.channels) {
        if (dbias) store_element(dbias, s.param_dtype, channel, all[2 * threadIdx.x]);
        if (dweight) store_element(dweight, s.param_dtype, channel, all[2 * threadIdx.x + 1]);
    }
}

__global__ void __launch_bounds__(kThreads) k_parameter_gradients(const float2* __restrict__ sums, void* __restrict__ dweight,
                                                                  void* __restrict__ dbias, Shape s) {
    __shared__ float lds[kThreads * 2 + 64];
    add_parameter_gradients(sums, s.n, dweight, dbias, s, blockIdx.x, lds);
}

// ---- the split form --------------------------------------------------------------------------------------------------
struct Place {
    uint32_t image, slab, channel, row, begin, end;
    bool active;
};

template <int V>
__device__ __forceinline__ Place place_of(const Shape& s, uint32_t block) {
    Place p;
    p.slab = block % s.slabs;
    p.image = block / s.slabs;
    p.row = threadIdx.x / s.columns;
    p.channel = threadIdx.x % s.columns * V;
    p.active = p.row < s.rows;
    p.begin = p.slab * s.slab_pixels;
    p.end = min(p.begin + s.slab_pixels, s.pixels);
    return p;
}

// Sums of per_group neighbouring channels, for all groups: totals[channel / V * N + channel % V + which * V] -> sums[group].
// A power of two of lanes shares a group.
template <int V, int N>
__device__ __forceinline__ void group_sums(const float* totals, int which, const Shape& s, float* sums) {
    uint32_t lanes = 64;
    while (lanes > 1 && lanes * s.groups > (uint32_t)kThreads) lanes >>= 1;
    const uint32_t lane = threadIdx.x % lanes;
    for (uint32_t base = 0; base < s.groups; base += kThreads / lanes) {
        const uint32_t group = base + threadIdx.x / lanes;
        float sum = 0.0f;
        if (group < s.groups)
            for (uint32_t c = group * s.per_group + lane; c < (group + 1) * s.per_group; c += lanes)
                sum += totals[c / V * N + c % V + which * V];
        for (uint32_t o = lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor(sum, (int)o, 64);
        if (lane == 0 && group < s.groups) sums[group] = sum;
    }
    __syncthreads();
}

// {mean, sum of squared deviations} of every (image, slab, group)
template <int D, int V>
__global__ void __launch_bounds__(kThreads) k_moments(const void* __restrict__ x, float2* __restrict__ partial, Shape s) {
    INPC_DYNAMIC_LDS(float, lds);   // column_sums, then one float per group
    float* group = lds + kThreads * V + 32 * V;
    const Place p = place_of<V>(s, blockIdx.x);
    float mean[V], m2[V], count = 0.0f, values[V];
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
                const float of_these = sum * (1.0f / kUnroll), d = of_these - mean[j];
#pragma unroll
                for (int k = 0; k < kUnroll; ++k) squares = fmaf(v[k][j] - of_these, v[k][j] - of_these, squares);
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
    const float in_group = (float)(p.end - p.begin) * (float)s.per_group;
    // the group's mean, then everybody's deviations from it
#pragma unroll
    for (int j = 0; j < V; ++j) values[j] = count * mean[j];
    group_sums<V, V>(column_sums<V>(values, s.columns, s.rows, lds), 0, s, group);
    if (p.active) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float d = mean[j] - group[(p.channel + j) / s.per_group] / in_group;
            values[j] = fmaf(count * d, d, m2[j]);
        }
    }
    float* squares = group + s.groups;
    group_sums<V, V>(column_sums<V>(values, s.columns, s.rows, lds), 0, s, squares);
    for (uint32_t g = threadIdx.x; g < s.groups; g += kThreads)
        partial[(size_t)blockIdx.x * s.groups + g] = make_float2(group[g] / in_group, squares[g]);
}

__device__ __forceinline__ float slab_count(const Shape& s, uint32_t slab) {
    return (float)(min((slab + 1) * s.slab_pixels, s.pixels) - slab * s.slab_pixels) * (float)s.per_group;
}

// The moments of one image's groups from its slabs': threads side by side take the groups, the others every so many slabs.
__device__ __forceinline__ void fold_moments(const float2* partial, const Shape& s, float4* lds, float2* result) {
    const uint32_t lanes = kThreads / s.groups, group = threadIdx.x % s.groups, lane = threadIdx.x / s.groups;
    float n = 0.0f, mean = 0.0f, m2 = 0.0f;
    if (lane < lanes)
        for (uint32_t slab = lane; slab < s.slabs; slab += lanes) {
            const float2 b = partial[(size_t)slab * s.groups + group];
            merge_moments(n, mean, m2, slab_count(s, slab), b.x, b.y);
        }
    lds[threadIdx.x] = make_float4(n, mean, m2, 0.0f);
    uint32_t half = 1;
    while (half < lanes) half <<= 1;
    for (half >>= 1; half > 0; half >>= 1) {
        __syncthreads();
        if (lane < half && lane + half < lanes) {
            float4 a = lds[threadIdx.x];
            const float4 b = lds[threadIdx.x + half * s.groups];
            merge_moments(a.x, a.y, a.z, b.x, b.y, b.z);
            lds[threadIdx.x] = a;
        }
    }
    __syncthreads();
    if (threadIdx.x < s.groups) {
        const float4 a = lds[threadIdx.x];
        result[threadIdx.x] = make_float2(a.y, 1.0f / sqrtf(a.z / a.x + s.eps));
    }
    __syncthreads();
}

// The same for maps of many groups, a wave per (image, group)
__global__ void __launch_bounds__(kThreads) k_combine_moments(const float2* __restrict__ partial, float2* __restrict__ moments,
                                                              Shape s) {
    const uint32_t item = blockIdx.x * (kThreads / 64) + threadIdx.x / 64u, image = item / s.groups, group = item % s.groups;
    if (image >= s.n) return;
    float n = 0.0f, mean = 0.0f, m2 = 0.0f;
    for (uint32_t slab = lane_id(); slab < s.slabs; slab += 64) {
        const float2 b = partial[((size_t)image * s.slabs + slab) * s.groups + group];
        merge_moments(n, mean, m2, slab_count(s, slab), b.x, b.y);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float nb = __shfl_xor(n, o, 64), mean_b = __shfl_xor(mean, o, 64), m2_b = __shfl_xor(m2, o, 64);
        merge_moments(n, mean, m2, nb, mean_b, m2_b);
    }
    if (lane_id() == 0) moments[item] = make_float2(mean, 1.0f / sqrtf(m2 / n + s.eps));
}

template <int V>
__device__ __forceinline__ Moments<V> channel_moments(const float2* of_image, const Shape& s, uint32_t channel) {
    Moments<V> m;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float2 v = of_image[(channel + j) / s.per_group];
        m.mean[j] = v.x;
        m.rstd[j] = v.y;
    }
    return m;
}

// `partial` is null where k_combine_moments has run; else the first block of each image also writes its moments.
template <int D, int V>
__global__ void __launch_bounds__(kThreads) k_apply(const void* __restrict__ x, const float2* __restrict__ partial,
                                                    const void* __restrict__ weight, const void* __restrict__ bias,
                                                    void* __restrict__ y, float2* __restrict__ moments, Shape s, Dropout d) {
    __shared__ float4 lds[kThreads];
    __shared__ float2 folded[kThreads];
    const Place p = place_of<V>(s, blockIdx.x);
    float2* global = moments + (size_t)p.image * s.groups;
    if (partial) {
        fold_moments(partial + (size_t)p.image * s.slabs * s.groups, s, lds, folded);
        if (p.slab == 0 && threadIdx.x < s.groups) global[threadIdx.x] = folded[threadIdx.x];
    }
    if (!p.active) return;
    const Moments<V> m = partial ? channel_moments<V>(folded, s, p.channel) : channel_moments<V>(global, s, p.channel);
    const Parameters<V> c = load_parameters<V>(s, weight, bias, p.channel);
    const uint64_t seed = dropout_seed(d);
    const size_t base = (size_t)p.image * s.x_image + p.channel;
    const size_t out = (size_t)p.image * s.pixels * s.channels + p.channel;
    uint32_t r = p.begin + p.row;
    for (; r + (kUnroll - 1) * s.rows < p.end; r += kUnroll * s.rows) {
        PackedVector<D, V> packed[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) packed[k] = load_packed<D, V>(x, base + (size_t)(r + k * s.rows) * s.x_pixel);
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
            apply_vector<D, V, V>(s, d, seed, m, c, packed[k], y, out + (size_t)(r + k * s.rows) * s.channels);
    }
    for (; r < p.end; r += s.rows)
        apply_vector<D, V, V>(s, d, seed, m, c, load_packed<D, V>(x, base + (size_t)r * s.x_pixel), y, out + (size_t)r * s.channels);
}

// {sum dz, sum dz * xhat} of every (image, slab, channel), and both weighted and summed of every (image, slab, group)
template <int D, int V>
__global__ void __launch_bounds__(kThreads) k_gradient_sums(const void* __restrict__ x, const void* __restrict__ dy,
                                                            const float2* __restrict__ moments, const void* __restrict__ weight,
                                                            const void* __restrict__ bias, float2* __restrict__ of_channels,
                                                            float2* __restrict__ of_groups, Shape s, Dropout d) {
    INPC_DYNAMIC_LDS(float, lds);   // column_sums of 2 V values per thread, then two floats per group
    float *group_a = lds + (kThreads + 32) * 2 * V, *group_b = group_a + s.groups;
    const Place p = place_of<V>(s, blockIdx.x);
    float total[2 * V];
#pragma unroll
    for (int j = 0; j < 2 * V; ++j) total[j] = 0.0f;
    Parameters<V> c;
    if (p.active) {
        const Moments<V> m = channel_moments<V>(moments + (size_t)p.image * s.groups, s, p.channel);
        c = load_parameters<V>(s, weight, bias, p.channel);
        const uint64_t seed = dropout_seed(d);
        const size_t base = (size_t)p.image * s.x_image + p.channel, gbase = (size_t)p.image * s.g_image + p.channel;
        const size_t out = (size_t)p.image * s.pixels * s.channels + p.channel;
        const auto add = [&](uint32_t r, const PackedVector<D, V>& px, const PackedVector<D, V>& pg) {
            float v[V], g[V];
            gradient_vector<D, V, V>(s, d, seed, m, c, px, pg, out + (size_t)r * s.channels, v, g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                total[j] += g[j];
                total[V + j] = fmaf(g[j], v[j], total[V + j]);
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
            for (int k = 0; k < kUnroll; ++k) add(r + k * s.rows, px[k], pg[k]);
        }
        for (; r < p.end; r += s.rows)
            add(r, load_packed<D, V>(x, base + (size_t)r * s.x_pixel), load_packed<D, V>(dy, gbase + (size_t)r * s.g_pixel));
    }
    float* totals = (float*)column_sums<2 * V>(total, s.columns, s.rows, lds);
    for (uint32_t i = threadIdx.x; i < s.channels; i += kThreads) {
        float *sum = totals + i / V * (2 * V) + i % V, *product = sum + V;
        of_channels[(size_t)blockIdx.x * s.channels + i] = make_float2(*sum, *product);
        const float w = weight ? load_element(weight, s.param_dtype, i) : 1.0f;
        *sum *= w;
        *product *= w;
    }
    __syncthreads();
    group_sums<V, 2 * V>(totals, 0, s, group_a);
    group_sums<V, 2 * V>(totals, 1, s, group_b);
    for (uint32_t g = threadIdx.x; g < s.groups; g += kThreads)
        of_groups[(size_t)blockIdx.x * s.groups + g] = make_float2(group_a[g], group_b[g]);
}

// The means A and B of one image's groups from its slabs' sums, as fold_moments
__device__ __forceinline__ void fold_gradients(const float2* partial, const Shape& s, float2* lds, float2* result) {
    const uint32_t lanes = kThreads / s.groups, group = threadIdx.x % s.groups, lane = threadIdx.x / s.groups;
    float2 t = make_float2(0.0f, 0.0f);
    if (lane < lanes)
        for (uint32_t slab = lane; slab < s.slabs; slab += lanes) {
            const float2 b = partial[(size_t)slab * s.groups + group];
            t.x += b.x;
            t.y += b.y;
        }
    lds[threadIdx.x] = t;
    uint32_t half = 1;
    while (half < lanes) half <<= 1;
    for (half >>= 1; half > 0; half >>= 1) {
        __syncthreads();
        if (lane < half && lane + half < lanes) {
            lds[threadIdx.x].x += lds[threadIdx.x + half * s.groups].x;
            lds[threadIdx.x].y += lds[threadIdx.x + half * s.groups].y;
        }
    }
    __syncthreads();
    if (threadIdx.x < s.groups) {
        const float count = (float)s.pixels * (float)s.per_group;
        result[threadIdx.x] = make_float2(lds[threadIdx.x].x / count, lds[threadIdx.x].y / count);
    }
    __syncthreads();
}

__global__ void __launch_bounds__(kThreads) k_combine_gradients(const float2* __restrict__ partial, float2* __restrict__ means,
                                                                Shape s) {
    const uint32_t item = blockIdx.x * (kThreads / 64) + threadIdx.x / 64u, image = item / s.groups, group = item % s.groups;
    if (image >= s.n) return;
    float a = 0.0f, b = 0.0f;
    for (uint32_t slab = lane_id(); slab < s.slabs; slab += 64) {
        const float2 v = partial[((size_t)image * s.slabs + slab) * s.groups + group];
        a += v.x;
        b += v.y;
    }
    a = wave_sum(a);
    b = wave_sum(b);
    const float count = (float)s.pixels * (float)s.per_group;
    if (lane_id() == 0) means[item] = make_float2(a / count, b / count);
}

// The first `parameter_blocks` blocks add up dweight and dbias, the others write dx. `means` where k_combine_gradients has run,
// else null.
template <int D, int V>
__global__ void __launch_bounds__(kThreads) k_input_gradient(const void* __restrict__ x, const void* __restrict__ dy,
                                                             const float2* __restrict__ moments, const float2* __restrict__ of_channels,
                                                             const float2* __restrict__ of_groups, const float2* __restrict__ means,
                                                             const void* __restrict__ weight, const void* __restrict__ bias,
                                                             void* __restrict__ dx, void* __restrict__ dweight,
                                                             void* __restrict__ dbias, uint32_t parameter_blocks, Shape s, Dropout d) {
    __shared__ float lds[kThreads * 2 + 64];
    __shared__ float2 folded[kThreads];
    if (blockIdx.x < parameter_blocks) {
        add_parameter_gradients(of_channels, (size_t)s.n * s.slabs, dweight, dbias, s, blockIdx.x, lds);
        return;
    }
    const Place p = place_of<V>(s, blockIdx.x - parameter_blocks);
    const float2* ab = means + (size_t)p.image * s.groups;
    if (!means) {
        fold_gradients(of_groups + (size_t)p.image * s.slabs * s.groups, s, (float2*)lds, folded);
        ab = folded;
    }
    if (!p.active) return;
    const Moments<V> m = channel_moments<V>(moments + (size_t)p.image * s.groups, s, p.channel);
    const Parameters<V> c = load_parameters<V>(s, weight, bias, p.channel);
    float mean_a[V], mean_b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float2 v = ab[(p.channel + j) / s.per_group];
        mean_a[j] = v.x;
        mean_b[j] = v.y;
    }
    const uint64_t seed = dropout_seed(d);
    const size_t base = (size_t)p.image * s.x_image + p.channel, gbase = (size_t)p.image * s.g_image + p.channel;
    const size_t out = (size_t)p.image * s.pixels * s.channels + p.channel;
    uint32_t r = p.begin + p.row;
    for (; r + (kUnroll - 1) * s.rows < p.end; r += kUnroll * s.rows) {
        PackedVector<D, V> px[kUnroll], pg[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            px[k] = load_packed<D, V>(x, base + (size_t)(r + k * s.rows) * s.x_pixel);
            pg[k] = load_packed<D, V>(dy, gbase + (size_t)(r + k * s.rows) * s.g_pixel);
        }
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
            input_gradient_vector<D, V, V>(s, d, seed, m, mean_a, mean_b, c, px[k], pg[k], dx,
                                           out + (size_t)(r + k * s.rows) * s.channels);
    }
    for (; r < p.end; r += s.rows)
        input_gradient_vector<D, V, V>(s, d, seed, m, mean_a, mean_b, c, load_packed<D, V>(x, base + (size_t)r * s.x_pixel),
                                       load_packed<D, V>(dy, gbase + (size_t)r * s.g_pixel), dx, out + (size_t)r * s.channels);
}

// ---- host side -------------------------------------------------------------------------------------------------------

// Elements of a vector: the largest power of two up to 16 bytes that divides the channels, every stride and every pointer.
// `divisible` and `pointers` are the bitwise or of these: a power of two divides all of them iff it divides that.
inline int vector_width(size_t bytes, uint64_t divisible, uintptr_t pointers) {
    int v = (int)(16 / bytes);
    while (v > 1 && (divisible % v != 0 || pointers % (v * bytes) != 0)) v /= 2;
    return v;
}

inline Shape base_shape(const inpc_group_norm_config& cfg) {
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
    return s;
}

// Bytes of one group of one image up to which the single form runs.
constexpr uint64_t kSingleBytes = 128 * 1024;

inline bool runs_single(const inpc_group_norm_config& cfg, int v) {
    const uint64_t bytes = (uint64_t)cfg.n_pixels * (cfg.channels / cfg.groups) * element_bytes(cfg.dtype);
    return bytes <= kSingleBytes || cfg.channels / (uint32_t)v > (uint32_t)kThreads || cfg.groups > (uint32_t)kThreads;
}

// Threads of a block of the single form: as many as the group has vectors, in whole waves.
inline Shape single_shape(const inpc_group_norm_config& cfg, int v, int most, uint32_t& threads) {
    Shape s = base_shape(cfg);
    const uint64_t vectors = (uint64_t)s.per_group / (uint32_t)v, all = vectors * s.pixels;
    threads = 64;
    while (threads < (uint32_t)most && threads < all) threads *= 2;
    s.columns = (uint32_t)std::min<uint64_t>(vectors, threads);
    s.rows = threads / s.columns;
    return s;
}

inline Shape split_shape(const inpc_group_norm_config& cfg, int v) {
    Shape s = base_shape(cfg);
    s.columns = cfg.channels / (uint32_t)v;
    s.rows = kThreads / s.columns;
    const uint64_t per_image = std::max<uint64_t>(1, kFillBlocks / s.n), step = (uint64_t)s.rows * kUnroll;
    const uint64_t wanted = (s.pixels + per_image - 1) / per_image;
    s.slab_pixels = (uint32_t)((wanted + step - 1) / step * step);
    s.slabs = div_up(s.pixels, s.slab_pixels);
    return s;
}

// What a call may need, whatever its alignment: [sums per (image, channel)] or [sums per (image, slab, group)] [sums per
// (image, slab, channel)] [means per (image, group)]
struct Workspace {
    size_t of_groups, of_channels, means, bytes;
};
inline Workspace split_workspace(const Shape& s, bool backward) {
    Workspace w;
    const size_t slabs = (size_t)s.n * s.slabs;
    w.of_groups = 0;
    w.of_channels = align_up(slabs * s.groups * sizeof(float2), 256);
    w.means = w.of_channels + (backward ? align_up(slabs * s.channels * sizeof(float2), 256) : 0);
    w.bytes = w.means + (backward ? align_up((size_t)s.n * s.groups * sizeof(float2), 256) : 0);
    return w;
}
inline size_t workspace_bytes(const inpc_group_norm_config& cfg, bool backward) {
    size_t most = backward && cfg.n_images > 1 ? (size_t)cfg.n_images * cfg.channels * sizeof(float2) : 0;
    for (int v = (int)(16 / element_bytes(cfg.dtype)); v >= 1; v /= 2)
        if (cfg.channels % (uint32_t)v == 0 && !runs_single(cfg, v))
            most = std::max(most, split_workspace(split_shape(cfg, v), backward).bytes);
    return most;
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
    // blocks are counted in 31 bits
    if ((uint64_t)cfg->n_images * cfg->groups > 0x7FFFFFFFu || (uint64_t)cfg->n_images + kFillBlocks > 0x7FFFFFFFu)
        return fail(INPC_E_UNSUPPORTED, "%s: too many images", what);
    if (!(cfg->eps >= 0.0f)) return fail(INPC_E_INVALID_ARGUMENT, "%s: eps must not be negative", what);
    if (!valid_probability(cfg->dropout_p)) return fail(INPC_E_INVALID_ARGUMENT, "%s: the dropout probability is outside [0, 1]", what);
    return INPC_OK;
}

inline int check_workspace(const inpc_group_norm_config& cfg, bool backward, const void* workspace, size_t bytes, const char* what) {
    const size_t needed = workspace_bytes(cfg, backward);
    if (needed != 0 && (!workspace || bytes < needed || (uintptr_t)workspace % 16 != 0))
        return fail(INPC_E_WORKSPACE, "%s: the workspace holds %zu bytes, %zu are needed, 16-byte aligned", what, bytes, needed);
    return INPC_OK;
}

#define INPC_NORM_LAUNCH_LDS(name, kernel, grid, block, lds_bytes, stream, ...)                                 \
    do {                                                                                                        \
        ::inpc::timing_begin(name, stream);                                                                     \
        hipLaunchKernelGGL((kernel), grid, block, lds_bytes, stream, __VA_ARGS__);                              \
        ::inpc::timing_end(stream);                                                                             \
        hipError_t _e = hipGetLastError();                                                                      \
        if (_e != hipSuccess)                                                                                   \
            return ::inpc::fail(INPC_E_HIP, "launch of %s failed: %s", name, hipGetErrorString(_e));            \
    } while (0)

template <int D, int V>
int forward_single(const inpc_group_norm_config& cfg, const void* x, const void* weight, const void* bias, void* y, float2* moments,
                   hipStream_t stream) {
    uint32_t threads = 0;
    const Shape s = single_shape(cfg, V, kMaxThreads, threads);
    const Dropout d = make_dropout(cfg.dropout_p, cfg.seed, cfg.seed_dev, cfg.offset);
    INPC_LAUNCH("group_norm_single", (k_single<D, V>), dim3(s.n * s.groups), dim3(threads), stream, x, weight, bias, y, moments, s, d);
    return INPC_OK;
}

template <int D, int V>
int backward_single(const inpc_group_norm_config& cfg, const void* x, const void* dy, const float2* moments, const void* weight,
                    const void* bias, void* dx, void* dweight, void* dbias, char* ws, hipStream_t stream) {
    uint32_t threads = 0;
    const Shape s = single_shape(cfg, V, kMaxThreadsBackward, threads);
    const Dropout d = make_dropout(cfg.dropout_p, cfg.seed, cfg.seed_dev, cfg.offset);
    const bool later = s.n > 1 && (dweight || dbias);
    float2* sums = later ? (float2*)ws : nullptr;
    INPC_NORM_LAUNCH_LDS("group_norm_single_backward", (k_single_backward<D, V>), dim3(s.n * s.groups), dim3(threads),
                         (size_t)(threads + 32) * 2 * V * sizeof(float), stream, x, dy, moments, weight, bias, dx,
                         later ? (void*)nullptr : dweight, later ? (void*)nullptr : dbias, sums, s, d);
    if (later)
        INPC_LAUNCH("group_norm_parameter_gradients", k_parameter_gradients, dim3(div_up(s.channels, kParameterColumns)),
                    dim3(kThreads), stream, sums, dweight, dbias, s);
    return INPC_OK;
}

template <int D, int V>
int forward_split(const inpc_group_norm_config& cfg, const void* x, const void* weight, const void* bias, void* y, float2* moments,
                  char* ws, hipStream_t stream) {
    const Shape s = split_shape(cfg, V);
    const Dropout d = make_dropout(cfg.dropout_p, cfg.seed, cfg.seed_dev, cfg.offset);
    const bool fold = (uint64_t)s.slabs * s.groups <= kFoldedSums;
    float2* partial = (float2*)(ws + split_workspace(s, false).of_groups);
    INPC_NORM_LAUNCH_LDS("group_norm_moments", (k_moments<D, V>), dim3(s.n * s.slabs), dim3(kThreads),
                         ((size_t)(kThreads + 32) * V + 2 * s.groups) * sizeof(float), stream, x, partial, s);
    if (!fold)
        INPC_LAUNCH("group_norm_combine_moments", k_combine_moments, dim3(div_up(s.n * s.groups, kThreads / 64)), dim3(kThreads),
                    stream, partial, moments, s);
    INPC_LAUNCH("group_norm_apply", (k_apply<D, V>), dim3(s.n * s.slabs), dim3(kThreads), stream, x,
                fold ? (const float2*)partial : (const float2*)nullptr, weight, bias, y, moments, s, d);
    return INPC_OK;
}

template <int D, int V>
int backward_split(const inpc_group_norm_config& cfg, const void* x, const void* dy, const float2* moments, const void* weight,
                   const void* bias, void* dx, void* dweight, void* dbias, char* ws, hipStream_t stream) {
    const Shape s = split_shape(cfg, V);
    const Dropout d = make_dropout(cfg.dropout_p, cfg.seed, cfg.seed_dev, cfg.offset);
    const Workspace w = split_workspace(s, true);
    const bool fold = (uint64_t)s.slabs * s.groups <= kFoldedSums;
    float2 *of_groups = (float2*)(ws + w.of_groups), *of_channels = (float2*)(ws + w.of_channels), *means = (float2*)(ws + w.means);
    INPC_NORM_LAUNCH_LDS("group_norm_gradient_sums", (k_gradient_sums<D, V>), dim3(s.n * s.slabs), dim3(kThreads),
                         ((size_t)(kThreads + 32) * 2 * V + 2 * s.groups) * sizeof(float), stream, x, dy, moments, weight, bias,
                         of_channels, of_groups, s, d);
    if (dx && !fold)
        INPC_LAUNCH("group_norm_combine_gradients", k_combine_gradients, dim3(div_up(s.n * s.groups, kThreads / 64)), dim3(kThreads),
                    stream, of_groups, means, s);
    const uint32_t parameter_blocks = dweight || dbias ? div_up(s.channels, kParameterColumns) : 0;
    INPC_LAUNCH("group_norm_input_gradient", (k_input_gradient<D, V>), dim3(parameter_blocks + (dx ? s.n * s.slabs : 0)),
                dim3(kThreads), stream, x, dy, moments, of_channels, of_groups, fold ? (const float2*)nullptr : (const float2*)means,
                weight, bias, dx, dweight, dbias, parameter_blocks, s, d);
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

inline int forward(const inpc_group_norm_config& cfg, const void* x, const void* weight, const void* bias, void* y, float2* moments,
                   char* ws, hipStream_t stream) {
    const size_t bytes = element_bytes(cfg.dtype);
    const uint64_t divisible = cfg.channels | cfg.input_image_stride | cfg.input_pixel_stride;
    const uintptr_t pointers = (uintptr_t)x | (uintptr_t)y;
    const int v = vector_width(bytes, divisible, pointers);
    if (!runs_single(cfg, v)) return INPC_NORM_DISPATCH(forward_split, cfg.dtype, v, cfg, x, weight, bias, y, moments, ws, stream);
    const int in_group = vector_width(bytes, divisible | cfg.channels / cfg.groups, pointers);
    return INPC_NORM_DISPATCH(forward_single, cfg.dtype, in_group, cfg, x, weight, bias, y, moments, stream);
}

inline int backward(const inpc_group_norm_config& cfg, const void* x, const void* dy, const float2* moments, const void* weight,
                    const void* bias, void* dx, void* dweight, void* dbias, char* ws, hipStream_t stream) {
    const size_t bytes = element_bytes(cfg.dtype);
    const uint64_t divisible = cfg.channels | cfg.input_image_stride | cfg.input_pixel_stride | cfg.grad_image_stride | cfg.grad_pixel_stride;
    const uintptr_t pointers = (uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx;
    const int v = vector_width(bytes, divisible, pointers);
    if (!runs_single(cfg, v))
        return INPC_NORM_DISPATCH(backward_split, cfg.dtype, v, cfg, x, dy, moments, weight, bias, dx, dweight, dbias, ws, stream);
    const int in_group = vector_width(bytes, divisible | cfg.channels / cfg.groups, pointers);
    return INPC_NORM_DISPATCH(backward_single, cfg.dtype, in_group, cfg, x, dy, moments, weight, bias, dx, dweight, dbias, ws, stream);
}

}  // namespace norm
}  // namespace inpc
