// groupnorm.hpp — group norm with an activation and optional dropout over channels-last feature maps, forward and backward.
//
//   xhat = (x - mean) / sqrt(var + eps)   mean, var (biased) over the pixels of one image and the channels of one group
//   z = xhat * weight + bias,  y = activation(z),  then dropout (elements.hpp)
//   backward: dz = dy * activation'(z);  dbias = sum dz, dweight = sum dz * xhat over images and pixels;
//   dx = (weight * dz - A - xhat * B) / sqrt(var + eps), A and B the group's means of weight * dz and weight * dz * xhat
//
// Two forms. "single": a block per (image, group) does everything in one launch, for small maps, whose launches and latencies
// cost more than their bytes. "split": a block per run of pixels (a slab) of an image and tile of its channels, as wide as a block can
// be, so that it reads whole runs of memory; one launch writes each slab's sums, the next adds them up at the start of every block (or a
// launch in between does) and applies. In both a thread keeps one vector of channels (16 bytes where channel counts, strides
// and pointers allow). Sums are fp32 in an order that depends on sizes and alignments alone (no atomics); deviations are
// taken from a value of the data, so that nothing cancels however far the values are from 0.
//
// What bounds it: memory. Forward reads x twice and writes y, backward reads x and dy twice and writes dx; up to some 200 MB
// the second read comes from the 256 MB memory-side cache. 1240x824x32 fp16 (65 MB), SiLU: moments 15 us (4.3 TB/s), apply
// 27 us (4.8 TB/s read and written), gradient sums 29 us (4.5 TB/s), input gradient 37 us (5.3 TB/s); without the activation the
// gradient sums take 26 us. A plain copy of that size reaches 5.9 TB/s from the cache and 4.9 TB/s from memory.
#pragma once

#include <algorithm>
#include <utility>

#include "elements.hpp"

namespace inpc {
namespace norm {

constexpr int kMaxThreads = 512;         // of the single form
constexpr int kThreads = 512;            // of the split form
// Vectors a thread has in flight, forward, and of x and of dy each, backward. Twice as many in the backward pass cost a wave of
// occupancy: gradient sums of 65 MB of fp16 31 -> 40 us; half as many change nothing.
constexpr int kUnroll = 4;
constexpr int kUnrollBackward = 2;
// Blocks of a launch that sums: two on each compute unit. With 1024 the blocks' own reductions weigh more (gradient sums of
// 65 MB 31 -> 37 us); with 256 nothing is gained there (31 us) and an input gradient of as many blocks takes 35 us instead of 32.
constexpr uint32_t kSumBlocks = 512;
// Maps of up to 48 MB take half as many, which leaves fewer sums to add up: moments of 33 MB 13.4 -> 11.2 us, of 16 MB 6.7 -> 6.9.
constexpr uint32_t kSmallSumBlocks = 256;
constexpr uint64_t kSmallMap = 48ull << 20;
// Where the sums of a tile of an image are at most this many, every applying block adds them up itself; beyond a launch in
// between does: for 17 to 32 groups in one tile of one image of more than 48 MB, and for maps of gigabytes (kLongestRun). 65 MB, 8 groups (4000 sums): apply 27 us against 23 us + 4.4 us; 33 MB, 32 groups (8000 sums): 20 us against
// 16 us + 4.5 us, and a launch less for the host; the same with 16000 sums: 26 us against 16 us + 4.5 us.
constexpr uint32_t kFoldedSums = 8192;
// Blocks of a launch that applies and does not add up. 65 MB: 22.7 us with 1024, 23.4 with 2048, 27.9 with 4096.
constexpr uint32_t kApplyBlocks = 1024;
// Vectors of a thread at most: a longer chain of fp32 additions costs digits (five images of 4100x4100x64 bf16 with 2575 each: the
// parameters' gradients of equal values were off by 280 u). Larger maps, of more than 2 GB, take two, three, ... times the blocks: whole rounds of
// them cost nothing (2.3 to 2.7 GB forward and backward 3.7 to 4.3 ms either way), a fourth more blocks cost a tenth.
constexpr uint32_t kLongestRun = 512;
constexpr uint32_t kTileGroups = 32;     // groups of a tile of channels at most: a block's threads share them out at once
constexpr uint32_t kParameterColumns = 32;

struct Shape {
    uint64_t x_image, x_pixel;   // strides of x in elements (channels are adjacent); y and dx are dense
    uint64_t g_image, g_pixel;   // of the gradient of y
    uint32_t n, pixels, channels, groups, per_group;
    uint32_t columns, rows;      // threads of a block: vectors side by side, pixels at once
    uint32_t tiles, tile_groups; // split form: tiles of channels, and whole groups in each (fewer in the last)
    uint32_t parts;              // ... or, where a group is too wide for a block, this many tiles to each group (tile_groups is 1)
    uint32_t tile_channels;      // ... channels of a tile (fewer in the last)
    uint32_t slabs, slab_pixels; // ... and runs of pixels of each tile of an image
    int32_t activation, param_dtype;
    float eps;
    bool streamed;               // split form: the result is stored past the caches
};

// f(0), ..., f(N - 1) written out with constant arguments: an array indexed by them stays in registers, which a loop that the
// compiler only unrolls late does not guarantee.
template <typename F, int... K>
__device__ __forceinline__ void written_out(F& f, std::integer_sequence<int, K...>) {
    (f(std::integral_constant<int, K>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void written_out(F f) {
    written_out(f, std::make_integer_sequence<int, N>{});
}

// ---- sums over a block -----------------------------------------------------------------------------------------------
// Sum over `lanes` neighbouring lanes (a power of two), in all of them
__device__ __forceinline__ float lanes_sum(float v, uint32_t lanes) {
    for (uint32_t o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, (int)o, 64);
    return v;
}

// The sum of all threads' values, in every thread. `lds`: one float per wave; free again when the next barrier has passed.
__device__ __forceinline__ float block_sum(float v, float* lds) {
    v = lanes_sum(v, 64);
    const uint32_t waves = blockDim.x / 64u;
    __syncthreads();
    if (lane_id() == 0) lds[threadIdx.x / 64u] = v;
    __syncthreads();
    float total = 0.0f;
    for (uint32_t w = 0; w < waves; ++w) total += lds[w];
    return total;
}

// The largest power of two of lanes, up to a wave, that `parts` parts of a block can have each
__device__ __forceinline__ uint32_t lanes_for(uint32_t parts) {
    uint32_t lanes = 64;
    while (lanes > 1 && lanes * parts > blockDim.x) lanes >>= 1;
    return lanes;
}

// Adds V values per thread over the threads of a column (thread = row * columns + column). Returns where the totals lie in LDS,
// [column][V], for every thread to read until the next barrier after the next call. `lds` holds column_floats<V>(blockDim.x).
template <int V>
constexpr size_t column_floats(size_t threads) { return threads * (V + 1) + threads * V / 2; }

template <int V>
__device__ __forceinline__ float* column_sums(const float (&v)[V], uint32_t columns, uint32_t rows, float* lds) {
    const uint32_t width = columns * V, stride = width + 1, row = threadIdx.x / columns;   // an odd stride: no bank twice
    __syncthreads();
    if (row < rows)
#pragma unroll
        for (int j = 0; j < V; ++j) lds[row * stride + threadIdx.x % columns * V + j] = v[j];
    __syncthreads();
    if (rows == 1) return lds;
    float* total = lds + blockDim.x * (V + 1);
    const uint32_t lanes = lanes_for(width), lane = threadIdx.x % lanes;
    for (uint32_t base = 0; base < width; base += blockDim.x / lanes) {
        const uint32_t channel = base + threadIdx.x / lanes;
        float sum = 0.0f;
        if (channel < width)
            for (uint32_t r = lane; r < rows; r += lanes) sum += lds[r * stride + channel];
        sum = lanes_sum(sum, lanes);
        if (lane == 0 && channel < width) total[channel] = sum;
    }
    __syncthreads();
    return total;
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
// A vector's V channels are Q slots of channels that share a group: 1 where the vector lies in one group, 2 where it lies in
// two of half a vector each, else V. z = (x - mean) * scale + bias, scale = weight / sqrt(var + eps).
template <int V, int Q>
struct Affine {
    float mean[Q], rstd[Q], scale[V], bias[V];
};

// `moments`: of the group of channel `first`, the vector's first channel being `channel`
template <int V, int Q>
__device__ __forceinline__ Affine<V, Q> load_affine(const Shape& s, const float2* moments, uint32_t first, uint32_t channel,
                                                    const void* weight, const void* bias) {
    Affine<V, Q> a;
    load_elements<V>(weight, s.param_dtype, channel, 1.0f, a.scale);
    load_elements<V>(bias, s.param_dtype, channel, 0.0f, a.bias);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const float2 m = moments[(channel - first + q * (V / Q)) / s.per_group];
        a.mean[q] = m.x;
        a.rstd[q] = m.y;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) a.scale[j] *= a.rstd[j / (V / Q)];
    return a;
}

// A thread's vectors in one run of pixels of a feature map, `rows` pixels apart: vector k at base + k * step + lane. All but
// `lane` is the same for the whole block, so that an address costs scalar arithmetic and one register per thread.
struct Rows {
    char* base;
    uint64_t step;   // bytes
    uint32_t lane;   // bytes
    bool streamed;   // stores go past the caches
};
// `first`: the element that the run's first pixel and the block's first channel make
template <int D, int V>
__device__ __forceinline__ Rows rows_of(const void* map, uint64_t first, uint64_t pixel_stride, const Shape& s) {
    return Rows{(char*)map + first * kElementBytes<D>, s.rows * pixel_stride * kElementBytes<D>,
                (uint32_t)((threadIdx.x / s.columns * (uint32_t)pixel_stride + threadIdx.x % s.columns * V) * kElementBytes<D>), false};
}
template <int D, int V>
__device__ __forceinline__ PackedVector<D, V> load_row(const Rows& m, uint32_t k, uint32_t skip = 0) {
    return *(const PackedVector<D, V>*)(m.base + k * m.step + (m.lane + skip * kElementBytes<D>));
}

template <int D, int V>
__device__ __forceinline__ void store_row(const Rows& m, uint32_t k, uint32_t skip, const float (&v)[V]) {
    auto* to = (PackedVector<D, V>*)(m.base + k * m.step + (m.lane + skip * kElementBytes<D>));
    if (m.streamed) store_streamed(to, pack<D, V>(v));
    else *to = pack<D, V>(v);
}

// The same for element numbers: of the result, which is dense
struct Numbers {
    uint64_t first;
    uint32_t step, lane;
};
template <int V>
__device__ __forceinline__ Numbers numbers_of(uint64_t first, const Shape& s) {
    return Numbers{first, s.rows * s.channels, threadIdx.x / s.columns * s.channels + threadIdx.x % s.columns * V};
}
__device__ __forceinline__ uint64_t number_of(const Numbers& n, uint32_t k, uint32_t skip = 0) {
    return n.first + (uint64_t)k * n.step + (n.lane + skip);
}

template <int D, int V, int Q>
__device__ __forceinline__ void apply_vector(const Shape& s, const Dropout& d, uint64_t seed, const Affine<V, Q>& a,
                                             const PackedVector<D, V>& packed, const Rows& y, const Numbers& numbers,
                                             uint32_t k, uint32_t skip = 0) {
    float v[V];
    unpack<D, V>(packed, v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = fmaf(v[j] - a.mean[j / (V / Q)], a.scale[j], a.bias[j]);
    activate<V>(s.activation, v);
    if (d.on) dropout_apply<V>(d, seed, number_of(numbers, k, skip), v);
    store_row<D, V>(y, k, skip, v);
}

// x - mean in v and dz in g
template <int D, int V, int Q>
__device__ __forceinline__ void gradient_vector(const Shape& s, const Dropout& d, uint64_t seed, const Affine<V, Q>& a,
                                                const PackedVector<D, V>& px, const PackedVector<D, V>& pg, uint64_t number,
                                                float (&v)[V], float (&g)[V]) {
    float z[V];
    unpack<D, V>(px, v);
    unpack<D, V>(pg, g);
    if (d.on) dropout_apply<V>(d, seed, number, g);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        v[j] -= a.mean[j / (V / Q)];
        z[j] = fmaf(v[j], a.scale[j], a.bias[j]);
    }
    activate_backward<V>(s.activation, z, g);
}

// dx = dz * scale - k1 - (x - mean) * k2, k1 = A / sqrt(var + eps), k2 = B / (var + eps)
template <int D, int V, int Q>
__device__ __forceinline__ void input_gradient_vector(const Shape& s, const Dropout& d, uint64_t seed, const Affine<V, Q>& a,
                                                      const float (&k1)[Q], const float (&k2)[Q], const PackedVector<D, V>& px,
                                                      const PackedVector<D, V>& pg, const Rows& dx, const Numbers& numbers,
                                                      uint32_t k, uint32_t skip = 0) {
    float v[V], g[V];
    gradient_vector<D, V, Q>(s, d, seed, a, px, pg, number_of(numbers, k, skip), v, g);
#pragma unroll
    for (int j = 0; j < V; ++j) g[j] = fmaf(-v[j], k2[j / (V / Q)], fmaf(g[j], a.scale[j], -k1[j / (V / Q)]));
    store_row<D, V>(dx, k, skip, g);
}

// The same rows `skip` elements further
template <int D>
__device__ __forceinline__ Rows shifted(Rows m, uint32_t skip) {
    m.lane += skip * kElementBytes<D>;
    return m;
}

// f(k, vector k of the map, or of both) for all vectors that a thread has in a run of `size` pixels: N at a time, loaded before
// the first is used. `k` is the same for the whole block.
template <int D, int V, int N, typename F>
__device__ __forceinline__ void stream(const Rows& x, uint32_t rows, uint32_t size, uint32_t row, F f) {
    if (row >= size) return;
    const uint32_t whole = size / rows, rest = size % rows;
    uint32_t k = 0;
    for (; k + N <= whole; k += N) {
        PackedVector<D, V> packed[N];
        written_out<N>([&](auto i) { packed[i] = load_row<D, V>(x, k + i); });
        written_out<N>([&](auto i) { f(k + i, packed[i]); });
    }
    for (; k < whole; ++k) f(k, load_row<D, V>(x, k));
    if (row < rest) f(whole, load_row<D, V>(x, whole));
}
template <int D, int V, int N, typename F>
__device__ __forceinline__ void stream(const Rows& x, const Rows& g, uint32_t rows, uint32_t size, uint32_t row, F f) {
    if (row >= size) return;
    const uint32_t whole = size / rows, rest = size % rows;
    uint32_t k = 0;
    for (; k + N <= whole; k += N) {
        PackedVector<D, V> px[N], pg[N];
        written_out<N>([&](auto i) {
            px[i] = load_row<D, V>(x, k + i);
            pg[i] = load_row<D, V>(g, k + i);
        });
        written_out<N>([&](auto i) { f(k + i, px[i], pg[i]); });
    }
    for (; k < whole; ++k) f(k, load_row<D, V>(x, k), load_row<D, V>(g, k));
    if (row < rest) f(whole, load_row<D, V>(x, whole), load_row<D, V>(g, whole));
}

// A thread's mean and sum of squared deviations, for each slot of its vectors. Batches of kBatch vectors are summed as differences from
// the batch's first value, then joined to the batches before them (Chan, Golub, LeVeque, "Updating formulae and a pairwise algorithm
// for computing sample variances", 1979), whose mean is kept as a difference from the thread's first value, so that nothing cancels
// far from 0. What cancels in s2 - s1^2 / m within a batch of m <= 4 * 8 values costs at most a factor of m in the last place relative
// to the group's sum of squares, which is at least the pivot's squared distance from the mean; that is reached where one value in
// front makes up the whole variance. One pivot for all of a thread's values is no faster (moments of 65 MB of fp16 14.8 us either way),
// and the rounding of its sums grows with the square of their number: with such a value and 4096 vectors per thread (64x64x2056 fp32 in one
// block) the result's standard deviation was 0.57.
constexpr uint32_t kBatch = 4;

template <int V, int Q>
struct Differences {
    float n, origin[Q], mean[Q], dev[Q];   // of the batches that are joined: values, first value, mean - origin, squared deviations
    float open, pivot[Q], s1[Q], s2[Q];    // of the last batch: values, first value, sums of differences and of their squares
    __device__ __forceinline__ Differences() {
        n = open = 0.0f;
#pragma unroll
        for (int q = 0; q < Q; ++q) origin[q] = mean[q] = dev[q] = pivot[q] = s1[q] = s2[q] = 0.0f;
    }
    // `k`: the vector's number in a run of the thread's, the same for the whole block
    __device__ __forceinline__ void add(const float (&v)[V], uint32_t k) {
        constexpr int W = V / Q;   // channels of a slot
        if (k % kBatch == 0) {
            join();
            const bool first = n == 0.0f;
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                pivot[q] = v[q * W];
                origin[q] = first ? pivot[q] : origin[q];
            }
        }
        open += (float)W;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            float a[2] = {0.0f, 0.0f}, b[2] = {0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const float d = v[q * W + j] - pivot[q];
                a[j & 1] += d;
                b[j & 1] = fmaf(d, d, b[j & 1]);
            }
            s1[q] += a[0] + a[1];
            s2[q] += b[0] + b[1];
        }
    }
    // Once more behind the last vector
    __device__ __forceinline__ void join() {
        if (open == 0.0f) return;
        const float all = n + open, share = __builtin_amdgcn_rcpf(open), r = open * __builtin_amdgcn_rcpf(all), weight = n * r;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const float own = s1[q] * share, rest = fmaf(-s1[q], own, s2[q]), d = (pivot[q] - origin[q]) + own - mean[q];
            dev[q] += fmaf(weight * d, d, rest < 0.0f ? 0.0f : rest);   // a NaN stays one
            mean[q] = fmaf(d, r, mean[q]);
            s1[q] = s2[q] = 0.0f;
        }
        n = all;
        open = 0.0f;
    }
    // the values' sum, and the sum of their squared deviations from `of_group`
    __device__ __forceinline__ float sum(int q) const { return fmaf(n, origin[q], n * mean[q]); }
    __device__ __forceinline__ float deviations(int q, float of_group) const {
        const float d = (origin[q] - of_group) + mean[q];
        return fmaf(n * d, d, dev[q]);
    }
};

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
    const uint32_t column = threadIdx.x % s.columns, vectors = s.per_group / V;
    const uint32_t row = threadIdx.x / s.columns < s.rows ? threadIdx.x / s.columns : 0xFFFFFFFFu;
    const uint64_t out = (uint64_t)image * s.pixels * s.channels + first;
    const Rows rx = rows_of<D, V>(x, image * s.x_image + first, s.x_pixel, s), ry = rows_of<D, V>(y, out, s.channels, s);
    Differences<V, 1> sums;
    for (uint32_t c = column; c < vectors; c += s.columns)
        stream<D, V, kUnroll>(shifted<D>(rx, (c - column) * V), s.rows, s.pixels, row, [&](uint32_t k, const PackedVector<D, V>& packed) {
            float v[V];
            unpack<D, V>(packed, v);
            sums.add(v, k);
        });
    sums.join();
    const float all = (float)s.pixels * (float)s.per_group;
    const float mean = block_sum(sums.sum(0), lds) / all;
    const float2 m = make_float2(mean, 1.0f / sqrtf(block_sum(sums.deviations(0, mean), lds) / all + s.eps));
    if (threadIdx.x == 0) moments[b] = m;
    const uint64_t seed = dropout_seed(d);
    const Numbers numbers = numbers_of<V>(out, s);
    for (uint32_t c = column; c < vectors; c += s.columns) {
        const uint32_t skip = (c - column) * V;
        const Affine<V, 1> a = load_affine<V, 1>(s, &m, first + c * V, first + c * V, weight, bias);
        stream<D, V, kUnroll>(shifted<D>(rx, skip), s.rows, s.pixels, row, [&](uint32_t k, const PackedVector<D, V>& packed) {
            apply_vector<D, V, 1>(s, d, seed, a, packed, ry, numbers, k, skip);
        });
    }
}

// With one image dbias and dweight come from here, with more the sums of every (image, channel) do.
template <int D, int V>
__global__ void __launch_bounds__(kMaxThreads) k_single_backward(const void* __restrict__ x, const void* __restrict__ dy,
                                                                 const float2* __restrict__ moments, const void* __restrict__ weight,
                                                                 const void* __restrict__ bias, void* __restrict__ dx,
                                                                 void* __restrict__ dweight, void* __restrict__ dbias,
                                                                 float2* __restrict__ sums, Shape s, Dropout d) {
    INPC_DYNAMIC_LDS(float, lds);   // column_sums
    __shared__ float waves[kMaxThreads / 64];
    const uint32_t b = swizzled_block(), image = b / s.groups, first = b % s.groups * s.per_group;
    const uint32_t column = threadIdx.x % s.columns, vectors = s.per_group / V;
    const uint32_t row = threadIdx.x / s.columns < s.rows ? threadIdx.x / s.columns : 0xFFFFFFFFu;
    const uint64_t out = (uint64_t)image * s.pixels * s.channels + first, seed = dropout_seed(d);
    const Rows rx = rows_of<D, V>(x, image * s.x_image + first, s.x_pixel, s), rg = rows_of<D, V>(dy, image * s.g_image + first, s.g_pixel, s);
    const Numbers numbers = numbers_of<V>(out, s);
    const float2 m = moments[b];
    float a = 0.0f, bb = 0.0f;
    for (uint32_t tile = 0; tile < vectors; tile += s.columns) {
        const uint32_t c = tile + column, skip = tile * V;
        float total[2 * V];
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) total[j] = 0.0f;
        if (c < vectors) {
            const Affine<V, 1> affine = load_affine<V, 1>(s, &m, first + c * V, first + c * V, weight, bias);
            stream<D, V, kUnrollBackward>(shifted<D>(rx, skip), shifted<D>(rg, skip), s.rows, s.pixels, row,
                                          [&](uint32_t k, const PackedVector<D, V>& px, const PackedVector<D, V>& pg) {
                                              float v[V], g[V];
                                              gradient_vector<D, V, 1>(s, d, seed, affine, px, pg, number_of(numbers, k, skip), v, g);
#pragma unroll
                                              for (int j = 0; j < V; ++j) {
                                                  total[j] += g[j];
                                                  total[V + j] = fmaf(g[j], v[j], total[V + j]);
                                              }
                                          });
        }
        const uint32_t channels = min(s.columns, vectors - tile) * V;
        const float* totals = column_sums<2 * V>(total, s.columns, s.rows, lds);
        for (uint32_t i = threadIdx.x; i < channels; i += blockDim.x) {
            const uint32_t channel = first + tile * V + i;
            const float* of_channel = totals + i / V * (2 * V) + i % V;
            const float2 sum = make_float2(of_channel[0], of_channel[V] * m.y);
            const float w = weight ? load_element(weight, s.param_dtype, channel) : 1.0f;
            a = fmaf(w, sum.x, a);
            bb = fmaf(w, sum.y, bb);
            if (sums) sums[(size_t)image * s.channels + channel] = sum;
            if (dbias) store_element(dbias, s.param_dtype, channel, sum.x);
            if (dweight) store_element(dweight, s.param_dtype, channel, sum.y);
        }
    }
    if (!dx) return;
    const float count = (float)s.pixels * (float)s.per_group;
    const float k1[1] = {block_sum(a, waves) / count * m.y}, k2[1] = {block_sum(bb, waves) / count * m.y * m.y};
    const Rows rdx = rows_of<D, V>(dx, out, s.channels, s);
    for (uint32_t c = column; c < vectors; c += s.columns) {
        const uint32_t skip = (c - column) * V;
        const Affine<V, 1> affine = load_affine<V, 1>(s, &m, first + c * V, first + c * V, weight, bias);
        stream<D, V, kUnrollBackward>(shifted<D>(rx, skip), shifted<D>(rg, skip), s.rows, s.pixels, row,
                                      [&](uint32_t k, const PackedVector<D, V>& px, const PackedVector<D, V>& pg) {
                                          input_gradient_vector<D, V, 1>(s, d, seed, affine, k1, k2, px, pg, rdx, numbers, k, skip);
                                      });
    }
}

// dbias and dweight from `rows` rows of channel sums, kParameterColumns channels to a block; `lds`: column_floats<2>
__device__ __forceinline__ void add_parameter_gradients(const float2* sums, uint32_t rows, void* dweight, void* dbias, const Shape& s,
                                                        uint32_t block, float* lds) {
    const uint32_t channel = block * kParameterColumns + threadIdx.x % kParameterColumns;
    float total[2] = {0.0f, 0.0f};
    if (channel < s.channels)
#pragma unroll 4
        for (uint32_t r = threadIdx.x / kParameterColumns; r < rows; r += kThreads / kParameterColumns) {
            const float2 v = sums[(size_t)r * s.channels + channel];
            total[0] += v.x;
            total[1] += v.y;
        }
    const float* all = column_sums<2>(total, kParameterColumns, kThreads / kParameterColumns, lds);
    if (threadIdx.x < kParameterColumns && channel < s.channels) {
        if (dbias) store_element(dbias, s.param_dtype, channel, all[2 * threadIdx.x]);
        if (dweight) store_element(dweight, s.param_dtype, channel, all[2 * threadIdx.x + 1]);
    }
}

__global__ void __launch_bounds__(kThreads) k_parameter_gradients(const float2* __restrict__ sums, uint32_t rows,
                                                                  void* __restrict__ dweight, void* __restrict__ dbias, Shape s) {
    __shared__ float lds[column_floats<2>(kThreads)];
    add_parameter_gradients(sums, rows, dweight, dbias, s, blockIdx.x, lds);
}

// ---- the split form --------------------------------------------------------------------------------------------------
// What a block works on: a slab of pixels and a tile of channels (whole groups, or a part of one) of one image
struct Place {
    uint32_t image, tile, part, channel, width;   // `channel`: the tile's first; `width`: its channels
    uint32_t group, groups, group_width;          // its first group, its groups, and the channels of each in the tile
    uint32_t slab, begin, size;
};

__device__ __forceinline__ Place place_of(const Shape& s, uint32_t block) {
    Place p;
    const uint32_t rest = block / s.slabs;
    p.tile = rest % s.tiles;
    p.image = rest / s.tiles;
    if (s.parts == 1) {
        p.part = 0;
        p.group = p.tile * s.tile_groups;
        p.groups = min(s.tile_groups, s.groups - p.group);
        p.group_width = s.per_group;
    } else {
        p.part = p.tile % s.parts;
        p.group = p.tile / s.parts;
        p.groups = 1;
        p.group_width = min(s.tile_channels, s.per_group - p.part * s.tile_channels);
    }
    p.channel = p.group * s.per_group + p.part * s.tile_channels;
    p.width = p.groups * p.group_width;
    p.slab = block % s.slabs;
    p.begin = p.slab * s.slab_pixels;
    p.size = min(s.slab_pixels, s.pixels - p.begin);
    return p;
}

// ... and its run of pixels in a map
template <int D, int V>
__device__ __forceinline__ Rows rows_at(const void* map, const Place& p, uint64_t image_stride, uint64_t pixel_stride, const Shape& s) {
    return rows_of<D, V>(map, p.image * image_stride + p.begin * pixel_stride + p.channel, pixel_stride, s);
}
template <int V>
__device__ __forceinline__ Numbers numbers_at(const Place& p, const Shape& s) {
    return numbers_of<V>(((uint64_t)p.image * s.pixels + p.begin) * s.channels + p.channel, s);
}

// Slab sums lie [image][tile][group of the tile][slab]: those of a group follow each other, also of one in parts
__device__ __forceinline__ size_t sums_at(const Shape& s, const Place& p, uint32_t group) {
    return ((size_t)(p.image * s.tiles + p.tile) * s.tile_groups + group) * s.slabs;
}

// The calling thread's row in its block; a row of no slab where it has none or its channels are behind the last
__device__ __forceinline__ uint32_t thread_row(const Shape& s, const Place& p, uint32_t vector) {
    const uint32_t row = threadIdx.x / s.columns;
    return row < s.rows && threadIdx.x % s.columns * vector < p.width ? row : 0xFFFFFFFFu;
}

// Sums over the slots of each group of a tile: values[row * width + slot], `per_group` neighbouring slots of all rows to a group.
// A power of two of lanes shares a group; at most kTileGroups groups: all at once.
__device__ __forceinline__ void group_sums(const float* values, uint32_t width, uint32_t rows, uint32_t per_group, uint32_t groups,
                                           float* sums) {
    const uint32_t lanes = lanes_for(groups), lane = threadIdx.x % lanes, group = threadIdx.x / lanes;
    float sum = 0.0f;
    if (group < groups) {
        const uint32_t count = rows * per_group;
        if (per_group == 1)
            for (uint32_t r = lane; r < count; r += lanes) sum += values[r * width + group];
        else
            for (uint32_t i = lane; i < count; i += lanes) sum += values[i / per_group * width + group * per_group + i % per_group];
    }
    sum = lanes_sum(sum, lanes);
    if (lane == 0 && group < groups) sums[group] = sum;
    __syncthreads();
}

// {mean, sum of squared deviations} of every (image, slab, group)
template <int D, int V, int Q>
__global__ void __launch_bounds__(kThreads) k_moments(const void* __restrict__ x, float2* __restrict__ partial, Shape s) {
    constexpr int W = V / Q;   // channels of a slot
    __shared__ float lds[kThreads * Q];
    __shared__ float group[kTileGroups], squares[kTileGroups];
    const Place p = place_of(s, blockIdx.x);
    const uint32_t row = thread_row(s, p, V);
    const Rows rows = rows_at<D, V>(x, p, s.x_image, s.x_pixel, s);
    Differences<V, Q> sums;
    stream<D, V, kUnroll>(rows, s.rows, p.size, row, [&](uint32_t k, const PackedVector<D, V>& packed) {
        float v[V];
        unpack<D, V>(packed, v);
        sums.add(v, k);
    });
    sums.join();
    // the group's mean, then everybody's deviations from it
    const uint32_t groups = p.groups, width = s.columns * Q, slots = p.group_width / W;
    const uint32_t slot = threadIdx.x % s.columns * Q, at = threadIdx.x / s.columns * width + slot;
    const bool in_block = threadIdx.x / s.columns < s.rows;
    const float in_group = (float)p.size * (float)p.group_width;
    if (in_block)
#pragma unroll
        for (int q = 0; q < Q; ++q) lds[at + q] = sums.sum(q);
    __syncthreads();
    group_sums(lds, width, s.rows, slots, groups, group);
    if (in_block)
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            // the slots of a last tile's missing groups, or of a last part's missing channels, are nobody's
            const float of_group = (slot + q) / slots < groups ? group[(slot + q) / slots] / in_group : 0.0f;
            lds[at + q] = sums.deviations(q, of_group);
        }
    __syncthreads();
    group_sums(lds, width, s.rows, slots, groups, squares);
    if (threadIdx.x < groups)
        partial[sums_at(s, p, threadIdx.x) + p.slab] = make_float2(group[threadIdx.x] / in_group, squares[threadIdx.x]);
}

// A group's moments from its slabs' (of all its parts), by a power of two of lanes, in all of them: a lane's slabs with the first
// one's mean as the pivot, then the lanes' deviations from the mean of all. `mine` is null for lanes of no group.
__device__ __forceinline__ float2 fold_moments(const float2* mine, const Shape& s, uint32_t lane, uint32_t lanes) {
    const float count = (float)s.pixels * (float)s.per_group, of_slab = (float)s.slab_pixels * (float)s.per_group;
    const uint32_t last_pixels = s.pixels - (s.slabs - 1) * s.slab_pixels, entries = s.parts * s.slabs;
    const float of_last = (float)last_pixels * (float)s.per_group;
    float n = 0.0f, pivot = 0.0f, s1 = 0.0f, s2 = 0.0f;
    const auto add = [&](const float2& v, float weight) {
        const float d = v.x - pivot;
        n += weight;
        s1 = fmaf(weight, d, s1);
        s2 += fmaf(weight * d, d, v.y);
    };
    if (mine && lane < entries) {
        pivot = mine[lane].x;
        if (s.parts == 1) {
#pragma unroll 8
            for (uint32_t slab = lane; slab < s.slabs; slab += lanes) add(mine[slab], slab + 1 < s.slabs ? of_slab : of_last);
        } else {
            for (uint32_t i = lane; i < entries; i += lanes) {
                const uint32_t part = i / s.slabs, slab = i % s.slabs;
                add(mine[i], (float)(slab + 1 < s.slabs ? s.slab_pixels : last_pixels) *
                                 (float)min(s.tile_channels, s.per_group - part * s.tile_channels));
            }
        }
    }
    const float share = n > 0.0f ? s1 / n : 0.0f;
    const float mean = lanes_sum(fmaf(n, pivot, s1), lanes) / count, d = pivot + share - mean;
    const float squares = lanes_sum(fmaf(n * d, d, fmaf(-s1, share, s2)), lanes);
    return make_float2(mean, 1.0f / sqrtf((squares < 0.0f ? 0.0f : squares) / count + s.eps));
}

// ... and the means A and B of the gradient pass
__device__ __forceinline__ float2 fold_gradients(const float2* mine, const Shape& s, uint32_t lane, uint32_t lanes) {
    float a = 0.0f, b = 0.0f;
    if (mine)
#pragma unroll 8
        for (uint32_t i = lane; i < s.parts * s.slabs; i += lanes) {
            a += mine[i].x;
            b += mine[i].y;
        }
    const float count = (float)s.pixels * (float)s.per_group;
    return make_float2(lanes_sum(a, lanes) / count, lanes_sum(b, lanes) / count);
}

// Of one tile of an image, into LDS: by every block of the launch that needs them where they are few ...
template <typename F>
__device__ __forceinline__ void fold_tile(const float2* partial, const Shape& s, const Place& p, float2* folded, F fold) {
    const uint32_t groups = p.groups, lanes = lanes_for(groups), lane = threadIdx.x % lanes, group = threadIdx.x / lanes;
    const float2* first = partial + sums_at(s, p, 0) - (size_t)p.part * s.slabs;
    const float2 m = fold(group < groups ? first + (size_t)group * s.slabs : nullptr, s, lane, lanes);
    if (lane == 0 && group < groups) folded[group] = m;
    __syncthreads();
}

// ... else in a launch of its own, a wave per (image, group)
__device__ __forceinline__ const float2* sums_of_wave(const float2* partial, const Shape& s, uint32_t item) {
    const uint32_t image = item / s.groups, group = item % s.groups;
    if (image >= s.n) return nullptr;
    return partial + ((size_t)(image * s.tiles + group / s.tile_groups * s.parts) * s.tile_groups + group % s.tile_groups) * s.slabs;
}

__global__ void __launch_bounds__(kThreads) k_combine_moments(const float2* __restrict__ partial, float2* __restrict__ moments, Shape s) {
    const uint32_t item = blockIdx.x * (kThreads / 64) + threadIdx.x / 64u;
    const float2* mine = sums_of_wave(partial, s, item);
    const float2 m = fold_moments(mine, s, lane_id(), 64);
    if (mine && lane_id() == 0) moments[item] = m;
}

// The first `parameter_blocks` blocks add up dweight and dbias.
__global__ void __launch_bounds__(kThreads) k_combine_gradients(const float2* __restrict__ of_groups, const float2* __restrict__ of_channels,
                                                                float2* __restrict__ means, void* __restrict__ dweight,
                                                                void* __restrict__ dbias, uint32_t parameter_blocks, Shape s) {
    __shared__ float lds[column_floats<2>(kThreads)];
    if (blockIdx.x < parameter_blocks) {
        add_parameter_gradients(of_channels, s.n * s.slabs, dweight, dbias, s, blockIdx.x, lds);
        return;
    }
    const uint32_t item = (blockIdx.x - parameter_blocks) * (kThreads / 64) + threadIdx.x / 64u;
    const float2* mine = sums_of_wave(of_groups, s, item);
    const float2 m = fold_gradients(mine, s, lane_id(), 64);
    if (mine && lane_id() == 0) means[item] = m;
}

// `partial` is null where k_combine_moments has run; else the first block of each tile of an image also writes its moments.
template <int D, int V, int Q>
__global__ void __launch_bounds__(kThreads) k_apply(const void* __restrict__ x, const float2* __restrict__ partial,
                                                    const void* __restrict__ weight, const void* __restrict__ bias,
                                                    void* __restrict__ y, float2* __restrict__ moments, Shape s, Shape of_sums, Dropout d) {
    __shared__ float2 folded[kTileGroups];
    const Place p = place_of(s, blockIdx.x);
    float2* of_tile = moments + (size_t)p.image * s.groups + p.group;
    const float2* m = of_tile;
    if (partial) {
        fold_tile(partial, of_sums, p, folded, fold_moments);
        if (p.slab == 0 && p.part == 0 && threadIdx.x < p.groups) of_tile[threadIdx.x] = folded[threadIdx.x];
        m = folded;
    }
    const uint32_t row = thread_row(s, p, V);
    if (row >= p.size) return;
    const Affine<V, Q> a = load_affine<V, Q>(s, m, p.channel, p.channel + threadIdx.x % s.columns * V, weight, bias);
    const uint64_t seed = dropout_seed(d);
    Rows ry = rows_at<D, V>(y, p, (uint64_t)s.pixels * s.channels, s.channels, s);
    ry.streamed = s.streamed;
    const Numbers numbers = numbers_at<V>(p, s);
    stream<D, V, kUnroll>(rows_at<D, V>(x, p, s.x_image, s.x_pixel, s), s.rows, p.size, row, [&](uint32_t k, const PackedVector<D, V>& packed) {
        apply_vector<D, V, Q>(s, d, seed, a, packed, ry, numbers, k);
    });
}

// {sum dz, sum dz * xhat} of every (image, slab, channel), and both weighted and summed of every (image, slab, group)
template <int D, int V, int Q>
__global__ void __launch_bounds__(kThreads) k_gradient_sums(const void* __restrict__ x, const void* __restrict__ dy,
                                                            const float2* __restrict__ all_moments, const void* __restrict__ weight,
                                                            const void* __restrict__ bias, float2* __restrict__ of_channels,
                                                            float2* __restrict__ of_groups, Shape s, Dropout d) {
    __shared__ float lds[column_floats<2 * V>(kThreads)];
    const Place p = place_of(s, blockIdx.x);
    const uint32_t row = thread_row(s, p, V);
    const float2* moments = all_moments + (size_t)p.image * s.groups;
    float total[2 * V];
#pragma unroll
    for (int j = 0; j < 2 * V; ++j) total[j] = 0.0f;
    if (row < p.size) {
        const Affine<V, Q> a = load_affine<V, Q>(s, moments, 0, p.channel + threadIdx.x % s.columns * V, weight, bias);
        const uint64_t seed = dropout_seed(d);
        const Numbers numbers = numbers_at<V>(p, s);
        stream<D, V, kUnrollBackward>(rows_at<D, V>(x, p, s.x_image, s.x_pixel, s), rows_at<D, V>(dy, p, s.g_image, s.g_pixel, s),
                                      s.rows, p.size, row, [&](uint32_t k, const PackedVector<D, V>& px, const PackedVector<D, V>& pg) {
                                          float v[V], g[V];
                                          gradient_vector<D, V, Q>(s, d, seed, a, px, pg, number_of(numbers, k), v, g);
#pragma unroll
                                          for (int j = 0; j < V; ++j) {
                                              total[j] += g[j];
                                              total[V + j] = fmaf(g[j], v[j], total[V + j]);
                                          }
                                      });
    }
    const uint32_t groups = p.groups, first = p.group, channels = p.width;
    float2* mine = of_channels + ((size_t)p.image * s.slabs + p.slab) * s.channels + p.channel;
    float* totals = column_sums<2 * V>(total, s.columns, s.rows, lds);
    // a channel's two sums, and weighted in place
    for (uint32_t i = threadIdx.x; i < channels; i += kThreads) {
        float* of_channel = totals + i / V * (2 * V) + i % V;
        const float2 sum = make_float2(of_channel[0], of_channel[V] * moments[first + i / s.per_group].y);
        const float w = weight ? load_element(weight, s.param_dtype, p.channel + i) : 1.0f;
        mine[i] = sum;
        of_channel[0] = sum.x * w;
        of_channel[V] = sum.y * w;
    }
    __syncthreads();
    const uint32_t lanes = lanes_for(groups), lane = threadIdx.x % lanes, group = threadIdx.x / lanes;
    float a = 0.0f, b = 0.0f;
    if (group < groups)
        for (uint32_t i = group * p.group_width + lane; i < (group + 1) * p.group_width; i += lanes) {
            const float* of_channel = totals + i / V * (2 * V) + i % V;
            a += of_channel[0];
            b += of_channel[V];
        }
    a = lanes_sum(a, lanes);
    b = lanes_sum(b, lanes);
    if (lane == 0 && group < groups) of_groups[sums_at(s, p, group) + p.slab] = make_float2(a, b);
}

// `means` is null where k_combine_gradients has not run: then the first `parameter_blocks` blocks add up dweight and dbias.
template <int D, int V, int Q>
__global__ void __launch_bounds__(kThreads) k_input_gradient(const void* __restrict__ x, const void* __restrict__ dy,
                                                             const float2* __restrict__ moments, const float2* __restrict__ of_channels,
                                                             const float2* __restrict__ of_groups, const float2* __restrict__ means,
                                                             const void* __restrict__ weight, const void* __restrict__ bias,
                                                             void* __restrict__ dx, void* __restrict__ dweight,
                                                             void* __restrict__ dbias, uint32_t parameter_blocks, Shape s, Shape of_sums, Dropout d) {
    __shared__ float lds[column_floats<2>(kThreads)];
    __shared__ float2 folded[kTileGroups];
    if (blockIdx.x < parameter_blocks) {
        add_parameter_gradients(of_channels, s.n * of_sums.slabs, dweight, dbias, s, blockIdx.x, lds);
        return;
    }
    const Place p = place_of(s, blockIdx.x - parameter_blocks);
    const float2* ab = means + (size_t)p.image * s.groups + p.group;
    if (!means) {
        fold_tile(of_groups, of_sums, p, folded, fold_gradients);
        ab = folded;
    }
    const uint32_t row = thread_row(s, p, V), channel = p.channel + threadIdx.x % s.columns * V;
    if (row >= p.size) return;
    const Affine<V, Q> a = load_affine<V, Q>(s, moments + (size_t)p.image * s.groups, 0, channel, weight, bias);
    float k1[Q], k2[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const float2 v = ab[(channel - p.channel + q * (V / Q)) / s.per_group];
        k1[q] = v.x * a.rstd[q];
        k2[q] = v.y * a.rstd[q] * a.rstd[q];
    }
    const uint64_t seed = dropout_seed(d);
    Rows rdx = rows_at<D, V>(dx, p, (uint64_t)s.pixels * s.channels, s.channels, s);
    rdx.streamed = s.streamed;
    const Numbers numbers = numbers_at<V>(p, s);
    stream<D, V, kUnrollBackward>(rows_at<D, V>(x, p, s.x_image, s.x_pixel, s), rows_at<D, V>(dy, p, s.g_image, s.g_pixel, s),
                                  s.rows, p.size, row, [&](uint32_t k, const PackedVector<D, V>& px, const PackedVector<D, V>& pg) {
                                      input_gradient_vector<D, V, Q>(s, d, seed, a, k1, k2, px, pg, rdx, numbers, k);
                                  });
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

// Bytes of one group of one image up to which the single form runs. Forward + backward, kernels alone: groups of 16 KB (39x26x256
// bf16, 8 images) single 9 + 16 us, split 14 + 24 us; of 64 KB (64x64x32 fp32) 13 + 21 against 12 + 17 us, with two launches less,
// so that a step as a whole takes 107 to 113 against 120 us; of 93 KB (77x101x30 bf16, 3 images) 19 + 30 against 10 + 12 us.
constexpr uint64_t kSingleBytes = 64 * 1024;

// Groups of a tile of the split form with vectors of v elements: as many as fit, with boundaries on vectors' boundaries; 0 where
// not even the fewest do (nor do they then with shorter vectors, which fill a block with as many fewer channels).
inline uint32_t tile_groups_of(const inpc_group_norm_config& cfg, int v) {
    const uint32_t per_group = cfg.channels / cfg.groups;
    uint32_t unit = 1;   // groups whose channels are whole vectors
    while ((uint64_t)unit * per_group % (uint32_t)v != 0) unit *= 2;
    const uint64_t fit = std::min<uint64_t>((uint64_t)kThreads * v / per_group, kTileGroups);
    return (uint32_t)std::min<uint64_t>(cfg.groups, fit / unit * unit);
}

// Tiles of each group where it is too wide for one; v divides its channels.
inline uint32_t parts_of(const inpc_group_norm_config& cfg, int v) { return div_up(cfg.channels / cfg.groups / (uint32_t)v, kThreads); }

// Blocks of a launch: fewer than 2^32 threads, with room for the blocks that add up the parameters' gradients
constexpr uint64_t kMostBlocks = 0xFFFFFFFFu / kThreads - INPC_GROUP_NORM_MAX_CHANNELS / kParameterColumns;

// A group that is too wide for a block (4096 values of 16 bits, 512 single elements) is cut into parts, so that neither a whole image's
// time nor its chains of additions are one block's: forward and backward of 200x200x515 fp16 in one group take 61 ms in the single form and
// 0.21 ms in parts, of 64 images of 16x16x515 350 and 146 us. The single form stays where parts would take more blocks than a launch
// has: such images have few pixels.
inline bool runs_single(const inpc_group_norm_config& cfg, int v) {
    const uint64_t bytes = (uint64_t)cfg.n_pixels * (cfg.channels / cfg.groups) * element_bytes(cfg.dtype);
    return bytes <= kSingleBytes || (tile_groups_of(cfg, v) == 0 && (uint64_t)cfg.n_images * cfg.groups * parts_of(cfg, v) > kMostBlocks);
}

// Threads of a block of the single form: as many as the group has vectors, in whole waves.
inline Shape single_shape(const inpc_group_norm_config& cfg, int v, uint32_t& threads) {
    Shape s = base_shape(cfg);
    const uint64_t vectors = (uint64_t)s.per_group / (uint32_t)v, all = vectors * s.pixels;
    threads = 64;
    while (threads < (uint32_t)kMaxThreads && threads < all) threads *= 2;
    s.columns = (uint32_t)std::min<uint64_t>(vectors, threads);
    s.rows = threads / s.columns;
    return s;
}

inline uint64_t map_bytes(const inpc_group_norm_config& cfg) {
    return (uint64_t)cfg.n_images * cfg.n_pixels * cfg.channels * element_bytes(cfg.dtype);
}

inline Shape split_shape(const inpc_group_norm_config& cfg, int v, uint32_t blocks) {
    Shape s = base_shape(cfg);
    s.tile_groups = tile_groups_of(cfg, v);
    s.parts = 1;
    if (s.tile_groups != 0) {
        s.tiles = div_up(s.groups, s.tile_groups);
        s.columns = s.tile_groups * s.per_group / (uint32_t)v;
    } else {
        s.tile_groups = 1;
        s.parts = parts_of(cfg, v);
        s.tiles = s.groups * s.parts;
        s.columns = div_up(s.per_group / (uint32_t)v, s.parts);
    }
    s.tile_channels = s.columns * (uint32_t)v;
    s.rows = kThreads / s.columns;
    const uint64_t runs = (uint64_t)s.n * s.tiles, longest = (uint64_t)s.rows * kLongestRun;
    uint64_t per_run = std::max<uint64_t>(1, blocks / runs);
    per_run *= (s.pixels + per_run * longest - 1) / (per_run * longest);   // whole rounds of blocks
    const uint64_t wanted = (s.pixels + per_run - 1) / per_run;
    const uint32_t step = s.rows * kUnroll;
    s.slab_pixels = (uint32_t)((wanted + step - 1) / step * step);
    s.slabs = div_up(s.pixels, s.slab_pixels);
    return s;
}

inline Shape sums_shape(const inpc_group_norm_config& cfg, int v) {
    return split_shape(cfg, v, map_bytes(cfg) <= kSmallMap ? kSmallSumBlocks : kSumBlocks);
}

// Where a call's maps together (x and y, or x, dy and dx) are larger than this, the result is stored past the caches: what it
// would push out of the 256 MB memory-side cache is the map that is read for the second time. Maps of 130 MB: forward 87 -> 73 us,
// backward 149 -> 128 us, also with an operator behind it that reads y (124 -> 121 us); of 65 MB and less nothing is gained, and
// that next operator finds less of y in the cache (62.4 -> 62.8 us).
constexpr uint64_t kStreamedBytes = 192ull << 20;

inline bool streams(const inpc_group_norm_config& cfg, int maps) {
    return map_bytes(cfg) * maps > kStreamedBytes;
}

inline bool folds(const Shape& s) { return (uint64_t)s.slabs * s.parts * s.tile_groups <= kFoldedSums; }

// Whether a call may run with vectors of v elements: a group in parts is whole vectors
inline bool vector_fits(const inpc_group_norm_config& cfg, int v) {
    return (tile_groups_of(cfg, v) != 0 ? cfg.channels : cfg.channels / cfg.groups) % (uint32_t)v == 0;
}

// What a call may need: [sums per (image, tile, group of a tile, slab)] [backward: sums per (image, slab, channel)] [means per
// (image, group)], the second with one slab in the single form.
struct Workspace {
    size_t of_groups, of_channels, means, bytes;
};
inline Workspace split_workspace(const Shape& s, bool backward) {
    Workspace w;
    w.of_groups = 0;
    w.of_channels = align_up((size_t)s.n * s.tiles * s.tile_groups * s.slabs * sizeof(float2), 256);
    w.means = w.of_channels + (backward ? align_up((size_t)s.n * s.slabs * s.channels * sizeof(float2), 256) : 0);
    w.bytes = w.means + (backward ? (size_t)s.n * s.groups * sizeof(float2) : 0);
    return w;
}
// ... whatever the alignment of its tensors
inline size_t workspace_bytes(const inpc_group_norm_config& cfg, bool backward) {
    size_t most = backward && cfg.n_images > 1 ? (size_t)cfg.n_images * cfg.channels * sizeof(float2) : 0;
    for (int v = (int)(16 / element_bytes(cfg.dtype)); v >= 1; v /= 2)
        if (vector_fits(cfg, v) && !runs_single(cfg, v))
            most = std::max(most, split_workspace(sums_shape(cfg, v), backward).bytes);
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
    // a thread's offset in a block's rows is counted in 32 bits
    if (cfg->input_pixel_stride >= (1u << 19) || cfg->grad_pixel_stride >= (1u << 19))
        return fail(INPC_E_UNSUPPORTED, "%s: pixel strides are below 2^19 elements", what);
    // a launch has fewer than 2^32 threads: at most a block per (image, group), or for large groups per (image, tile)
    if ((uint64_t)cfg->n_images * cfg->groups > 0xFFFFFFFFu / kThreads)
        return fail(INPC_E_UNSUPPORTED, "%s: too many images: at most %u groups in all", what, 0xFFFFFFFFu / kThreads);
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
    const Shape s = single_shape(cfg, V, threads);
    const Dropout d = make_dropout(cfg.dropout_p, cfg.seed, cfg.seed_dev, cfg.offset);
    INPC_LAUNCH("group_norm_single", (k_single<D, V>), dim3(s.n * s.groups), dim3(threads), stream, x, weight, bias, y, moments, s, d);
    return INPC_OK;
}

template <int D, int V>
int backward_single(const inpc_group_norm_config& cfg, const void* x, const void* dy, const float2* moments, const void* weight,
                    const void* bias, void* dx, void* dweight, void* dbias, char* ws, hipStream_t stream) {
    uint32_t threads = 0;
    const Shape s = single_shape(cfg, V, threads);
    const Dropout d = make_dropout(cfg.dropout_p, cfg.seed, cfg.seed_dev, cfg.offset);
    const bool later = s.n > 1 && (dweight || dbias);
    float2* sums = later ? (float2*)ws : nullptr;
    INPC_NORM_LAUNCH_LDS("group_norm_single_backward", (k_single_backward<D, V>), dim3(s.n * s.groups), dim3(threads),
                         column_floats<2 * V>(threads) * sizeof(float), stream, x, dy, moments, weight, bias, dx,
                         later ? (void*)nullptr : dweight, later ? (void*)nullptr : dbias, sums, s, d);
    if (later)
        INPC_LAUNCH("group_norm_parameter_gradients", k_parameter_gradients, dim3(div_up(s.channels, kParameterColumns)),
                    dim3(kThreads), stream, sums, s.n, dweight, dbias, s);
    return INPC_OK;
}

// k<D, V, Q> with the slots that vectors of V channels fall into
#define INPC_NORM_SLOTS(k, per_group, ...)                                             \
    do {                                                                               \
        if ((per_group) % V == 0) {                                                    \
            __VA_ARGS__((k<D, V, 1>))                                                  \
        } else if (V > 2 && (per_group) * 2 == V) {                                    \
            __VA_ARGS__((k<D, V, (V > 2 ? 2 : V)>))                                      \
        } else {                                                                       \
            __VA_ARGS__((k<D, V, V>))                                                  \
        }                                                                              \
    } while (0)

template <int D, int V>
int forward_split(const inpc_group_norm_config& cfg, const void* x, const void* weight, const void* bias, void* y, float2* moments,
                  char* ws, hipStream_t stream) {
    const Shape s = sums_shape(cfg, V);
    const Dropout d = make_dropout(cfg.dropout_p, cfg.seed, cfg.seed_dev, cfg.offset);
    float2* partial = (float2*)(ws + split_workspace(s, false).of_groups);
#define INPC_NORM_MOMENTS(k) INPC_LAUNCH("group_norm_moments", k, dim3(s.n * s.tiles * s.slabs), dim3(kThreads), stream, x, partial, s);
    INPC_NORM_SLOTS(k_moments, s.per_group, INPC_NORM_MOMENTS);
#undef INPC_NORM_MOMENTS
    const bool fold = folds(s);
    if (!fold)
        INPC_LAUNCH("group_norm_combine_moments", k_combine_moments, dim3(div_up(s.n * s.groups, kThreads / 64)), dim3(kThreads), stream,
                    partial, moments, s);
    Shape a = split_shape(cfg, V, fold ? kSumBlocks : kApplyBlocks);
    a.streamed = streams(cfg, 2);
    const float2* to_fold = fold ? partial : nullptr;
#define INPC_NORM_APPLY(k)                                                                                                              \
    INPC_LAUNCH("group_norm_apply", k, dim3(a.n * a.tiles * a.slabs), dim3(kThreads), stream, x, to_fold, weight, bias, y, moments, a, s, d);
    INPC_NORM_SLOTS(k_apply, s.per_group, INPC_NORM_APPLY);
#undef INPC_NORM_APPLY
    return INPC_OK;
}

template <int D, int V>
int backward_split(const inpc_group_norm_config& cfg, const void* x, const void* dy, const float2* moments, const void* weight,
                   const void* bias, void* dx, void* dweight, void* dbias, char* ws, hipStream_t stream) {
    const Shape s = sums_shape(cfg, V);
    const Dropout d = make_dropout(cfg.dropout_p, cfg.seed, cfg.seed_dev, cfg.offset);
    const Workspace w = split_workspace(s, true);
    float2 *of_groups = (float2*)(ws + w.of_groups), *of_channels = (float2*)(ws + w.of_channels), *means = (float2*)(ws + w.means);
#define INPC_NORM_SUMS(k)                                                                                                           \
    INPC_LAUNCH("group_norm_gradient_sums", k, dim3(s.n * s.tiles * s.slabs), dim3(kThreads), stream, x, dy, moments, weight, bias,  \
                of_channels, of_groups, s, d);
    INPC_NORM_SLOTS(k_gradient_sums, s.per_group, INPC_NORM_SUMS);
#undef INPC_NORM_SUMS
    // dweight and dbias are added up next to whatever comes next
    const bool fold = folds(s) && dx;
    const uint32_t parameter_blocks = dweight || dbias ? div_up(s.channels, kParameterColumns) : 0;
    if (!fold)
        INPC_LAUNCH("group_norm_combine_gradients", k_combine_gradients,
                    dim3(parameter_blocks + (dx ? div_up(s.n * s.groups, kThreads / 64) : 0)), dim3(kThreads), stream, of_groups,
                    of_channels, means, dweight, dbias, parameter_blocks, s);
    if (!dx) return INPC_OK;
    Shape a = split_shape(cfg, V, fold ? kSumBlocks : kApplyBlocks);
    a.streamed = streams(cfg, 3);
    const uint32_t first_blocks = fold ? parameter_blocks : 0;
    const float2* combined = fold ? nullptr : means;
#define INPC_NORM_GRADIENT(k)                                                                                                       \
    INPC_LAUNCH("group_norm_input_gradient", k, dim3(first_blocks + a.n * a.tiles * a.slabs), dim3(kThreads), stream, x, dy, moments, \
                of_channels, of_groups, combined, weight, bias, dx, dweight, dbias, first_blocks, a, s, d);
    INPC_NORM_SLOTS(k_input_gradient, s.per_group, INPC_NORM_GRADIENT);
#undef INPC_NORM_GRADIENT
    return INPC_OK;
}

// Of a map without values: the parameters' gradients are sums over nothing.
inline int backward_of_nothing(const inpc_group_norm_config& cfg, void* dweight, void* dbias, hipStream_t stream) {
    const Shape s = base_shape(cfg);
    if (dweight || dbias)
        INPC_LAUNCH("group_norm_parameter_gradients", k_parameter_gradients, dim3(div_up(s.channels, kParameterColumns)), dim3(kThreads),
                    stream, (const float2*)nullptr, 0u, dweight, dbias, s);
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
    int v = vector_width(bytes, divisible, pointers);
    const int in_group = vector_width(bytes, divisible | cfg.channels / cfg.groups, pointers);
    if (tile_groups_of(cfg, v) == 0) v = in_group;
    if (!runs_single(cfg, v)) return INPC_NORM_DISPATCH(forward_split, cfg.dtype, v, cfg, x, weight, bias, y, moments, ws, stream);
    return INPC_NORM_DISPATCH(forward_single, cfg.dtype, in_group, cfg, x, weight, bias, y, moments, stream);
}

inline int backward(const inpc_group_norm_config& cfg, const void* x, const void* dy, const float2* moments, const void* weight,
                    const void* bias, void* dx, void* dweight, void* dbias, char* ws, hipStream_t stream) {
    const size_t bytes = element_bytes(cfg.dtype);
    const uint64_t divisible = cfg.channels | cfg.input_image_stride | cfg.input_pixel_stride | cfg.grad_image_stride | cfg.grad_pixel_stride;
    const uintptr_t pointers = (uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx;
    int v = vector_width(bytes, divisible, pointers);
    const int in_group = vector_width(bytes, divisible | cfg.channels / cfg.groups, pointers);
    if (tile_groups_of(cfg, v) == 0) v = in_group;
    if (!runs_single(cfg, v))
        return INPC_NORM_DISPATCH(backward_split, cfg.dtype, v, cfg, x, dy, moments, weight, bias, dx, dweight, dbias, ws, stream);
    return INPC_NORM_DISPATCH(backward_single, cfg.dtype, in_group, cfg, x, dy, moments, weight, bias, dx, dweight, dbias, ws, stream);
}

}  // namespace norm
}  // namespace inpc
