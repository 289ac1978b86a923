// dropout.hpp — y = 0 where the mask drops the element, x / (1 - p) elsewhere; the backward pass is the same map on the
// gradient, with the mask computed again (elements.hpp) instead of stored. x and y may be the same memory.
//
// What bounds it: memory. 8,388,352 x 64 bf16 values (1.07 GB) 340 us back to back, 6.3 TB/s read and written; 65 MB of fp16 21 us (6.2 TB/s, in
// part from the memory-side cache). The generator's twenty products per eight values are hidden behind that; with a draw per
// four values (32 bits each) they would take as long as the memory does for 16-bit types.
#pragma once

#include <algorithm>

#include "elements.hpp"

namespace inpc {
namespace dropout {

constexpr int kBlock = 256;
constexpr uint64_t kLaunch = 1ull << 32;   // values of a launch, which has fewer than 2^32 threads

// A thread takes eight consecutive elements, one draw of the generator. WIDE: both pointers are 16-byte aligned. No loop over
// vectors: one costs a tenth (65 MB 20.6 -> 22.7 us).
template <int D, bool WIDE>
__global__ void __launch_bounds__(kBlock) k_dropout(const void* x, void* y, uint64_t begin, uint64_t count, Dropout d) {
    const uint64_t first = begin + ((uint64_t)blockIdx.x * kBlock + threadIdx.x) * 8u;
    if (first >= count) return;
    const uint64_t seed = dropout_seed(d);
    constexpr int W = D == INPC_DTYPE_F32 ? 4 : 8;
    if (WIDE && first + 8 <= count) {
        float v[8], part[W];
#pragma unroll
        for (int k = 0; k < 8 / W; ++k) {
            load_vector<D, W>(x, first + k * W, part);
#pragma unroll
            for (int j = 0; j < W; ++j) v[k * W + j] = part[j];
        }
        dropout_apply<8>(d, seed, first, v);
#pragma unroll
        for (int k = 0; k < 8 / W; ++k) {
#pragma unroll
            for (int j = 0; j < W; ++j) part[j] = v[k * W + j];
            store_vector<D, W>(y, first + k * W, part);
        }
        return;
    }
    const uint32_t kept = dropout_kept<8>(d, seed, first);
    const uint32_t n = (uint32_t)min((unsigned long long)(count - first), 8ull);
    for (uint32_t j = 0; j < n; ++j) {
        float one[1];
        load_vector<D, 1>(x, first + j, one);
        one[0] = (kept >> j) & 1u ? rounded_product(one[0], d.scale) : 0.0f;
        store_vector<D, 1>(y, first + j, one);
    }
}

template <int D>
int launch(const void* x, void* y, uint64_t count, const Dropout& d, hipStream_t stream) {
    const bool wide = ((uintptr_t)x | (uintptr_t)y) % 16 == 0;
    for (uint64_t begin = 0; begin < count; begin += kLaunch) {
        const dim3 blocks((uint32_t)((std::min(count - begin, kLaunch) + 8 * kBlock - 1) / (8 * kBlock)));
        if (wide) {
            INPC_LAUNCH("dropout", (k_dropout<D, true>), blocks, dim3(kBlock), stream, x, y, begin, count, d);
        } else {
            INPC_LAUNCH("dropout", (k_dropout<D, false>), blocks, dim3(kBlock), stream, x, y, begin, count, d);
        }
    }
    return INPC_OK;
}

}  // namespace dropout
}  // namespace inpc
