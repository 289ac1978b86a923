// dropout.hpp — y = 0 where the mask drops the element, x / (1 - p) elsewhere; the backward pass is the same map on the
// gradient, with the mask computed again (elements.hpp) instead of stored. x and y may be the same memory.
//
// What bounds it: memory. 8,388,352 x 64 bf16 values (1.07 GB) 340 us, 6.3 TB/s read and written; 65 MB of fp16 21 us (6.2 TB/s, in
// part from the memory-side cache). The generator's twenty products per eight values are hidden behind that; with a draw per
// four values (32 bits each) they would take as long as the memory does for 16-bit types.
#pragma once

#include <algorithm>

#include "elements.hpp"

namespace inpc {
namespace dropout {

constexpr int kBlock = 256;
constexpr uint64_t kMostBlocks = 1u << 20;   // a launch has fewer than 2^32 threads: beyond 2^31 values a thread takes several vectors

// A thread takes eight consecutive elements, one draw of the generator. WIDE: both pointers are 16-byte aligned.
template <int D, bool WIDE>
__global__ void __launch_bounds__(kBlock) k_dropout(const void* x, void* y, uint64_t count, Dropout d) {
    const uint64_t seed = dropout_seed(d), stride = (uint64_t)gridDim.x * kBlock * 8u;
    constexpr int W = D == INPC_DTYPE_F32 ? 4 : 8;
    for (uint64_t first = ((uint64_t)blockIdx.x * kBlock + threadIdx.x) * 8u; first < count; first += stride) {
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
        } else {
            const uint32_t kept = dropout_kept<8>(d, seed, first);
            const uint32_t n = (uint32_t)min((unsigned long long)(count - first), 8ull);
            for (uint32_t j = 0; j < n; ++j) {
                float one[1];
                load_vector<D, 1>(x, first + j, one);
                one[0] = (kept >> j) & 1u ? rounded_product(one[0], d.scale) : 0.0f;
                store_vector<D, 1>(y, first + j, one);
            }
        }
    }
}

template <int D>
int launch(const void* x, void* y, uint64_t count, const Dropout& d, hipStream_t stream) {
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((count + 8 * kBlock - 1) / (8 * kBlock), kMostBlocks);
    if (((uintptr_t)x | (uintptr_t)y) % 16 == 0) {
        INPC_LAUNCH("dropout", (k_dropout<D, true>), dim3(blocks), dim3(kBlock), stream, x, y, count, d);
    } else {
        INPC_LAUNCH("dropout", (k_dropout<D, false>), dim3(blocks), dim3(kBlock), stream, x, y, count, d);
    }
    return INPC_OK;
}

}  // namespace dropout
}  // namespace inpc
