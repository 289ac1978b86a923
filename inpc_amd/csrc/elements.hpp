// elements.hpp — vectors of fp32 / fp16 / bf16 values in memory, computed with in fp32, and the generator of the dropout
// masks: shared by the operators on feature maps (groupnorm.hpp) and on plain arrays (dropout.hpp).
#pragma once

#include <hip/hip_fp16.h>

#include <cmath>

#include "common.hpp"

namespace inpc {

// ---- element types ---------------------------------------------------------------------------------------------
template <int D>
constexpr int kElementBytes = D == INPC_DTYPE_F32 ? 4 : 2;

inline bool known_dtype(int32_t d) { return d == INPC_DTYPE_F32 || d == INPC_DTYPE_F16 || d == INPC_DTYPE_BF16; }
inline size_t element_bytes(int32_t d) { return d == INPC_DTYPE_F32 ? 4 : 2; }

__device__ __forceinline__ float f16_value(uint32_t bits) { return __half2float(__builtin_bit_cast(__half, (uint16_t)bits)); }
__device__ __forceinline__ float bf16_value(uint32_t bits) { return float_of_bits(bits << 16); }

// Both 16-bit types are rounded to nearest, ties to even, once, when a result is stored.
__device__ __forceinline__ uint32_t f16_bits(float v) { return (uint32_t)__builtin_bit_cast(uint16_t, __float2half_rn(v)); }
__device__ __forceinline__ uint32_t bf16_bits(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
    return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v);   // gfx950 has the conversion as an instruction
#else
    if (v != v) return 0x7FC0u;
    const uint32_t u = float_bits_of(v);
    return (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
#endif
}

template <int D>
__device__ __forceinline__ float value16(uint32_t bits) {
    return D == INPC_DTYPE_F16 ? f16_value(bits) : bf16_value(bits);
}
template <int D>
__device__ __forceinline__ uint32_t bits16(float v) {
    return D == INPC_DTYPE_F16 ? f16_bits(v) : bf16_bits(v);
}

// A vector of V elements as it lies in memory: at most 16 bytes, aligned to its own size.
template <int BYTES>
struct Packed;
template <>
struct Packed<16> { using type = uint4; };
template <>
struct Packed<8> { using type = uint2; };
template <>
struct Packed<4> { using type = uint32_t; };
template <>
struct Packed<2> { using type = uint16_t; };
template <int D, int V>
using PackedVector = typename Packed<V * kElementBytes<D>>::type;

__device__ __forceinline__ void to_words(const uint4& p, uint32_t (&w)[4]) { w[0] = p.x; w[1] = p.y; w[2] = p.z; w[3] = p.w; }
__device__ __forceinline__ void to_words(const uint2& p, uint32_t (&w)[4]) { w[0] = p.x; w[1] = p.y; }
__device__ __forceinline__ void to_words(uint32_t p, uint32_t (&w)[4]) { w[0] = p; }
__device__ __forceinline__ void to_words(uint16_t p, uint32_t (&w)[4]) { w[0] = p; }
__device__ __forceinline__ void from_words(const uint32_t (&w)[4], uint4& p) { p = make_uint4(w[0], w[1], w[2], w[3]); }
__device__ __forceinline__ void from_words(const uint32_t (&w)[4], uint2& p) { p = make_uint2(w[0], w[1]); }
__device__ __forceinline__ void from_words(const uint32_t (&w)[4], uint32_t& p) { p = w[0]; }
__device__ __forceinline__ void from_words(const uint32_t (&w)[4], uint16_t& p) { p = (uint16_t)w[0]; }

// A store that leaves the caches to what is read again.
__device__ __forceinline__ void store_streamed(uint4* to, const uint4& p) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef uint32_t words __attribute__((ext_vector_type(4)));
    __builtin_nontemporal_store(words{p.x, p.y, p.z, p.w}, (words*)to);
#else
    *to = p;
#endif
}
template <typename T>
__device__ __forceinline__ void store_streamed(T* to, const T& p) { *to = p; }   // narrower ones are not worth it

template <int D, int V>
__device__ __forceinline__ void unpack(const PackedVector<D, V>& p, float (&v)[V]) {
    uint32_t w[4] = {0, 0, 0, 0};
    to_words(p, w);
#pragma unroll
    for (int j = 0; j < V; ++j)
        v[j] = D == INPC_DTYPE_F32 ? float_of_bits(w[j % 4]) : value16<D>((w[j / 2 % 4] >> (16 * (j & 1))) & 0xFFFFu);
}

template <int D, int V>
__device__ __forceinline__ PackedVector<D, V> pack(const float (&v)[V]) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (D == INPC_DTYPE_F32) w[j % 4] = float_bits_of(v[j]);
        else w[j / 2 % 4] |= bits16<D>(v[j]) << (16 * (j & 1));
    }
    PackedVector<D, V> p;
    from_words(w, p);
    return p;
}

template <int D, int V>
__device__ __forceinline__ PackedVector<D, V> load_packed(const void* base, size_t element) {
    return *(const PackedVector<D, V>*)((const char*)base + element * kElementBytes<D>);
}
template <int D, int V>
__device__ __forceinline__ void load_vector(const void* base, size_t element, float (&v)[V]) {
    unpack<D, V>(load_packed<D, V>(base, element), v);
}
template <int D, int V>
__device__ __forceinline__ void store_vector(void* base, size_t element, const float (&v)[V]) {
    *(PackedVector<D, V>*)((char*)base + element * kElementBytes<D>) = pack<D, V>(v);
}

// One element of a small array whose type is only known at run time (weights and biases).
__device__ __forceinline__ float load_element(const void* base, int32_t dtype, size_t i) {
    if (dtype == INPC_DTYPE_F32) return ((const float*)base)[i];
    const uint32_t bits = ((const uint16_t*)base)[i];
    return dtype == INPC_DTYPE_F16 ? f16_value(bits) : bf16_value(bits);
}
// V neighbouring ones, `otherwise` where there are none. The type is asked once, so that all loads are on their way together.
template <int V>
__device__ __forceinline__ void load_elements(const void* base, int32_t dtype, size_t first, float otherwise, float (&v)[V]) {
    if (!base) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = otherwise;
    } else if (dtype == INPC_DTYPE_F32) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = ((const float*)base)[first + j];
    } else {
        uint16_t bits[V];
#pragma unroll
        for (int j = 0; j < V; ++j) bits[j] = ((const uint16_t*)base)[first + j];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = dtype == INPC_DTYPE_F16 ? f16_value(bits[j]) : bf16_value(bits[j]);
    }
}
__device__ __forceinline__ void store_element(void* base, int32_t dtype, size_t i, float v) {
    if (dtype == INPC_DTYPE_F32) ((float*)base)[i] = v;
    else ((uint16_t*)base)[i] = (uint16_t)(dtype == INPC_DTYPE_F16 ? f16_bits(v) : bf16_bits(v));
}

// ---- dropout ---------------------------------------------------------------------------------------------------
// Element i of a call is dropped iff u(i) < T, T = round(p * 2^32), u(i) uniform on 32 bits: its upper half is the 16-bit
// half i % 8 of draw 0 of block i / 8, its lower half the same of draw 1. A draw is Philox4x32-10 (Salmon, Moraes, Dror,
// Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) with the seed as the key and (block mod 2^32, block div
// 2^32 + 2^31 * draw, offset mod 2^32, offset div 2^32) as the counter. The upper half decides unless it equals T's, so
// eight elements (a 16-byte vector of a 16-bit type) cost one draw, and the second is made for one vector in 8192 or less:
// twenty 32x32->64-bit products, the generator's whole cost at quarter rate, per vector instead of per half.
struct Dropout {
    uint64_t seed, offset;
    const uint64_t* seed_dev;   // where not null: the seed's place in device memory; null where nothing is dropped, whatever the caller's
    uint32_t upper, lower;      // T = upper * 2^16 + lower, upper <= 2^16
    float scale;                // 1 / (1 - p); 0 where everything is dropped
    uint32_t on;
};

inline Dropout make_dropout(double p, uint64_t seed, const uint64_t* seed_dev, uint64_t offset) {
    const uint64_t threshold = (uint64_t)std::nearbyint(p * 4294967296.0);
    return Dropout{seed, offset, p > 0.0 ? seed_dev : nullptr, (uint32_t)(threshold >> 16), (uint32_t)(threshold & 0xFFFFu),
                   p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f, p > 0.0 ? 1u : 0u};
}

inline bool valid_probability(double p) { return p >= 0.0 && p <= 1.0; }

__device__ __forceinline__ void philox4x32_10(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c[0] * 0xD2511F53u, b = (uint64_t)c[2] * 0xCD9E8D57u;
        c[0] = (uint32_t)(b >> 32) ^ c[1] ^ k0;
        c[1] = (uint32_t)b;
        c[2] = (uint32_t)(a >> 32) ^ c[3] ^ k1;
        c[3] = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
}

__device__ __forceinline__ void dropout_draw(const Dropout& d, uint64_t seed, uint64_t block, uint32_t draw, uint32_t (&c)[4]) {
    c[0] = (uint32_t)block;
    c[1] = (uint32_t)(block >> 32) + (draw << 31);
    c[2] = (uint32_t)d.offset;
    c[3] = (uint32_t)(d.offset >> 32);
    philox4x32_10(c, (uint32_t)seed, (uint32_t)(seed >> 32));
}

__device__ __forceinline__ uint64_t dropout_seed(const Dropout& d) { return d.seed_dev ? *d.seed_dev : d.seed; }

// Half `lane` (0..7) of the four words of a draw.
__device__ __forceinline__ uint32_t draw_half(const uint32_t (&c)[4], uint32_t lane) {
    const uint32_t lo = lane & 4u ? c[2] : c[0], hi = lane & 4u ? c[3] : c[1];
    return ((lane & 2u ? hi : lo) >> (16u * (lane & 1u))) & 0xFFFFu;
}

// Elements first .. first + V - 1 (first a multiple of V, V a divisor of 8): bit j of the result is set where element j stays.
template <int V>
__device__ __forceinline__ uint32_t dropout_kept(const Dropout& d, uint64_t seed, uint64_t first) {
    uint32_t c[4];
    dropout_draw(d, seed, first >> 3, 0, c);
    const uint32_t lane0 = V == 8 ? 0u : (uint32_t)first & 7u;
    uint32_t kept = 0, tied = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const uint32_t h = draw_half(c, lane0 + j);
        kept |= h > d.upper ? 1u << j : 0u;
        tied |= h == d.upper ? 1u << j : 0u;
    }
    if (tied) {
        if (d.lower == 0) return kept | tied;
        dropout_draw(d, seed, first >> 3, 1, c);
#pragma unroll
        for (int j = 0; j < V; ++j)
            if ((tied >> j) & 1u) kept |= draw_half(c, lane0 + j) >= d.lower ? 1u << j : 0u;
    }
    return kept;
}

// a * b rounded to fp32. Without the barrier the compiler joins the product with a following conversion to fp16 into one
// mixed-precision instruction that rounds once, and the result would depend on the type it is stored in.
__device__ __forceinline__ float rounded_product(float a, float b) {
    float v = a * b;
#if defined(__HIP_DEVICE_COMPILE__)
    asm("" : "+v"(v));
#endif
    return v;
}

// v *= 1 / (1 - p) where the element stays, 0 elsewhere (whatever v was, a NaN included).
template <int V>
__device__ __forceinline__ void dropout_apply(const Dropout& d, uint64_t seed, uint64_t first, float (&v)[V]) {
    const uint32_t kept = dropout_kept<V>(d, seed, first);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (kept >> j) & 1u ? rounded_product(v[j], d.scale) : 0.0f;
}

}  // namespace inpc
