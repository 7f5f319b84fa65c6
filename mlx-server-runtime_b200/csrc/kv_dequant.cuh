// Packed KV codes to exact 16-bit pairs and their values. A code ORed into the mantissa of
// a 16-bit float with a fixed exponent is offset + code exactly, the offset is subtracted
// exactly, and one packed FMA gives s * q + b with a single rounding: the value the cache
// stands for, the same in every kernel that reads it.
#pragma once

#include "common.cuh"
#include "paged_ops.h"

namespace mlxq {

template <typename T>
struct Pk;
template <>
struct Pk<__nv_bfloat16> {
    using V2 = __nv_bfloat162;
};
template <>
struct Pk<__half> {
    using V2 = __half2;
};

template <typename T>
__device__ __forceinline__ uint32_t pk_add(uint32_t a, uint32_t b) {
    using V2 = typename Pk<T>::V2;
    V2 r = __hadd2(*reinterpret_cast<V2*>(&a), *reinterpret_cast<V2*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
}
template <typename T>
__device__ __forceinline__ uint32_t pk_fma(uint32_t a, uint32_t b, uint32_t c) {
    using V2 = typename Pk<T>::V2;
    V2 r = __hfma2(*reinterpret_cast<V2*>(&a), *reinterpret_cast<V2*>(&b),
                   *reinterpret_cast<V2*>(&c));
    return *reinterpret_cast<uint32_t*>(&r);
}
template <typename T>
__device__ __forceinline__ uint32_t pk_round(float a, float b) {  // a in the low half
    if constexpr (__is_same(T, __nv_bfloat16)) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&r);
    } else {
        const __half2 r = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}
__device__ __forceinline__ float ex2(float x) {  // 2^x, results below 2^-126 as zero
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
    return r;
}

// Two 4-bit codes at bits 0-3 and 16-19 of h (other bits arbitrary) as an exact pair.
template <typename T>
__device__ __forceinline__ uint32_t nibbles_pair(uint32_t h) {
    constexpr uint32_t magic = __is_same(T, __nv_bfloat16) ? 0x43004300u : 0x64006400u;
    constexpr uint32_t minus = __is_same(T, __nv_bfloat16) ? 0xC300C300u : 0xE400E400u;
    return pk_add<T>(lop_and_or<0x000F000Fu>(h, magic), minus);
}

// Two 8-bit codes in bytes 0 and 2 of h (bytes 1 and 3 arbitrary) as an exact pair. f16
// takes all eight bits behind 0x64 (1024 + q). bf16 holds seven behind 0x43 (128 + low
// seven bits), so 128 is subtracted only where the code's top bit is clear.
template <typename T>
__device__ __forceinline__ uint32_t bytes_pair(uint32_t h) {
    if constexpr (__is_same(T, __nv_bfloat16)) {
        const uint32_t top = prmt(h, 0u, 0xAA88u);  // 0xffff where the code's top bit is set
        return pk_add<T>(lop_and_or<0x007F007Fu>(h, 0x43004300u), ~top & 0xC300C300u);
    } else {
        return pk_add<T>(lop_and_or<0x00FF00FFu>(h, 0x64006400u), 0xE400E400u);
    }
}

__device__ __forceinline__ uint32_t pk_splat(uint32_t h) { return prmt(h, h, 0x1010u); }

// Pair p of a row's packed words w as values (p is a compile-time constant after
// unrolling). The two elements of a pair are not neighbours in general (see pair_dims).
//   16 bits: word p              8 bits: bytes p%2 and p%2 + 2 of word p/2
//    4 bits: nibbles p%4 and p%4 + 4 of word p/4
template <typename T, int BITS>
__device__ __forceinline__ uint32_t row_pair(const uint32_t* w, int p, uint32_t s2, uint32_t b2) {
    if constexpr (BITS == 16) {
        return w[p];
    } else if constexpr (BITS == 8) {
        return pk_fma<T>(bytes_pair<T>(w[p / 2] >> (8 * (p % 2))), s2, b2);
    } else {
        return pk_fma<T>(nibbles_pair<T>(w[p / 4] >> (4 * (p % 4))), s2, b2);
    }
}
template <int BITS>
__host__ __device__ constexpr int pair_dim(int p, int e) {
    return BITS == 16 ? 2 * p + e : BITS == 8 ? 4 * (p / 2) + p % 2 + 2 * e
                                              : 8 * (p / 4) + p % 4 + 4 * e;
}

// Element i of two rows' packed words wa, wb as a pair of values (row a in the low half);
// s2, b2: (scale of a, scale of b), (bias of a, bias of b).
template <typename T, int BITS>
__device__ __forceinline__ uint32_t cross_pair(const uint32_t* wa, const uint32_t* wb, int i,
                                               uint32_t s2, uint32_t b2) {
    if constexpr (BITS == 16) {
        return prmt(wa[i / 2], wb[i / 2], (i % 2) ? 0x7632u : 0x5410u);
    } else if constexpr (BITS == 8) {
        const int j = i % 4;
        // bytes: a_j, a_j, b_j, b_j
        return pk_fma<T>(bytes_pair<T>(prmt(wa[i / 4], wb[i / 4], 0x4400u + 0x1111u * j)), s2, b2);
    } else {
        const uint32_t h = prmt(wa[i / 8], wb[i / 8], (i % 8) < 4 ? 0x5410u : 0x7632u);
        return pk_fma<T>(nibbles_pair<T>(h >> (4 * (i % 4))), s2, b2);
    }
}

// Eight values in order from the words that hold them.
template <typename T, int BITS>
__device__ __forceinline__ uint4 in_order(const uint32_t* w, uint32_t s2, uint32_t b2) {
    uint32_t p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = row_pair<T, BITS>(w, j, s2, b2);
    if constexpr (BITS == 8)  // pairs (0,2) (1,3) (4,6) (5,7)
        return make_uint4(prmt(p[0], p[1], 0x5410u), prmt(p[0], p[1], 0x7632u),
                          prmt(p[2], p[3], 0x5410u), prmt(p[2], p[3], 0x7632u));
    // pairs (0,4) (1,5) (2,6) (3,7)
    return make_uint4(prmt(p[0], p[1], 0x5410u), prmt(p[2], p[3], 0x5410u),
                      prmt(p[0], p[1], 0x7632u), prmt(p[2], p[3], 0x7632u));
}

// Eight values of a pool: chunk `at` of eight elements of its rows.
template <typename T, int BITS>
__device__ __forceinline__ uint4 cache_chunk(const KvCache& c, bool is_v, size_t at) {
    const void* data = is_v ? c.v : c.k;
    if constexpr (BITS == 16) {
        return static_cast<const uint4*>(data)[at];
    } else {
        uint32_t w[BITS / 4];
        if constexpr (BITS == 8) {
            const uint2 v = static_cast<const uint2*>(data)[at];
            w[0] = v.x;
            w[1] = v.y;
        } else {
            w[0] = static_cast<const uint32_t*>(data)[at];
        }
        const size_t g = at * 8 / c.gs;
        return in_order<T, BITS>(w, pk_splat(static_cast<const uint16_t*>(is_v ? c.vs : c.ks)[g]),
                                 pk_splat(static_cast<const uint16_t*>(is_v ? c.vb : c.kb)[g]));
    }
}

}  // namespace mlxq
