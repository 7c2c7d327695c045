// logits.hpp - rows of logits as logprobs.hip and verify.hip read them.
#pragma once

#include "common.hpp"

namespace ouro {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ float logit(const T *x, int64_t i) {
    float v;
    if constexpr (sizeof(T) == 4)
        v = x[i];
    else
        v = bf16_bits_to_f32(x[i]);
    return v != v ? -INFINITY : v;
}

// A row in 16-byte vectors from the last multiple of 16 bytes at or before its
// start: vector q holds elements q VL - shift .. q VL - shift + VL - 1.
template <typename T>
struct LogitRow {
    static constexpr int VL = 16 / sizeof(T);
    const T *x;
    int n, shift;
    __device__ __forceinline__ LogitRow(const T *row, int len) : x(row), n(len) {
        shift = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    }
    __device__ __forceinline__ int first(int q) const { return q * VL - shift; }
    // Vector q as bits: whole where it lies in the row, else its elements one by
    // one with -inf in the places of others.
    __device__ __forceinline__ u32x4_t load(int q) const {
        const int e0 = first(q);
        if (e0 >= 0 && e0 + VL <= n) return *reinterpret_cast<const u32x4_t *>(x + e0);
        u32x4_t r;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if constexpr (sizeof(T) == 4) {
                const int e = e0 + w;
                r[w] = e >= 0 && e < n ? __float_as_uint(x[e]) : 0xff800000u;
            } else {
                const int e = e0 + 2 * w;
                const uint32_t lo = e >= 0 && e < n ? x[e] : 0xff80u, hi = e + 1 >= 0 && e + 1 < n ? x[e + 1] : 0xff80u;
                r[w] = lo | hi << 16;
            }
        }
        return r;
    }
    // Element e of a vector as it is, and with NaN as -inf.
    static __device__ __forceinline__ float raw(const u32x4_t &v, int e) {
        if constexpr (sizeof(T) == 4) return __uint_as_float(v[e]);
        return __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
    }
    static __device__ __forceinline__ float at(const u32x4_t &v, int e) {
        const float f = raw(v, e);
        return f != f ? -INFINITY : f;
    }
};

}  // namespace ouro
