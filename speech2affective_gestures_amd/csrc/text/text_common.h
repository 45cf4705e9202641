// Shared by the text-model kernels: fp32 / bf16 element access, 16-byte vectors, sums across a wavefront.
#pragma once
#include "../s2ag_common.h"
#include "s2ag_text.h"

namespace s2ag {
namespace text {

typedef __bf16 bf16_t;
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// The elements that 16 bytes hold, widened to fp32 (exact) and rounded back (to nearest even, the one rounding of a result).
// `_any`: at any multiple of the element's size; one 16-byte access all the same.
typedef bf16x8 bf16x8_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void load(const float* p, float* v) {
        const f32x4 q = *reinterpret_cast<const f32x4*>(p);
        for (int i = 0; i < 4; ++i) v[i] = (float)q[i];
    }
    static __device__ __forceinline__ void store(float* p, const float* v) {
        f32x4 q;
        for (int i = 0; i < 4; ++i) q[i] = (float)v[i];
        *reinterpret_cast<f32x4*>(p) = q;
    }
    static __device__ __forceinline__ void load_any(const float* p, float* v) {
        const f32x4 q = *reinterpret_cast<const f32x4_any*>(p);
        for (int i = 0; i < 4; ++i) v[i] = (float)q[i];
    }
    static __device__ __forceinline__ void store_any(float* p, const float* v) {
        f32x4 q;
        for (int i = 0; i < 4; ++i) q[i] = (float)v[i];
        *reinterpret_cast<f32x4_any*>(p) = q;
    }
};
template <> struct Vec<bf16_t> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void load(const bf16_t* p, float* v) {
        const bf16x8 q = *reinterpret_cast<const bf16x8*>(p);
        for (int i = 0; i < 8; ++i) v[i] = (float)q[i];
    }
    static __device__ __forceinline__ void store(bf16_t* p, const float* v) {
        bf16x8 q;
        for (int i = 0; i < 8; ++i) q[i] = (bf16_t)v[i];
        *reinterpret_cast<bf16x8*>(p) = q;
    }
    static __device__ __forceinline__ void load_any(const bf16_t* p, float* v) {
        const bf16x8 q = *reinterpret_cast<const bf16x8_any*>(p);
        for (int i = 0; i < 8; ++i) v[i] = (float)q[i];
    }
    static __device__ __forceinline__ void store_any(bf16_t* p, const float* v) {
        bf16x8 q;
        for (int i = 0; i < 8; ++i) q[i] = (bf16_t)v[i];
        *reinterpret_cast<bf16x8_any*>(p) = q;
    }
};

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline long long round_up(long long v, long long m) { return (v + m - 1) / m * m; }

__device__ __forceinline__ long long load_id(const void* ids, int i32, long long i) {
    return i32 ? (long long)reinterpret_cast<const int*>(ids)[i] : reinterpret_cast<const long long*>(ids)[i];
}

}  // namespace text
}  // namespace s2ag
