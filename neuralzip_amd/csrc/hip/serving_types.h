// serving_types.h -- value types of the serving-step kernels: loads to and
// stores from 32-bit floats. Device code only.
#ifndef NZ_SERVING_TYPES_H
#define NZ_SERVING_TYPES_H

#include <hip/hip_runtime.h>

#include <stdint.h>

namespace {

using bf16_t = __bf16;

template <typename T>
__device__ __forceinline__ float to_float(T x) { return static_cast<float>(x); }

// Rounded to nearest, ties to even; NaN stays NaN.
template <typename T>
__device__ __forceinline__ T from_float(float x) { return static_cast<T>(x); }

template <typename T, int N>
using vec = T __attribute__((ext_vector_type(N)));

// Eight neighbours, in 16-byte accesses.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
    constexpr int kRun = 16 / sizeof(T);
#pragma unroll
    for (int r = 0; r < 8 / kRun; ++r) {
        const vec<T, kRun> v = *reinterpret_cast<const vec<T, kRun>*>(p + r * kRun);
#pragma unroll
        for (int i = 0; i < kRun; ++i) x[r * kRun + i] = to_float(static_cast<T>(v[i]));
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x) {
    constexpr int kRun = 16 / sizeof(T);
#pragma unroll
    for (int r = 0; r < 8 / kRun; ++r) {
        vec<T, kRun> v;
#pragma unroll
        for (int i = 0; i < kRun; ++i) v[i] = from_float<T>(x[r * kRun + i]);
        *reinterpret_cast<vec<T, kRun>*>(p + r * kRun) = v;
    }
}

// (a, b) turned by the angle whose cosine and sine are c and s.
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
    const float x = a * c - b * s;
    b = b * c + a * s;
    a = x;
}

}  // namespace

#endif
