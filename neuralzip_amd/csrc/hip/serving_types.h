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

// Elements of a 16-byte access.
template <typename T>
constexpr uint32_t run_of() { return 16 / sizeof(T); }

// Eight elements as 16-byte runs `apart` elements from one another.
template <typename T>
__device__ __forceinline__ void load_runs(const T* p, uint32_t apart, float* x) {
    constexpr uint32_t kRun = run_of<T>();
#pragma unroll
    for (uint32_t r = 0; r < 8 / kRun; ++r) {
        const vec<T, kRun> v = *reinterpret_cast<const vec<T, kRun>*>(p + r * apart);
#pragma unroll
        for (uint32_t i = 0; i < kRun; ++i) x[r * kRun + i] = to_float(static_cast<T>(v[i]));
    }
}

// Streaming stores.
template <typename T>
__device__ __forceinline__ void store_runs(T* p, uint32_t apart, const float* x) {
    constexpr uint32_t kRun = run_of<T>();
#pragma unroll
    for (uint32_t r = 0; r < 8 / kRun; ++r) {
        vec<T, kRun> v;
#pragma unroll
        for (uint32_t i = 0; i < kRun; ++i) v[i] = from_float<T>(x[r * kRun + i]);
        __builtin_nontemporal_store(v, reinterpret_cast<vec<T, kRun>*>(p + r * apart));
    }
}

// N neighbouring 32-bit floats, on a 16-byte boundary.
template <uint32_t N>
__device__ __forceinline__ void load_floats(const float* p, float* x) {
#pragma unroll
    for (uint32_t i = 0; i < N; i += 4) {
        const vec<float, 4> v = *reinterpret_cast<const vec<float, 4>*>(p + i);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) x[i + j] = v[j];
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
