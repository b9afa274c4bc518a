// serving_types.h -- shared by the serving-step kernels: value types, their
// loads to and stores from 32-bit floats, a search in prefix sums. Device code
// only.
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

// Saturating, so that sums of absurd requests stay past every limit.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add(uint32_t v) {
    const int below = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false);
    return add_sat(v, static_cast<uint32_t>(below));
}

// Inclusive saturating prefix sum over the wavefront: shifts of 1, 2, 4 and 8
// lanes inside each row of 16, then the rows' carries.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v = dpp_add<0x111, 0xF>(v);
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);
    return dpp_add<0x143, 0xC>(v);
}

// The wavefront's last lane's value.
__device__ __forceinline__ uint32_t last_lane(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}

// The last i in [0, n) with first[i] <= x, where first[0] <= x.
__device__ __forceinline__ uint32_t owner(const uint32_t* first, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (first[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

}  // namespace

#endif
