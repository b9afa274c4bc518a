// attention_types.h -- shared by the attention kernels: matrix products of
// 16-byte pieces, column sums, device-scope scratch and the shape of a
// wavefront's tile of keys. Device code only.
#ifndef NZ_ATTENTION_TYPES_H
#define NZ_ATTENTION_TYPES_H

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "serving_types.h"

namespace {

// Workgroups are placed on the XCDs in turn.
constexpr uint32_t kXcds = 8;
constexpr float kLog2e = 1.44269504088896340736f;

using f32x4 = vec<float, 4>;

// 16-byte pieces of a lane, and the product of two matrices of such pieces:
// 16 rows (lane % 16) by 4 * kRun of depth (lane / 16, element) times the
// same by 16 columns. Whichever depth index an element stands for, it is the
// same in both. Softmax weights are at most 2^kLift: fp16 ones are lifted so
// that small ones keep their bits (2^-24 is fp16's least). 16-bit types take
// a weight as head(p), cut off, and the rest, rounded: one rounding to 8 or 11
// bits would err more than everything else before the result's own rounding,
// and matrix instructions are not what bounds the kernel. Beside a head the
// rest is kept from being 0, so that an infinite value stays infinite in both
// products; a weight too small for a head is all rest, and may be 0.
template <typename T> struct Piece;

template <> struct Piece<bf16_t> {
    static constexpr uint32_t kRun = 8;
    static constexpr float kLift = 0.0f, kLeast = 0x1p-126f;
    using type = vec<bf16_t, 8>;
    static __device__ __forceinline__ bf16_t head(float p) {
        return __builtin_bit_cast(bf16_t, static_cast<uint16_t>(__float_as_uint(p) >> 16));
    }
    static __device__ __forceinline__ f32x4 mma(type a, type b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

template <> struct Piece<_Float16> {
    static constexpr uint32_t kRun = 8;
    static constexpr float kLift = 15.0f, kLeast = 0x1p-24f;
    using type = vec<_Float16, 8>;
    static __device__ __forceinline__ _Float16 head(float p) {
        return static_cast<_Float16>(__builtin_amdgcn_cvt_pkrtz(p, p)[0]);
    }
    static __device__ __forceinline__ f32x4 mma(type a, type b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

template <> struct Piece<float> {
    static constexpr uint32_t kRun = 4;
    static constexpr float kLift = 0.0f, kLeast = 0.0f;
    using type = vec<float, 4>;
    static __device__ __forceinline__ float head(float p) { return p; }
    static __device__ __forceinline__ f32x4 mma(type a, type b, f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

template <bool PAST, typename V, typename T>
__device__ __forceinline__ V fetch(const T* src) {
    const V* const p = reinterpret_cast<const V*>(src);
    return PAST ? __builtin_nontemporal_load(p) : *p;
}

// Largest of a column's values over the four lanes that hold it: those 16 and
// 32 lanes away come by exchanges of rows of lanes.
__device__ __forceinline__ float column_max(float v) {
    const uint32_t x = __float_as_uint(v);
    const auto near = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    const uint32_t y = __float_as_uint(fmaxf(__uint_as_float(near[0]), __uint_as_float(near[1])));
    const auto far = __builtin_amdgcn_permlane32_swap(y, y, false, false);
    return fmaxf(__uint_as_float(far[0]), __uint_as_float(far[1]));
}

__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// What a maximum's scores are measured from: 0 where every key is masked.
__device__ __forceinline__ float finite_base(float top) { return top == -__builtin_inff() ? 0.0f : top; }

// Four elements of a row; zeros where it has no keys.
template <typename T>
__device__ __forceinline__ void store_row(T* dst, f32x4 sum, float weight) {
    vec<T, 4> x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = from_float<T>(weight == 0.0f ? 0.0f : sum[i] / weight);
    *reinterpret_cast<vec<T, 4>*>(dst) = x;
}

// Sums that another workgroup, maybe of another XCD, will read: stores and
// loads of device scope go past the caches that only one XCD sees. A release
// fence would write back all of the XCD's L2 instead. (The buffer forms, for
// 16 bytes at a time; offsets are in bytes from a row's first item.)
constexpr int kDeviceScope = 16;   // sc1
using rsrc_t = __amdgpu_buffer_rsrc_t;

__device__ __forceinline__ rsrc_t device_buffer(float* base) {
    return __builtin_amdgcn_make_buffer_rsrc(base, 0, 0xFFFFFFFFu, 0x00020000u);
}

__device__ __forceinline__ void put_four(rsrc_t buffer, uint32_t offset, f32x4 x) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(vec<uint32_t, 4>, x), buffer, offset, 0, kDeviceScope);
}

__device__ __forceinline__ f32x4 get_four(rsrc_t buffer, uint32_t offset) {
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(buffer, offset, 0, kDeviceScope));
}

__device__ __forceinline__ void put_pair(rsrc_t buffer, uint32_t offset, float x, float y) {
    __builtin_amdgcn_raw_buffer_store_b64(vec<uint32_t, 2>{__float_as_uint(x), __float_as_uint(y)}, buffer, offset, 0,
                                          kDeviceScope);
}

__device__ __forceinline__ vec<float, 2> get_pair(rsrc_t buffer, uint32_t offset) {
    return __builtin_bit_cast(vec<float, 2>, __builtin_amdgcn_raw_buffer_load_b64(buffer, offset, 0, kDeviceScope));
}

template <typename T, uint32_t DP>
struct Shape {
    static constexpr uint32_t kRun = Piece<T>::kRun;
    static constexpr uint32_t kKeySteps = DP / (4 * kRun);              // pieces of a key row per lane
    static constexpr uint32_t kValueRun = DP / 16 < kRun ? DP / 16 : kRun;   // neighbours a lane loads of a value row
    static constexpr uint32_t kValueSteps = DP / (16 * kValueRun);
    // keys a wavefront takes at a time, in runs of 16: fewer where a tile's
    // keys and values would not fit the registers
    static constexpr uint32_t kHalves = sizeof(T) == 4 && DP > 64 ? 1 : 2, kKeys = 16 * kHalves;
    static constexpr uint32_t kGroups = kKeys / (4 * kRun);             // value products per tile
};

}  // namespace

#endif
