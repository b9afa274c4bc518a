// attention_gfx950.hip -- attention of single tokens over a paged key-value
// cache: the plan that cuts the rows' contexts into items (nz_attention_plan)
// and the kernels that run it (nz_attention).
#include <hip/hip_runtime.h>

#include <stdint.h>
#include <stdio.h>

#include "neuralzip_hip.h"
#include "serving_types.h"

namespace {

// ------------------------------------------------------------------- plan

constexpr uint32_t kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
// Items start at multiples of the keys a wavefront takes at a time, and are
// cut no smaller than gives each wavefront of a workgroup one such tile.
constexpr uint32_t kTile = 32, kLeastItem = 128;

__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

__global__ __launch_bounds__(kPlanThreads) void nz_attention_plan_kernel(const int32_t* __restrict__ contexts,
                                                                         const int32_t* __restrict__ requests,
                                                                         uint32_t n_rows, uint32_t target,
                                                                         nz_attention_item* __restrict__ items) {
    __shared__ uint64_t sums[kPlanWaves];
    __shared__ uint32_t counts[kPlanWaves];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t keys = 0;
    for (uint32_t r = threadIdx.x; r < n_rows; r += kPlanThreads) keys += static_cast<uint32_t>(max(contexts[r], 0));
    keys = wave_sum(keys);
    if (lane == 0) sums[wave] = keys;
    __syncthreads();
    keys = 0;
#pragma unroll
    for (uint32_t w = 0; w < kPlanWaves; ++w) keys += sums[w];
    // the items' length: the sum of ceil(context / most) over the rows is at most n_rows + target
    uint64_t share = (keys + target - 1) / target;
    share = share < kLeastItem ? kLeastItem : (share + kTile - 1) / kTile * kTile;
    const uint32_t most = static_cast<uint32_t>(share < 0x80000000ull ? share : 0x80000000ull);
    uint32_t first = 0;
    for (uint32_t r0 = 0; r0 < n_rows; r0 += kPlanThreads) {
        const uint32_t r = r0 + threadIdx.x;
        const bool live = r < n_rows;
        const uint32_t context = live ? static_cast<uint32_t>(max(contexts[r], 0)) : 0;
        // a row's items are of equal length, in whole tiles
        uint32_t n = max((context + most - 1) / most, 1u);
        const uint32_t each = max(((context + n - 1) / n + kTile - 1) / kTile * kTile, kTile);
        n = live ? max((context + each - 1) / each, 1u) : 0;
        uint32_t scan = n;
#pragma unroll
        for (uint32_t d = 1; d < 64; d <<= 1) {
            const uint32_t below = __shfl_up(scan, d);
            if (lane >= d) scan += below;
        }
        __syncthreads();   // the last strip's reads of `counts`
        if (lane == 63) counts[wave] = scan;
        __syncthreads();
        uint32_t before = first, total = 0;
#pragma unroll
        for (uint32_t w = 0; w < kPlanWaves; ++w) {
            if (w < wave) before += counts[w];
            total += counts[w];
        }
        const uint32_t base = before + scan - n;
        for (uint32_t i = 0; i < n; ++i) {
            nz_attention_item item;
            item.row = static_cast<int32_t>(r);
            item.request = requests ? requests[r] : static_cast<int32_t>(r);
            item.begin = static_cast<int32_t>(i * each);
            item.end = static_cast<int32_t>(min(context, (i + 1) * each));
            item.index = static_cast<int32_t>(i);
            item.count = static_cast<int32_t>(n);
            item.first = static_cast<int32_t>(base);
            item.reserved = 0;
            items[base + i] = item;
        }
        first += total;
    }
    const nz_attention_item none = {-1, -1, 0, 0, 0, 0, 0, 0};
    for (uint32_t i = first + threadIdx.x; i < n_rows + target; i += kPlanThreads) items[i] = none;
}

// -------------------------------------------------------------- attention

constexpr uint32_t kWaves = 4, kThreads = 64 * kWaves;
// Query heads of one key-value head that a workgroup takes: the columns of a
// matrix instruction.
constexpr uint32_t kHeads = 16;
constexpr float kLog2e = 1.44269504088896340736f;

using f32x4 = vec<float, 4>;

// 16-byte pieces of a lane, and the product of two matrices of such pieces:
// 16 rows (lane % 16) by 4 * kRun of depth (lane / 16, element) times the
// same by 16 columns. Whichever depth index an element stands for, it is the
// same in both. Softmax weights are at most 2^kLift: fp16 ones are lifted so
// that small ones keep their bits (2^-24 is fp16's least). 16-bit types take
// a weight as head(p), cut off, and the rest, rounded: one rounding to 8 or 11
// bits would err more than everything else before the result's own rounding,
// and matrix instructions are not what bounds the kernel. The rest is kept
// from being 0, so that an infinite value stays infinite in both products.
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

// Largest of a column's values over the four lanes that hold it.
__device__ __forceinline__ float column_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

template <typename T, uint32_t DP>
struct Shape {
    static constexpr uint32_t kRun = Piece<T>::kRun;
    static constexpr uint32_t kKeySteps = DP / (4 * kRun);              // pieces of a key row per lane
    static constexpr uint32_t kValueRun = DP / 16 < kRun ? DP / 16 : kRun;   // neighbours a lane loads of a value row
    static constexpr uint32_t kValueSteps = DP / (16 * kValueRun);
    static constexpr uint32_t kGroups = kTile / (4 * kRun);             // value products per tile
};

// One item: 16 query heads' softmax over the keys begin .. end - 1 of one
// key-value head, tile by tile with a running maximum and sum. Scores are
// computed transposed (keys are rows, heads columns), so that a lane's
// scores of a tile are the very elements it needs as the second operand of
// the product with the values: its four rows of each 16 keys. The values are
// loaded whole rows at a time, each lane some neighbours of the keys its
// scores belong to, and transposed in registers; no LDS until the
// wavefronts' sums are joined.
template <typename T, uint32_t DP, bool FULL>
__global__ __launch_bounds__(kThreads) void nz_attention_kernel(nz_attention_args a) {
    using S = Shape<T, DP>;
    using P = Piece<T>;
    using piece = typename P::type;
    using value_run = vec<T, S::kValueRun>;
    __shared__ float lds_m[kWaves][kHeads], lds_l[kWaves][kHeads];
    __shared__ __align__(16) float lds_o[kWaves][kHeads][DP + 4];

    const uint32_t group = a.heads / a.kv_heads, blocks = (group + kHeads - 1) / kHeads;
    const uint32_t per_item = a.kv_heads * blocks;
    const uint32_t which = blockIdx.x / per_item, part = blockIdx.x % per_item;
    const nz_attention_item item = a.items[which];
    if (static_cast<uint32_t>(item.row) >= a.n_rows) return;
    const uint32_t kv_head = part / blocks, head0 = kv_head * group + part % blocks * kHeads;
    const uint32_t heads = min(kHeads, (kv_head + 1) * group - head0);
    const uint32_t lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t shift = 31 - __clz(a.page_size), place_mask = a.page_size - 1;
    const uint32_t end = static_cast<uint32_t>(item.end);
    const bool known = static_cast<uint32_t>(item.request) < a.n_requests;
    const int32_t* table = a.tables + static_cast<uint64_t>(known ? item.request : 0) * a.max_pages;

    piece q[S::kKeySteps];
    {
        const T* src = static_cast<const T*>(a.q) + item.row * a.q_row + (head0 + col) * a.q_head;
#pragma unroll
        for (uint32_t s = 0; s < S::kKeySteps; ++s) {
            const uint32_t d = s * 4 * S::kRun + quad * S::kRun;
            q[s] = piece{};
            if (col < heads && (FULL || d < a.head_dim)) q[s] = *reinterpret_cast<const piece*>(src + d);
        }
    }
    const float scale = a.scale * kLog2e;
    f32x4 o[S::kValueSteps][S::kValueRun] = {};
    float m = -__builtin_inff(), l = 0.0f;

    for (uint32_t t0 = static_cast<uint32_t>(item.begin) + wave * kTile; t0 < end; t0 += kWaves * kTile) {
        float score[2][4];
        const T* values[2];
        uint32_t limit[2];
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            // 16 keys of one page; where there is none, page 0 is read and everything masked
            const uint32_t t = t0 + 16 * h, entry = t >> shift;
            const int32_t p = known && t < end && entry < a.max_pages ? table[entry] : -1;
            const bool valid = static_cast<uint32_t>(p) < a.n_pages;
            const int64_t page = valid ? p : 0;
            limit[h] = valid ? end : 0;
            const T* keys = static_cast<const T*>(a.key_cache) + page * a.key_page + kv_head * a.key_head
                            + static_cast<int64_t>(t & place_mask) * a.key_slot;
            values[h] = static_cast<const T*>(a.value_cache) + page * a.value_page + kv_head * a.value_head
                        + static_cast<int64_t>(t & place_mask) * a.value_slot;
            f32x4 acc = {};
#pragma unroll
            for (uint32_t s = 0; s < S::kKeySteps; ++s) {
                const uint32_t d = s * 4 * S::kRun + quad * S::kRun;
                piece k = {};
                if (FULL || d < a.head_dim) k = *reinterpret_cast<const piece*>(keys + col * a.key_slot + d);
                acc = P::mma(k, q[s], acc);
            }
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                score[h][i] = t + 4 * quad + i < limit[h] ? acc[i] * scale : -__builtin_inff();
        }
        float top = m;
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) top = fmaxf(top, score[h][i]);
        top = column_max(top);
        const float base = top == -__builtin_inff() ? 0.0f : top;
        const float fade = __builtin_amdgcn_exp2f(m - base);
        m = top;
        l *= fade;
#pragma unroll
        for (uint32_t s = 0; s < S::kValueSteps; ++s)
#pragma unroll
            for (uint32_t e = 0; e < S::kValueRun; ++e) o[s][e] *= fade;
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                score[h][i] = __builtin_amdgcn_exp2f(score[h][i] - (base - P::kLift));
                l += score[h][i];
            }
        // the products with the values, 4 * kRun keys at a time
#pragma unroll
        for (uint32_t w = 0; w < S::kGroups; ++w) {
            piece p_hi, p_lo;
#pragma unroll
            for (uint32_t k = 0; k < S::kRun; ++k) {
                const float p = S::kRun == 8 ? score[k / 4][k % 4] : score[w][k];
                p_hi[k] = P::head(p);
                p_lo[k] = static_cast<T>(fmaxf(p - static_cast<float>(p_hi[k]), P::kLeast));
            }
#pragma unroll
            for (uint32_t s = 0; s < S::kValueSteps; ++s) {
                const uint32_t d = (s * 16 + col) * S::kValueRun;
                value_run v[S::kRun];
#pragma unroll
                for (uint32_t k = 0; k < S::kRun; ++k) {
                    const uint32_t h = S::kRun == 8 ? k / 4 : w, place = 4 * quad + k % 4;
                    v[k] = value_run{};
                    if ((FULL || d < a.head_dim) && t0 + 16 * h + place < limit[h])
                        v[k] = *reinterpret_cast<const value_run*>(values[h] + place * a.value_slot + d);
                }
#pragma unroll
                for (uint32_t e = 0; e < S::kValueRun; ++e) {
                    piece x;
#pragma unroll
                    for (uint32_t k = 0; k < S::kRun; ++k) x[k] = v[k][e];
                    o[s][e] = P::mma(x, p_hi, o[s][e]);
                    if (S::kRun == 8) o[s][e] = P::mma(x, p_lo, o[s][e]);
                }
            }
        }
    }

    l = column_sum(l);
    if (quad == 0) {
        lds_m[wave][col] = m;
        lds_l[wave][col] = l;
    }
#pragma unroll
    for (uint32_t s = 0; s < S::kValueSteps; ++s)
#pragma unroll
        for (uint32_t e = 0; e < S::kValueRun; ++e)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t d = (s * 16 + 4 * quad + i) * S::kValueRun + e;
                lds_o[wave][col][d] = o[s][e][i];
            }
    __syncthreads();
    // the item's sums: unnormalised, with their maximum and weight, or the row itself
    const bool whole = item.count == 1;
    for (uint32_t i = threadIdx.x; i < heads * DP; i += kThreads) {
        const uint32_t h = i / DP, d = i % DP;
        float top = -__builtin_inff();
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) top = fmaxf(top, lds_m[w][h]);
        const float base = top == -__builtin_inff() ? 0.0f : top;
        float sum = 0.0f, weight = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) {
            const float share = __builtin_amdgcn_exp2f(lds_m[w][h] - base);
            weight += share * lds_l[w][h];
            sum += share * lds_o[w][h][d];
        }
        if (d >= a.head_dim) continue;
        if (whole) {
            static_cast<T*>(a.out)[item.row * a.out_row + (head0 + h) * a.out_head + d] =
                from_float<T>(weight == 0.0f ? 0.0f : sum / weight);
        } else {
            float* dst = a.partials + (static_cast<uint64_t>(which) * a.heads + head0 + h) * (a.head_dim + 2);
            if (d == 0) dst[0] = top, dst[1] = weight;
            dst[2 + d] = sum;
        }
    }
}

// Rows of several items: the items' sums joined in their order.
template <typename T>
__global__ __launch_bounds__(256) void nz_attention_join_kernel(nz_attention_args a) {
    const nz_attention_item item = a.items[blockIdx.x];
    if (static_cast<uint32_t>(item.row) >= a.n_rows || item.index != 0 || item.count <= 1) return;
    const uint32_t step = a.head_dim + 2;
    for (uint32_t i = threadIdx.x; i < a.heads * a.head_dim; i += 256) {
        const uint32_t h = i / a.head_dim, d = i % a.head_dim;
        const float* src = a.partials + (static_cast<uint64_t>(blockIdx.x) * a.heads + h) * step;
        const uint64_t stride = static_cast<uint64_t>(a.heads) * step;
        float top = -__builtin_inff();
        for (int32_t k = 0; k < item.count; ++k) top = fmaxf(top, src[k * stride]);
        const float base = top == -__builtin_inff() ? 0.0f : top;
        float sum = 0.0f, weight = 0.0f;
        for (int32_t k = 0; k < item.count; ++k) {
            const float share = __builtin_amdgcn_exp2f(src[k * stride] - base);
            weight += share * src[k * stride + 1];
            sum += share * src[k * stride + 2 + d];
        }
        static_cast<T*>(a.out)[item.row * a.out_row + h * a.out_head + d] =
            from_float<T>(weight == 0.0f ? 0.0f : sum / weight);
    }
}

template <typename T, uint32_t DP>
void launch_attention_dim(const nz_attention_args& a, dim3 grid, hipStream_t stream) {
    if (a.head_dim == DP) hipLaunchKernelGGL((nz_attention_kernel<T, DP, true>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((nz_attention_kernel<T, DP, false>), grid, dim3(kThreads), 0, stream, a);
}

template <typename T>
void launch_attention(const nz_attention_args& a, hipStream_t stream) {
    const uint32_t group = a.heads / a.kv_heads;
    const dim3 grid(a.n_items * a.kv_heads * ((group + kHeads - 1) / kHeads));
    if (a.head_dim <= 64) launch_attention_dim<T, 64>(a, grid, stream);
    else if (a.head_dim <= 128) launch_attention_dim<T, 128>(a, grid, stream);
    else launch_attention_dim<T, 256>(a, grid, stream);
    hipLaunchKernelGGL(nz_attention_join_kernel<T>, dim3(a.n_items), dim3(256), 0, stream, a);
}

int launched(const char* what, char* message, size_t message_size) {
    const hipError_t rc = hipGetLastError();
    if (rc == hipSuccess) return 0;
    snprintf(message, message_size, "%s launch failed: %s", what, hipGetErrorString(rc));
    return -6;
}

}  // namespace

// The callers (capi_serving.cpp) have checked the arguments.

extern "C" int nz_hip_attention_plan(const int32_t* contexts, const int32_t* requests, uint32_t n_rows, uint32_t target,
                                     nz_attention_item* items, void* stream, char* message, size_t message_size) {
    hipLaunchKernelGGL(nz_attention_plan_kernel, dim3(1), dim3(kPlanThreads), 0, static_cast<hipStream_t>(stream),
                       contexts, requests, n_rows, target, items);
    return launched("attention plan", message, message_size);
}

extern "C" int nz_hip_attention(const nz_attention_args* args, void* stream, char* message, size_t message_size) {
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (args->type == NZ_BF16) launch_attention<bf16_t>(*args, st);
    else if (args->type == NZ_FP16) launch_attention<_Float16>(*args, st);
    else launch_attention<float>(*args, st);
    return launched("attention", message, message_size);
}
