// experts_gfx950.hip -- a mixture-of-experts layer for a few tokens: the
// router's choice (nz_route_experts) and the chosen experts' gated products
// (nz_expert_mlp).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "attention_types.h"
#include "neuralzip_hip.h"
#include "serving_types.h"

namespace {

// ------------------------------------------------------------------ router

constexpr uint32_t kRouteThreads = 1024, kRouteWaves = kRouteThreads / 64;

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// One token: its products with every expert's row, summed in 64 bits so that
// the choice does not depend on their order, then each expert's place among
// them by counting those before it.
template <typename T, typename W>
__global__ __launch_bounds__(kRouteThreads) void nz_route_kernel(nz_route_args a) {
    constexpr uint32_t kRun = run_of<W>();
    __shared__ double score[NZ_EXPERT_MAX], chance[NZ_EXPERT_MAX];
    __shared__ double sums[kRouteWaves], tops[kRouteWaves];
    extern __shared__ __align__(16) float x[];
    const uint32_t token = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T* src = static_cast<const T*>(a.x) + static_cast<int64_t>(token) * a.x_row;
    for (uint32_t d = threadIdx.x; d < a.hidden; d += kRouteThreads) x[d] = to_float(src[d]);
    __syncthreads();
    for (uint32_t e = wave; e < a.experts; e += kRouteWaves) {
        const W* row = static_cast<const W*>(a.weight) + static_cast<uint64_t>(e) * a.hidden;
        double sum = 0.0;
        for (uint32_t d = lane * kRun; d < a.hidden; d += 64 * kRun) {
            const vec<W, kRun> w = *reinterpret_cast<const vec<W, kRun>*>(row + d);
#pragma unroll
            for (uint32_t i = 0; i < kRun; ++i)
                sum = fma(static_cast<double>(to_float(static_cast<W>(w[i]))), static_cast<double>(x[d + i]), sum);
        }
        sum = wave_sum(sum);
        if (lane == 0) score[e] = sum;
    }
    __syncthreads();
    // (threads past the experts take part in the sums)
    const uint32_t e = threadIdx.x;
    double mine = e < a.experts ? score[e] : -INFINITY;
    if (mine != mine) mine = -INFINITY;
    double top = mine;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) top = fmax(top, __shfl_xor(top, d));
    if (lane == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kRouteWaves; ++w) top = fmax(top, tops[w]);
    double share;
    if (a.scoring == NZ_ROUTE_SIGMOID) {
        share = 1.0 / (1.0 + exp(-mine));
    } else {
        share = mine == top ? 1.0 : exp(mine - top);   // (infinite scores are equal)
        const double sum = wave_sum(e < a.experts ? share : 0.0);
        if (lane == 0) sums[wave] = sum;
        __syncthreads();
        double all = 0.0;
#pragma unroll
        for (uint32_t w = 0; w < kRouteWaves; ++w) all += sums[w];
        share /= all;
    }
    double rank = a.scoring == NZ_ROUTE_SIGMOID ? share : mine;
    if (a.bias != nullptr && e < a.experts) rank += static_cast<double>(a.bias[e]);
    if (rank != rank) rank = -INFINITY;
    __syncthreads();
    if (e < a.experts) score[e] = rank, chance[e] = share;
    __syncthreads();
    int32_t* const ids = a.ids + static_cast<uint64_t>(token) * a.top_k;
    __shared__ double picked[NZ_ROUTE_MAX_TOP];
    if (e < a.experts) {
        uint32_t before = 0;
        for (uint32_t j = 0; j < a.experts; ++j) {
            const double other = score[j];
            before += other > rank || (other == rank && j < e);
        }
        if (before < a.top_k) {
            ids[before] = static_cast<int32_t>(e);
            picked[before] = share;
        }
    }
    __syncthreads();
    if (threadIdx.x < a.top_k) {
        double all = 1.0;
        if (a.normalize) {
            all = 0.0;
            for (uint32_t k = 0; k < a.top_k; ++k) all += picked[k];
        }
        a.weights[static_cast<uint64_t>(token) * a.top_k + threadIdx.x] =
            all > 0.0 ? static_cast<float>(picked[threadIdx.x] / all * static_cast<double>(a.scale)) : 0.0f;
    }
}

// ----------------------------------------------------------------- experts

// Tokens of one pass over the experts' weights, at most: four blocks of columns.
constexpr uint32_t kTokens = NZ_EXPERT_TOKENS, kBlocks = kTokens / 16;
constexpr uint32_t kUpThreads = 256, kUpWaves = kUpThreads / 64;
constexpr uint32_t kDownThreads = 512, kDownWaves = kDownThreads / 64;
// Elements of the outputs that a workgroup makes for its tokens.
constexpr uint32_t kRows = 16;

// Which of a pass's tokens chose each expert, and the experts that any did, in
// rising order.
struct Choice {
    unsigned long long tokens[NZ_EXPERT_MAX];   // by expert, a bit per token
    uint32_t active[NZ_EXPERT_MAX];
    uint32_t n_active;
    uint32_t waves[kDownWaves];
    int32_t ids[kTokens * NZ_ROUTE_MAX_TOP];    // -1: none
};

__device__ __forceinline__ int64_t id_at(const nz_expert_args& a, uint64_t i) {
    return a.id_bytes == 8 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
}

template <uint32_t THREADS>
__device__ __forceinline__ void choose(const nz_expert_args& a, uint32_t token0, uint32_t tokens, Choice& c) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint32_t e = threadIdx.x; e < a.experts; e += THREADS) c.tokens[e] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < tokens * a.top_k; i += THREADS) {
        const uint64_t e = static_cast<uint64_t>(id_at(a, static_cast<uint64_t>(token0) * a.top_k + i));
        if (e < a.experts) atomicOr(&c.tokens[e], 1ull << i / a.top_k);
        c.ids[i] = e < a.experts ? static_cast<int32_t>(e) : -1;
    }
    __syncthreads();
    uint32_t before = 0;
    for (uint32_t e0 = 0; e0 < a.experts; e0 += THREADS) {
        const uint32_t e = e0 + threadIdx.x;
        const bool live = e < a.experts && c.tokens[e] != 0;
        const uint64_t bits = __ballot(live);
        if (lane == 0) c.waves[wave] = __popcll(bits);
        __syncthreads();
        uint32_t at = before;
        for (uint32_t w = 0; w < THREADS / 64; ++w) {
            if (w < wave) at += c.waves[w];
            before += c.waves[w];
        }
        if (live) c.active[at + __popcll(bits & ((1ull << lane) - 1))] = e;
        __syncthreads();
    }
    if (threadIdx.x == 0) c.n_active = before;
    __syncthreads();
}

// The place of an expert among a token's choices (the first, if it is there twice).
__device__ __forceinline__ uint32_t place_of(const nz_expert_args& a, const Choice& c, uint32_t token, uint32_t expert) {
    uint32_t place = 0;
    for (uint32_t k = a.top_k; k-- > 0;)
        if (c.ids[token * a.top_k + k] == static_cast<int32_t>(expert)) place = k;
    return place;
}

// A token's weight for an expert: the sum over its choices.
__device__ __forceinline__ float weight_of(const nz_expert_args& a, const Choice& c, uint32_t token0, uint32_t token,
                                           uint32_t expert) {
    const float* weights = a.weights + static_cast<uint64_t>(token0 + token) * a.top_k;
    float sum = 0.0f;
    for (uint32_t k = 0; k < a.top_k; ++k)
        if (c.ids[token * a.top_k + k] == static_cast<int32_t>(expert)) sum += weights[k];
    return sum;
}

__device__ __forceinline__ float activate(uint32_t kind, float x) {
    if (kind == NZ_EXPERT_SILU) return x / (1.0f + expf(-x));
    return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
}

// The gated activations of one expert's tokens, for kRows of its inner
// elements: act(gate x) * (up x), in 32 bits. Weight rows are the rows of the
// matrix instructions and tokens their columns; the wavefronts share the depth.
template <typename T>
__global__ __launch_bounds__(kUpThreads) void nz_expert_up_kernel(nz_expert_args a, float* __restrict__ acts,
                                                                  uint32_t* __restrict__ counters, uint32_t n_counters) {
    using P = Piece<T>;
    using piece = typename P::type;
    constexpr uint32_t kDepth = 4 * P::kRun;
    __shared__ Choice choice;
    __shared__ uint32_t list[kTokens];
    __shared__ float sums[kUpWaves][2][kTokens][kRows + 1];
    const uint32_t lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0)
        for (uint32_t i = threadIdx.x; i < n_counters; i += kUpThreads) counters[i] = 0;
    const uint32_t token0 = blockIdx.z * kTokens, tokens = min(kTokens, a.tokens - token0);
    choose<kUpThreads>(a, token0, tokens, choice);
    if (blockIdx.y >= choice.n_active) return;
    const uint32_t expert = choice.active[blockIdx.y];
    const uint64_t mask = choice.tokens[expert];
    const uint32_t count = __popcll(mask), blocks = (count + 15) / 16;
    if (threadIdx.x < 64 && mask >> threadIdx.x & 1) list[__popcll(mask & ((1ull << threadIdx.x) - 1))] = threadIdx.x;
    __syncthreads();
    const uint32_t row0 = blockIdx.x * kRows, row = min(row0 + col, a.inter - 1);
    const T* const gate = static_cast<const T*>(a.gate_up) + expert * a.gate_expert + row * a.gate_row;
    const T* const up = gate + a.inter * a.gate_row;
    const T* x[kBlocks];
#pragma unroll
    for (uint32_t b = 0; b < kBlocks; ++b)
        x[b] = static_cast<const T*>(a.x) + (token0 + (b * 16 + col < count ? list[b * 16 + col] : list[0])) * a.x_row;
    f32x4 sum[2][kBlocks] = {};
#pragma unroll 4
    for (uint32_t d0 = wave * kDepth; d0 < a.hidden; d0 += kUpWaves * kDepth) {
        const uint32_t d = d0 + quad * P::kRun;
        piece g = {}, u = {};
        if (d < a.hidden) {
            g = *reinterpret_cast<const piece*>(gate + d);
            u = *reinterpret_cast<const piece*>(up + d);
        }
#pragma unroll
        for (uint32_t b = 0; b < kBlocks; ++b) {
            if (b < blocks) {
                piece y = {};
                if (d < a.hidden && b * 16 + col < count) y = *reinterpret_cast<const piece*>(x[b] + d);
                sum[0][b] = P::mma(g, y, sum[0][b]);
                sum[1][b] = P::mma(u, y, sum[1][b]);
            }
        }
    }
#pragma unroll
    for (uint32_t b = 0; b < kBlocks; ++b)
        if (b < blocks)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                sums[wave][0][b * 16 + col][4 * quad + i] = sum[0][b][i];
                sums[wave][1][b * 16 + col][4 * quad + i] = sum[1][b][i];
            }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < count * kRows; i += kUpThreads) {
        const uint32_t c = i / kRows, r = i % kRows;
        float g = 0.0f, u = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kUpWaves; ++w) g += sums[w][0][c][r], u += sums[w][1][c][r];
        const uint32_t token = list[c];
        if (row0 + r < a.inter)
            acts[(static_cast<uint64_t>(token0 + token) * a.top_k + place_of(a, choice, token, expert)) * a.inter + row0 + r] =
                activate(a.activation, g) * u;
    }
}

// Activations as two pieces whose sum they are to 16 or 22 bits: one rounding
// to a weight's type would err as much as the result's own. fp16 pieces are
// those of the activations divided by 2^lift, so that neither large nor small
// ones leave fp16's range.
template <typename T>
__device__ __forceinline__ int split(const float (&x)[Piece<T>::kRun], typename Piece<T>::type& hi,
                                     typename Piece<T>::type& lo) {
    constexpr uint32_t kRun = Piece<T>::kRun;
    int lift = 0;
    if (sizeof(T) == 4) {
#pragma unroll
        for (uint32_t i = 0; i < kRun; ++i) hi[i] = static_cast<T>(x[i]);
        return 0;
    }
    if (std::is_same<T, _Float16>::value) {
        float most = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kRun; ++i) most = fmaxf(most, fabsf(x[i]));
        most = column_max(most);
        lift = __builtin_amdgcn_frexp_expf(most);
    }
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i) {
        const float y = std::is_same<T, _Float16>::value ? __builtin_amdgcn_ldexpf(x[i], -lift) : x[i];
        hi[i] = Piece<T>::head(y);
        const float head = static_cast<float>(hi[i]), rest = y - head;
        lo[i] = static_cast<T>(fabsf(head) < __builtin_inff() ? rest : 0.0f);
    }
    return lift;
}

// kRows elements of the outputs: over the chosen experts and their inner
// elements, each wavefront a share of them in a row, with the tokens that
// chose an expert as columns; the columns of an expert are added to their
// tokens' sums, times the weights, when it ends. `splits` workgroups share the
// experts; the last to arrive adds their sums in order.
template <typename T>
__global__ __launch_bounds__(kDownThreads) void nz_expert_down_kernel(nz_expert_args a, const float* __restrict__ acts,
                                                                      float* __restrict__ partials,
                                                                      uint32_t* __restrict__ counters, uint32_t splits) {
    using P = Piece<T>;
    using piece = typename P::type;
    constexpr uint32_t kDepth = 4 * P::kRun;
    __shared__ Choice choice;
    __shared__ __align__(16) float sums[kDownWaves][kTokens][kRows];
    __shared__ uint32_t list[kDownWaves][kTokens];
    __shared__ uint32_t last;
    const uint32_t lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t token0 = blockIdx.z * kTokens, tokens = min(kTokens, a.tokens - token0);
    for (uint32_t i = threadIdx.x; i < kDownWaves * kTokens * kRows; i += kDownThreads) (&sums[0][0][0])[i] = 0.0f;
    choose<kDownThreads>(a, token0, tokens, choice);
    const uint32_t row0 = blockIdx.x * kRows, row = min(row0 + col, a.hidden - 1);
    const uint32_t steps = (a.inter + kDepth - 1) / kDepth;
    const uint64_t all = static_cast<uint64_t>(choice.n_active) * steps;
    const uint32_t shares = splits * kDownWaves, mine = blockIdx.y * kDownWaves + wave;
    uint64_t at = all * mine / shares;
    const uint64_t until = all * (mine + 1) / shares;
    while (at < until) {
        const uint32_t n = static_cast<uint32_t>(at / steps), expert = choice.active[n];
        const uint32_t s0 = static_cast<uint32_t>(at % steps);
        const uint32_t s1 = static_cast<uint32_t>(min(static_cast<uint64_t>(steps), s0 + (until - at)));
        const uint64_t mask = choice.tokens[expert];
        const uint32_t count = __popcll(mask), blocks = (count + 15) / 16;
        if (mask >> lane & 1) list[wave][__popcll(mask & ((1ull << lane) - 1))] = lane;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const T* const down = static_cast<const T*>(a.down) + expert * a.down_expert + row * a.down_row;
        const float* x[kBlocks];
        uint32_t token[kBlocks];
#pragma unroll
        for (uint32_t b = 0; b < kBlocks; ++b) {
            token[b] = b * 16 + col < count ? list[wave][b * 16 + col] : 0;
            x[b] = acts;
            if (b * 16 + col < count)
                x[b] += (static_cast<uint64_t>(token0 + token[b]) * a.top_k + place_of(a, choice, token[b], expert)) * a.inter;
        }
        f32x4 sum[kBlocks] = {};
#pragma unroll 2
        for (uint32_t s = s0; s < s1; ++s) {
            const uint32_t d = s * kDepth + quad * P::kRun;
            piece w = {};
            if (d < a.inter) w = *reinterpret_cast<const piece*>(down + d);
#pragma unroll
            for (uint32_t b = 0; b < kBlocks; ++b) {
                if (b < blocks) {
                    float y[P::kRun] = {};
                    if (d < a.inter && b * 16 + col < count) load_floats<P::kRun>(x[b] + d, y);
                    piece hi, lo;
                    const int lift = split<T>(y, hi, lo);
                    f32x4 part = std::is_same<T, _Float16>::value ? f32x4{} : sum[b];
                    part = P::mma(w, hi, part);
                    if (sizeof(T) == 2) part = P::mma(w, lo, part);
                    if (std::is_same<T, _Float16>::value) {
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i) sum[b][i] += __builtin_amdgcn_ldexpf(part[i], lift);
                    } else {
                        sum[b] = part;
                    }
                }
            }
        }
#pragma unroll
        for (uint32_t b = 0; b < kBlocks; ++b) {
            if (b * 16 + col < count) {
                const float weight = weight_of(a, choice, token0, token[b], expert);
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) sums[wave][token[b]][4 * quad + i] += weight * sum[b][i];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the list's reads
        at += s1 - s0;
    }
    __syncthreads();
    T* const out = static_cast<T*>(a.out);
    const uint64_t plane = static_cast<uint64_t>(a.tokens) * a.hidden;
    const rsrc_t scratch = device_buffer(partials);
    for (uint32_t i = threadIdx.x; i < tokens * kRows / 4; i += kDownThreads) {
        const uint32_t t = i / (kRows / 4), r = i % (kRows / 4) * 4;
        if (row0 + r >= a.hidden) continue;
        f32x4 sum = {};
#pragma unroll
        for (uint32_t w = 0; w < kDownWaves; ++w) sum += *reinterpret_cast<const f32x4*>(&sums[w][t][r]);
        if (splits == 1) store_row(out + (token0 + t) * a.out_row + row0 + r, sum, 1.0f);
        else put_four(scratch, 4 * static_cast<uint32_t>(blockIdx.y * plane + (token0 + t) * static_cast<uint64_t>(a.hidden) + row0 + r), sum);
    }
    if (splits == 1) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wavefront's stores have arrived
    __syncthreads();
    if (threadIdx.x == 0)
        last = __hip_atomic_fetch_add(counters + blockIdx.z * gridDim.x + blockIdx.x, 1u, __ATOMIC_RELAXED,
                                      __HIP_MEMORY_SCOPE_AGENT) + 1 == splits;
    __syncthreads();
    if (!last) return;
    for (uint32_t i = threadIdx.x; i < tokens * kRows / 4; i += kDownThreads) {
        const uint32_t t = i / (kRows / 4), r = i % (kRows / 4) * 4;
        if (row0 + r >= a.hidden) continue;
        f32x4 sum = {};
        for (uint32_t k = 0; k < splits; ++k)
            sum += get_four(scratch, 4 * static_cast<uint32_t>(k * plane + (token0 + t) * static_cast<uint64_t>(a.hidden) + row0 + r));
        store_row(out + (token0 + t) * a.out_row + row0 + r, sum, 1.0f);
    }
}

uint32_t splits_of(uint32_t tokens, uint32_t hidden) {
    const uint32_t groups = (hidden + kRows - 1) / kRows * ((tokens + kTokens - 1) / kTokens);
    return std::min(8u, std::max(1u, (512 + groups - 1) / groups));
}

template <typename T>
void launch_experts(const nz_expert_args& a, hipStream_t stream) {
    const uint32_t passes = (a.tokens + kTokens - 1) / kTokens, splits = splits_of(a.tokens, a.hidden);
    const uint32_t rows = (a.hidden + kRows - 1) / kRows;
    float* const acts = static_cast<float*>(a.scratch);
    float* const partials = acts + static_cast<uint64_t>(a.tokens) * a.top_k * a.inter;
    uint32_t* const counters = reinterpret_cast<uint32_t*>(
        partials + (splits > 1 ? static_cast<uint64_t>(splits) * a.tokens * a.hidden : 0));
    const uint32_t most = std::min(a.experts, std::min(a.tokens, kTokens) * a.top_k);   // experts of a pass
    hipLaunchKernelGGL(nz_expert_up_kernel<T>, dim3((a.inter + kRows - 1) / kRows, most, passes), dim3(kUpThreads), 0,
                       stream, a, acts, counters, splits > 1 ? rows * passes : 0);
    hipLaunchKernelGGL(nz_expert_down_kernel<T>, dim3(rows, splits, passes), dim3(kDownThreads), 0, stream, a, acts,
                       partials, counters, splits);
}

template <typename T>
void launch_route(const nz_route_args& a, hipStream_t stream) {
    if (a.weight_type == NZ_FP32)
        hipLaunchKernelGGL((nz_route_kernel<T, float>), dim3(a.tokens), dim3(kRouteThreads), a.hidden * sizeof(float), stream, a);
    else
        hipLaunchKernelGGL((nz_route_kernel<T, T>), dim3(a.tokens), dim3(kRouteThreads), a.hidden * sizeof(float), stream, a);
}

}  // namespace

// The callers (capi_serving.cpp) have checked the arguments.

extern "C" int nz_hip_route_experts(const nz_route_args* args, void* stream, char* message, size_t message_size) {
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (args->type == NZ_BF16) launch_route<bf16_t>(*args, st);
    else if (args->type == NZ_FP16) launch_route<_Float16>(*args, st);
    else launch_route<float>(*args, st);
    return launched("routing", message, message_size);
}

extern "C" uint64_t nz_hip_expert_scratch(uint32_t tokens, uint32_t hidden, uint32_t inter, uint32_t top_k) {
    const uint64_t splits = splits_of(tokens, hidden), rows = (hidden + kRows - 1) / kRows;
    return (static_cast<uint64_t>(tokens) * top_k * inter + splits * tokens * hidden +
            rows * ((tokens + kTokens - 1) / kTokens)) * 4;
}

extern "C" int nz_hip_expert_mlp(const nz_expert_args* args, void* stream, char* message, size_t message_size) {
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (args->type == NZ_BF16) launch_experts<bf16_t>(*args, st);
    else if (args->type == NZ_FP16) launch_experts<_Float16>(*args, st);
    else launch_experts<float>(*args, st);
    return launched("experts", message, message_size);
}
