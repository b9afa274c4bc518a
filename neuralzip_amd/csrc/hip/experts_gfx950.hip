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

constexpr uint32_t kScoreThreads = 256, kScoreWaves = kScoreThreads / 64;

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// Eight neighbouring elements, wherever they lie in memory.
template <typename T>
__device__ __forceinline__ void load_eight(const T* src, float (&x)[8]) {
    T raw[8];
    __builtin_memcpy(raw, src, sizeof raw);
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) x[i] = to_float(raw[i]);
}

// Tokens' products with the experts' rows, a wavefront each, summed in 64 bits
// so that the choice does not depend on their order. (Both steps in one
// workgroup per token took 22 us for one token of 2048 elements and 128
// experts, which one compute unit multiplied; this 4.6, the latency of one
// row, and as much for 32 tokens of 4096 elements and 8.)
template <typename T, typename W>
__global__ __launch_bounds__(kScoreThreads) void nz_route_scores_kernel(nz_route_args a) {
    const uint32_t token = blockIdx.y, lane = threadIdx.x & 63, e = blockIdx.x * kScoreWaves + (threadIdx.x >> 6);
    if (e >= a.experts) return;
    const T* src = static_cast<const T*>(a.x) + static_cast<int64_t>(token) * a.x_row;
    const W* row = static_cast<const W*>(a.weight) + static_cast<uint64_t>(e) * a.hidden;
    double sums[2] = {};
#pragma unroll 4
    for (uint32_t d = lane * 8; d < a.hidden; d += 512) {
        float x[8], w[8];
        load_eight(src + d, x);
        load_runs(row + d, run_of<W>(), w);
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) sums[i % 2] = fma(static_cast<double>(w[i]), static_cast<double>(x[i]), sums[i % 2]);
    }
    const double sum = wave_sum(sums[0] + sums[1]);
    if (lane == 0) static_cast<double*>(a.scratch)[static_cast<uint64_t>(token) * a.experts + e] = sum;
}

// Whole numbers in the order of the values, NaN below all of them.
__device__ __forceinline__ int64_t order_of(double x) {
    const int64_t bits = __builtin_bit_cast(int64_t, x + 0.0);   // (-0 is 0)
    return x != x ? INT64_MIN : bits < 0 ? bits ^ INT64_MAX : bits;
}

// One token's choice, `parts` threads per expert: its place is the number of
// those before it, which they count together. (128 experts: 4.7 us,
// 5.5 with a thread per expert.)
__global__ __launch_bounds__(NZ_EXPERT_MAX) void nz_route_choice_kernel(nz_route_args a, uint32_t parts) {
    constexpr uint32_t kMaxWaves = NZ_EXPERT_MAX / 64;
    __shared__ double scores[NZ_EXPERT_MAX], sums[kMaxWaves], picked[NZ_ROUTE_MAX_TOP];
    __shared__ int64_t orders[NZ_EXPERT_MAX];
    const uint32_t token = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const uint32_t e = threadIdx.x / parts, part = threadIdx.x % parts;
    const bool live = e < a.experts, first = live && part == 0, sigmoid = a.scoring == NZ_ROUTE_SIGMOID;
    double mine = -INFINITY, rank = -INFINITY, share = 0.0;
    if (live) {
        mine = static_cast<const double*>(a.scratch)[static_cast<uint64_t>(token) * a.experts + e];
        if (sigmoid) share = 1.0 / (1.0 + exp(-mine));
        rank = sigmoid ? share : mine;
        if (a.bias != nullptr) rank += static_cast<double>(a.bias[e]);
        if (mine != mine) mine = -INFINITY, share = 0.0;   // NaN has no weight
    }
    const int64_t order = order_of(rank);
    if (first) scores[e] = mine, orders[e] = order;
    __syncthreads();
    uint32_t before = 0;
    double top = -INFINITY;
#pragma unroll 4
    for (uint32_t j = part; j < a.experts; j += parts) {
        const int64_t other = orders[j];
        before += other > order || (other == order && j < e);
        if (!sigmoid) top = fmax(top, scores[j]);
    }
    for (uint32_t d = 1; d < parts; d <<= 1) {
        before += __shfl_xor(before, d);
        top = fmax(top, __shfl_xor(top, d));
    }
    if (!sigmoid) {
        share = mine == top ? 1.0 : exp(mine - top);   // (infinite scores are equal)
        if (!a.normalize) {   // the chosen ones' sum divides them otherwise
            const double sum = wave_sum(first ? share : 0.0);
            if (lane == 0) sums[wave] = sum;
            __syncthreads();
            double all = 0.0;
            for (uint32_t w = 0; w < waves; ++w) all += sums[w];
            share /= all;
        }
    }
    if (first && before < a.top_k) {
        a.ids[static_cast<uint64_t>(token) * a.top_k + before] = static_cast<int32_t>(e);
        picked[before] = share;
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
constexpr uint32_t kRows = 16, kDownRows = 32;
// Pieces of a weight's row that a lane asks for before it multiplies any: a
// wavefront's are neighbours, whole lines of the memory.
constexpr uint32_t kBatch = 4;
// Workgroups that share a part of the outputs, at most.
constexpr uint32_t kMaxSplits = 8;

// Which of a pass's tokens chose each expert, and the experts that any did, in
// rising order. In a workgroup's dynamic LDS, as long as the layer needs.
struct Choice {
    unsigned long long* tokens;   // by expert, a bit per token
    uint32_t* active;
    int32_t* ids;                 // tokens x top_k, -1: none
    uint32_t n_active;

    static __host__ __device__ uint32_t bytes(uint32_t experts, uint32_t choices) {
        return (12 * experts + 4 * choices + 15) / 16 * 16;
    }
    __device__ Choice(unsigned char* lds, uint32_t experts)
        : tokens(reinterpret_cast<unsigned long long*>(lds)), active(reinterpret_cast<uint32_t*>(lds + 8 * experts)),
          ids(reinterpret_cast<int32_t*>(lds + 12 * experts)), n_active(0) {}
};

__device__ __forceinline__ int64_t id_at(const nz_expert_args& a, uint64_t i) {
    return a.id_bytes == 8 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
}

template <uint32_t THREADS>
__device__ __forceinline__ void choose(const nz_expert_args& a, uint32_t token0, uint32_t tokens, Choice& c) {
    __shared__ uint32_t waves[THREADS / 64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = tokens * a.top_k;
    const uint64_t first = static_cast<uint64_t>(token0) * a.top_k;
    uint64_t id = threadIdx.x < n ? static_cast<uint64_t>(id_at(a, first + threadIdx.x)) : 0;
    for (uint32_t e = threadIdx.x; e < a.experts; e += THREADS) c.tokens[e] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
        if (i != threadIdx.x) id = static_cast<uint64_t>(id_at(a, first + i));
        if (id < a.experts) atomicOr(&c.tokens[id], 1ull << i / a.top_k);
        c.ids[i] = id < a.experts ? static_cast<int32_t>(id) : -1;
    }
    __syncthreads();
    for (uint32_t e0 = 0; e0 < a.experts; e0 += THREADS) {
        const uint32_t e = e0 + threadIdx.x;
        const bool live = e < a.experts && c.tokens[e] != 0;
        const uint64_t bits = __ballot(live);
        if (lane == 0) waves[wave] = __popcll(bits);
        __syncthreads();
        uint32_t at = c.n_active;
#pragma unroll
        for (uint32_t w = 0; w < THREADS / 64; ++w) {
            if (w < wave) at += waves[w];
            c.n_active += waves[w];
        }
        if (live) c.active[at + __popcll(bits & ((1ull << lane) - 1))] = e;
        __syncthreads();
    }
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
// matrix instructions and tokens their columns, in up to NB blocks; the
// wavefronts share the depth. Bound by the weights' way from memory: 8 experts
// of 14336 x 4096 bf16 elements for 32 tokens in 365 us (5.1 TB/s); 8 of 768 x
// 2048 for one token in 13.4 (3.7), of which some 3.5 go by before the choice
// is known. (With batches of 8 pieces that layer took 40.9 us instead of 36.6,
// with registers for four wavefronts a SIMD the wide one 654 instead of 546.)
template <typename T, uint32_t NB>
__global__ __launch_bounds__(kUpThreads) void nz_expert_up_kernel(nz_expert_args a, float* __restrict__ acts,
                                                                  uint32_t* __restrict__ counters, uint32_t n_counters) {
    using P = Piece<T>;
    using piece = typename P::type;
    constexpr uint32_t kDepth = 4 * P::kRun;
    extern __shared__ __align__(16) unsigned char lds[];
    __shared__ uint32_t list[kTokens];
    __shared__ float sums[kUpWaves][2][16 * NB][kRows + 1];
    const uint32_t lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0)
        for (uint32_t i = threadIdx.x; i < n_counters; i += kUpThreads) counters[i] = 0;
    const uint32_t token0 = blockIdx.z * kTokens, tokens = min(kTokens, a.tokens - token0);
    Choice choice(lds, a.experts);
    choose<kUpThreads>(a, token0, tokens, choice);
    if (blockIdx.y >= choice.n_active) return;
    const uint32_t expert = choice.active[blockIdx.y];
    const uint64_t mask = choice.tokens[expert];
    const uint32_t count = __popcll(mask), blocks = __builtin_amdgcn_readfirstlane((count + 15) / 16);
    if (threadIdx.x < 64 && mask >> threadIdx.x & 1) list[__popcll(mask & ((1ull << threadIdx.x) - 1))] = threadIdx.x;
    __syncthreads();
    const uint32_t row0 = blockIdx.x * kRows, row = min(row0 + col, a.inter - 1);
    const T* const gate = static_cast<const T*>(a.gate_up) + expert * a.gate_expert + row * a.gate_row;
    const T* const up = gate + a.inter * a.gate_row;
    const T* x[NB];
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b)
        x[b] = static_cast<const T*>(a.x) + (token0 + list[b * 16 + col < count ? b * 16 + col : 0]) * a.x_row;
    f32x4 sum[2][NB] = {};
    // weights are asked for a batch ahead
    piece g[kBatch], u[kBatch];
    const auto fetch_weights = [&](uint32_t d0) {
#pragma unroll
        for (uint32_t j = 0; j < kBatch; ++j) {
            const uint32_t d = d0 + j * kDepth + quad * P::kRun;
            g[j] = u[j] = piece{};
            if (d < a.hidden) {
                g[j] = *reinterpret_cast<const piece*>(gate + d);
                u[j] = *reinterpret_cast<const piece*>(up + d);
            }
        }
    };
    constexpr uint32_t kStep = kUpWaves * kBatch * kDepth;
    fetch_weights(wave * kBatch * kDepth);
    for (uint32_t d0 = wave * kBatch * kDepth; d0 < a.hidden; d0 += kStep) {
        piece y[NB][kBatch], g_now[kBatch], u_now[kBatch];
#pragma unroll
        for (uint32_t j = 0; j < kBatch; ++j) g_now[j] = g[j], u_now[j] = u[j];
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
            for (uint32_t j = 0; j < kBatch; ++j) {
                const uint32_t d = d0 + j * kDepth + quad * P::kRun;
                y[b][j] = piece{};
                if (d < a.hidden && b * 16 + col < count) y[b][j] = *reinterpret_cast<const piece*>(x[b] + d);
            }
        fetch_weights(d0 + kStep);
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b)
            if (NB == 1 || b < blocks)
#pragma unroll
                for (uint32_t j = 0; j < kBatch; ++j) {
                    sum[0][b] = P::mma(g_now[j], y[b][j], sum[0][b]);
                    sum[1][b] = P::mma(u_now[j], y[b][j], sum[1][b]);
                }
    }
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b)
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
// ones leave fp16's range, whatever is infinite beside them. Beside a head the
// rest has its sign and is kept from being 0 (which errs by at most 2^-23 of the
// largest of the 32), so that an infinite weight or activation is infinite in
// both products; an activation below 2^-24 of the largest is all rest, and may
// be 0.
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
        most = fminf(column_max(most), 0x1.fffffep127f);
        lift = __builtin_amdgcn_frexp_expf(most);
    }
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i) {
        const float y = std::is_same<T, _Float16>::value ? __builtin_amdgcn_ldexpf(x[i], -lift) : x[i];
        hi[i] = Piece<T>::head(y);
        const float head = static_cast<float>(hi[i]);
        lo[i] = static_cast<T>(copysignf(__builtin_amdgcn_fmed3f(fabsf(y - head), fabsf(head), Piece<T>::kLeast), y));
    }
    return lift;
}

// kDownRows elements of the outputs: over the chosen experts and their inner
// elements, each wavefront a share of them in a row, with the tokens that
// chose an expert as columns; the columns of an expert are added to their
// tokens' sums, times the weights, when it ends. `splits` workgroups share the
// experts; the last to arrive adds their sums in order. Bound by the weights'
// way from memory and, for few tokens, by the latencies of the choice and of
// the last sums: 211 us (4.5 TB/s) and 12.3 us for the layers above. All of it
// is read again for every kTokens tokens: 65 tokens of the wide layer take 963 us,
// where 64 take 652.
template <typename T, uint32_t NB>
__global__ __launch_bounds__(kDownThreads) void nz_expert_down_kernel(nz_expert_args a, const float* __restrict__ acts,
                                                                      float* __restrict__ partials,
                                                                      uint32_t* __restrict__ counters, uint32_t splits) {
    using P = Piece<T>;
    using piece = typename P::type;
    constexpr uint32_t kDepth = 4 * P::kRun, kTiles = kDownRows / 16;
    constexpr bool kLifted = std::is_same<T, _Float16>::value;
    extern __shared__ __align__(16) unsigned char lds[];
    __shared__ __align__(16) float sums[kDownWaves][16 * NB][kDownRows];
    __shared__ uint32_t list[kDownWaves][kTokens];
    __shared__ uint32_t last;
    const uint32_t lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t token0 = blockIdx.z * kTokens, tokens = min(kTokens, a.tokens - token0);
    for (uint32_t i = threadIdx.x; i < kDownWaves * 16 * NB * kDownRows; i += kDownThreads) (&sums[0][0][0])[i] = 0.0f;
    Choice choice(lds, a.experts);
    choose<kDownThreads>(a, token0, tokens, choice);
    const uint32_t row0 = blockIdx.x * kDownRows;
    const uint32_t steps = (a.inter + kBatch * kDepth - 1) / (kBatch * kDepth);
    const uint32_t all = choice.n_active * steps, shares = splits * kDownWaves, mine = blockIdx.y * kDownWaves + wave;
    const uint32_t each = all / shares, more = all % shares;
    uint32_t at = mine * each + min(mine, more);
    const uint32_t until = at + each + (mine < more);
    while (at < until) {
        const uint32_t n = at / steps, s0 = at - n * steps, s1 = min(steps, s0 + (until - at));
        const uint32_t expert = __builtin_amdgcn_readfirstlane(choice.active[n]);
        const uint64_t mask = choice.tokens[expert];
        const uint32_t count = __popcll(mask), blocks = __builtin_amdgcn_readfirstlane((count + 15) / 16);
        if (mask >> lane & 1) list[wave][__popcll(mask & ((1ull << lane) - 1))] = lane;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const T* down[kTiles];
#pragma unroll
        for (uint32_t t = 0; t < kTiles; ++t)
            down[t] = static_cast<const T*>(a.down) + expert * a.down_expert + min(row0 + 16 * t + col, a.hidden - 1) * a.down_row;
        const float* x[NB];
        uint32_t token[NB];
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            token[b] = b * 16 + col < count ? list[wave][b * 16 + col] : 0;
            x[b] = acts;
            if (b * 16 + col < count)
                x[b] += (static_cast<uint64_t>(token0 + token[b]) * a.top_k + place_of(a, choice, token[b], expert)) * a.inter;
        }
        f32x4 sum[kTiles][NB] = {};
        piece next[kTiles][kBatch];   // weights, asked for a batch ahead
        const auto fetch_weights = [&](uint32_t s) {
#pragma unroll
            for (uint32_t t = 0; t < kTiles; ++t)
#pragma unroll
                for (uint32_t j = 0; j < kBatch; ++j) {
                    const uint32_t d = (s * kBatch + j) * kDepth + quad * P::kRun;
                    next[t][j] = piece{};
                    if (s < s1 && d < a.inter) next[t][j] = *reinterpret_cast<const piece*>(down[t] + d);
                }
        };
        fetch_weights(s0);
        for (uint32_t s = s0; s < s1; ++s) {
            piece w[kTiles][kBatch];
#pragma unroll
            for (uint32_t t = 0; t < kTiles; ++t)
#pragma unroll
                for (uint32_t j = 0; j < kBatch; ++j) w[t][j] = next[t][j];
            fetch_weights(s + 1);
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b)
                if (NB == 1 || b < blocks) {
                    float y[kBatch][P::kRun] = {};
#pragma unroll
                    for (uint32_t j = 0; j < kBatch; ++j) {
                        const uint32_t d = (s * kBatch + j) * kDepth + quad * P::kRun;
                        if (d < a.inter && b * 16 + col < count) load_floats<P::kRun>(x[b] + d, y[j]);
                    }
#pragma unroll
                    for (uint32_t j = 0; j < kBatch; ++j) {
                        piece hi, lo;
                        const int lift = split<T>(y[j], hi, lo);
#pragma unroll
                        for (uint32_t t = 0; t < kTiles; ++t) {
                            f32x4 part = kLifted ? f32x4{} : sum[t][b];
                            part = P::mma(w[t][j], hi, part);
                            if (sizeof(T) == 2) part = P::mma(w[t][j], lo, part);
                            if (kLifted) {
#pragma unroll
                                for (uint32_t i = 0; i < 4; ++i) sum[t][b][i] += __builtin_amdgcn_ldexpf(part[i], lift);
                            } else {
                                sum[t][b] = part;
                            }
                        }
                    }
                }
        }
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            if (b * 16 + col < count) {
                const float weight = weight_of(a, choice, token0, token[b], expert);
#pragma unroll
                for (uint32_t t = 0; t < kTiles; ++t) {
                    f32x4* const to = reinterpret_cast<f32x4*>(&sums[wave][token[b]][16 * t + 4 * quad]);
                    *to += weight * sum[t][b];
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the list's reads
        at += s1 - s0;
    }
    __syncthreads();
    T* const out = static_cast<T*>(a.out);
    const uint64_t plane = static_cast<uint64_t>(a.tokens) * a.hidden;
    const rsrc_t scratch = device_buffer(partials);
    const auto place = [&](uint32_t split, uint32_t t, uint32_t r) {
        return 4 * static_cast<uint32_t>(split * plane + (token0 + t) * static_cast<uint64_t>(a.hidden) + row0 + r);
    };
    for (uint32_t i = threadIdx.x; i < tokens * kDownRows / 4; i += kDownThreads) {
        const uint32_t t = i / (kDownRows / 4), r = i % (kDownRows / 4) * 4;
        if (row0 + r >= a.hidden) continue;
        f32x4 sum = {};
#pragma unroll
        for (uint32_t w = 0; w < kDownWaves; ++w) sum += *reinterpret_cast<const f32x4*>(&sums[w][t][r]);
        if (splits == 1) store_row(out + (token0 + t) * a.out_row + row0 + r, sum, 1.0f);
        else put_four(scratch, place(blockIdx.y, t, r), sum);
    }
    if (splits == 1) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wavefront's stores have arrived
    __syncthreads();
    if (threadIdx.x == 0)
        last = __hip_atomic_fetch_add(counters + blockIdx.z * gridDim.x + blockIdx.x, 1u, __ATOMIC_RELAXED,
                                      __HIP_MEMORY_SCOPE_AGENT) + 1 == splits;
    __syncthreads();
    if (!last) return;
    for (uint32_t i = threadIdx.x; i < tokens * kDownRows / 4; i += kDownThreads) {
        const uint32_t t = i / (kDownRows / 4), r = i % (kDownRows / 4) * 4;
        if (row0 + r >= a.hidden) continue;
        f32x4 part[kMaxSplits], sum = {};
#pragma unroll
        for (uint32_t k = 0; k < kMaxSplits; ++k) part[k] = get_four(scratch, place(min(k, splits - 1), t, r));
#pragma unroll
        for (uint32_t k = 0; k < kMaxSplits; ++k)
            if (k < splits) sum += part[k];
        store_row(out + (token0 + t) * a.out_row + row0 + r, sum, 1.0f);
    }
}

uint32_t down_groups(uint32_t hidden) { return (hidden + kDownRows - 1) / kDownRows; }

// Workgroups that share a part of the outputs: the fewest for which the rounds
// of one workgroup a compute unit (its registers leave room for no second) are
// at most a tenth longer than for the best number. (16 experts of 1096 x 520
// fp32 elements: 23 us with 8, the last 24 of 280 workgroups alone, and 18 with
// 7.)
uint32_t splits_of(uint32_t tokens, uint32_t hidden) {
    constexpr uint32_t kUnits = 256;
    const uint32_t groups = down_groups(hidden) * ((tokens + kTokens - 1) / kTokens);
    const auto rounds = [&](uint32_t splits) { return (groups * splits + kUnits - 1) / kUnits / static_cast<double>(splits); };
    double best = rounds(1);
    for (uint32_t s = 2; s <= kMaxSplits; ++s) best = std::min(best, rounds(s));
    uint32_t splits = 1;
    while (rounds(splits) > 1.1 * best) ++splits;
    return splits;
}

template <typename T, uint32_t NB>
void launch_blocks(const nz_expert_args& a, hipStream_t stream) {
    const uint32_t passes = (a.tokens + kTokens - 1) / kTokens, splits = splits_of(a.tokens, a.hidden);
    const uint32_t groups = down_groups(a.hidden);
    float* const acts = static_cast<float*>(a.scratch);
    float* const partials = acts + static_cast<uint64_t>(a.tokens) * a.top_k * a.inter;
    uint32_t* const counters = reinterpret_cast<uint32_t*>(
        partials + (splits > 1 ? static_cast<uint64_t>(splits) * a.tokens * a.hidden : 0));
    const uint32_t choices = std::min(a.tokens, kTokens) * a.top_k, most = std::min(a.experts, choices);   // of a pass
    const uint32_t lds = Choice::bytes(a.experts, choices);
    hipLaunchKernelGGL((nz_expert_up_kernel<T, NB>), dim3((a.inter + kRows - 1) / kRows, most, passes), dim3(kUpThreads),
                       lds, stream, a, acts, counters, splits > 1 ? groups * passes : 0);
    hipLaunchKernelGGL((nz_expert_down_kernel<T, NB>), dim3(groups, splits, passes), dim3(kDownThreads), lds, stream, a,
                       acts, partials, counters, splits);
}

template <typename T>
void launch_experts(const nz_expert_args& a, hipStream_t stream) {
    if (a.tokens <= 16) launch_blocks<T, 1>(a, stream);
    else if (a.tokens <= 32) launch_blocks<T, 2>(a, stream);
    else launch_blocks<T, kBlocks>(a, stream);
}

template <typename T>
void launch_route(const nz_route_args& a, hipStream_t stream) {
    const dim3 grid((a.experts + kScoreWaves - 1) / kScoreWaves, a.tokens);
    if (a.weight_type == NZ_FP32)
        hipLaunchKernelGGL((nz_route_scores_kernel<T, float>), grid, dim3(kScoreThreads), 0, stream, a);
    else
        hipLaunchKernelGGL((nz_route_scores_kernel<T, T>), grid, dim3(kScoreThreads), 0, stream, a);
    uint32_t parts = 1;
    while (parts < 8 && a.experts * parts * 2 <= NZ_EXPERT_MAX) parts *= 2;
    hipLaunchKernelGGL(nz_route_choice_kernel, dim3(a.tokens), dim3((a.experts * parts + 63) / 64 * 64), 0, stream, a, parts);
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
    const uint64_t splits = splits_of(tokens, hidden);
    return (static_cast<uint64_t>(tokens) * top_k * inter + splits * tokens * hidden +
            static_cast<uint64_t>(down_groups(hidden)) * ((tokens + kTokens - 1) / kTokens)) * 4;
}

extern "C" int nz_hip_expert_mlp(const nz_expert_args* args, void* stream, char* message, size_t message_size) {
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (args->type == NZ_BF16) launch_experts<bf16_t>(*args, st);
    else if (args->type == NZ_FP16) launch_experts<_Float16>(*args, st);
    else launch_experts<float>(*args, st);
    return launched("experts", message, message_size);
}
