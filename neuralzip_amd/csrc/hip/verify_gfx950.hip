// verify_gfx950.hip -- drafted tokens against the model's probabilities, from
// given random numbers, and the token after the last one kept
// (nz_verify_drafts).
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "neuralzip_hip.h"
#include "serving_types.h"

namespace {

// A row's vocabulary is cut into chunks, which one workgroup takes each.
constexpr uint32_t kThreads = 256, kWaves = kThreads / 64, kChunk = NZ_VERIFY_CHUNK, kEach = kChunk / kThreads;
constexpr uint32_t kPickThreads = 1024, kPickWaves = kPickThreads / 64, kPickEach = kChunk / kPickThreads;
constexpr uint32_t kNone = 0xFFFFFFFFu;

// What is known of a chunk of a row: its largest logit, where that is first,
// and the sum of the weights exp((x - top) / temperature).
struct Part {
    float top;
    uint32_t first;
    double sum;
};

// What the next token of a request is picked from: a row's probabilities, those
// without the draft that was refused in it, or what the draft's own
// probabilities leave of them.
enum Kind : uint32_t { kWhole, kWithout, kRest };

// What was decided for a request: the row that the next token is picked from,
// how many drafts were accepted before it, and the draft refused in it.
struct Decision {
    uint32_t row;       // kNone: the request has no row
    uint32_t accepted;
    uint32_t refused;
    Kind kind;
    Part whole;         // of the row
};

__host__ __device__ __forceinline__ uint32_t chunks_of(uint32_t vocab) { return (vocab + kChunk - 1) / kChunk; }

// NaN is no token's logit.
template <typename T>
__device__ __forceinline__ float logit(T x) {
    const float y = to_float(x);
    return y == y ? y : -__builtin_inff();
}

// A logit's weight where `top` is the largest one, which may be infinite.
__device__ __forceinline__ double weight_of(float x, float top, double temperature) {
    if (x == -__builtin_inff()) return 0.0;
    if (x == top) return 1.0;
    return exp((static_cast<double>(x) - static_cast<double>(top)) / temperature);
}

__device__ __forceinline__ float temperature_of(const nz_verify_args& a, uint32_t request) {
    return a.temperature ? fminf(a.temperature[request], 3.4e38f) : 1.0f;
}

__device__ __forceinline__ uint32_t row_limit(const nz_verify_args& a, uint32_t request) {
    return min(static_cast<uint32_t>(max(a.starts[request], 0)), a.n_rows);
}

// The request whose rows hold `row` (kNone: none does), by a wavefront: the
// last start that is no larger, 64 of them read at a time.
__device__ uint32_t request_of(const nz_verify_args& a, uint32_t row) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t low = 0, count = a.n_requests;   // of starts that may be the one
    while (count > 1) {
        const uint32_t step = (count + 63) / 64, at = lane * step;
        const bool below = at < count && row_limit(a, low + at) <= row;
        const uint64_t bits = __ballot(below);
        if (bits == 0) return kNone;
        const uint32_t last = 63 - __builtin_clzll(bits);
        low += last * step;
        count = min(step, count - last * step);
    }
    return row_limit(a, low) <= row && row < row_limit(a, low + 1) ? low : kNone;
}

// Sum over the workgroup, in a fixed order.
template <uint32_t WAVES>
__device__ __forceinline__ double block_sum(double v, double* lds) {
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    __syncthreads();   // the last call's reads
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double sum = 0.0;
#pragma unroll
    for (uint32_t w = 0; w < WAVES; ++w) sum += lds[w];
    return sum;
}

// One chunk of one row.
template <typename T>
__global__ __launch_bounds__(kThreads) void nz_verify_rows_kernel(nz_verify_args a, Part* __restrict__ parts) {
    __shared__ float tops[kWaves];
    __shared__ uint32_t firsts[kWaves];
    __shared__ double sums[kWaves];
    const uint32_t row = blockIdx.y, v0 = blockIdx.x * kChunk, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T* src = static_cast<const T*>(a.logits) + static_cast<int64_t>(row) * a.logits_row;
    float x[kEach];
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
        const uint32_t v = v0 + i * kThreads + threadIdx.x;
        x[i] = v < a.vocab ? logit(src[v]) : -__builtin_inff();
    }
    const uint32_t request = request_of(a, row);
    if (request == kNone) return;
    const float temperature = temperature_of(a, request);
    float top = x[0];
#pragma unroll
    for (uint32_t i = 1; i < kEach; ++i) top = fmaxf(top, x[i]);
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    if (lane == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) top = fmaxf(top, tops[w]);
    uint32_t first = kNone;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
        const uint32_t v = v0 + i * kThreads + threadIdx.x;
        if (x[i] == top && v < a.vocab) first = min(first, v);
    }
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) first = min(first, static_cast<uint32_t>(__shfl_xor(first, d)));
    if (lane == 0) firsts[wave] = first;
    double sum = 0.0;
    if (temperature > 0.0f) {
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) sum += weight_of(x[i], top, temperature);
    }
    sum = block_sum<kWaves>(sum, sums);
    if (threadIdx.x == 0) {
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) first = min(first, firsts[w]);
        parts[static_cast<uint64_t>(row) * gridDim.x + blockIdx.x] = Part{top, first, sum};
    }
}

// A row's largest logit, its first token and the sum of weights (of a greedy
// row: 1), by a wavefront; the same in every lane.
__device__ __forceinline__ Part row_of(const Part* parts, uint32_t chunks, float temperature) {
    const uint32_t lane = threadIdx.x & 63;
    Part row = {-__builtin_inff(), kNone, 0.0};
    for (uint32_t c = lane; c < chunks; c += 64) {
        const Part part = parts[c];
        if (part.top > row.top || (part.top == row.top && part.first < row.first)) row.top = part.top, row.first = part.first;
    }
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const float top = __shfl_xor(row.top, d);
        const uint32_t first = __shfl_xor(row.first, d);
        if (top > row.top || (top == row.top && first < row.first)) row.top = top, row.first = first;
    }
    if (row.top == -__builtin_inff()) return row;
    if (!(temperature > 0.0f)) {
        row.sum = 1.0;
        return row;
    }
    for (uint32_t c = lane; c < chunks; c += 64) row.sum += parts[c].sum * weight_of(parts[c].top, row.top, temperature);
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) row.sum += __shfl_xor(row.sum, d);
    return row;
}

// A token's weight in a row.
template <typename T>
__device__ __forceinline__ double weight_at(const nz_verify_args& a, uint32_t row, const Part& whole, float temperature,
                                            uint32_t v) {
    if (!(temperature > 0.0f)) return v == whole.first ? 1.0 : 0.0;
    return weight_of(logit(static_cast<const T*>(a.logits)[static_cast<int64_t>(row) * a.logits_row + v]), whole.top,
                     temperature);
}

// Accepts a request's drafts in turn, a wavefront per row; the result is the
// same in every thread.
template <typename T, uint32_t WAVES>
__device__ Decision decide(const nz_verify_args& a, const Part* parts, uint32_t request) {
    __shared__ Decision rows[WAVES];
    __shared__ bool stops[WAVES];
    const uint32_t chunks = chunks_of(a.vocab), wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint32_t begin = row_limit(a, request), end = row_limit(a, request + 1);
    const float temperature = temperature_of(a, request);
    for (uint32_t r0 = begin; r0 < end; r0 += WAVES) {
        const uint32_t row = r0 + wave;
        __syncthreads();   // the last rows' reads
        if (row < end) {
            Decision here = {row, row - begin, 0, kWhole, row_of(parts + static_cast<uint64_t>(row) * chunks, chunks, temperature)};
            bool stop = true;
            const int64_t draft = row + 1 < end ? a.tokens[row + 1] : -1;
            if (static_cast<uint64_t>(draft) < a.vocab && here.whole.sum > 0.0) {
                here.refused = static_cast<uint32_t>(draft);
                here.kind = a.draft_probs ? kRest : kWithout;
                const double p = weight_at<T>(a, row, here.whole, temperature, here.refused) / here.whole.sum;
                const double q = a.draft_probs
                                     ? static_cast<double>(a.draft_probs[static_cast<int64_t>(row) * a.draft_row + draft])
                                     : 1.0;
                stop = !(a.accept[row] * q < p);
            }
            if (lane == 0) rows[wave] = here, stops[wave] = stop;
        }
        __syncthreads();
        for (uint32_t w = 0; w < WAVES && r0 + w < end; ++w)
            if (stops[w]) return rows[w];
    }
    return Decision{kNone, 0, 0, kWhole, {-__builtin_inff(), kNone, 0.0}};
}

// With draft probabilities: the sums of max(p - q, 0) over the chunks of the
// row that a request's next token is picked from.
template <typename T>
__global__ __launch_bounds__(kThreads)
void nz_verify_rest_kernel(nz_verify_args a, const Part* __restrict__ parts, double* __restrict__ rests) {
    __shared__ double sums[kWaves];
    const uint32_t request = blockIdx.y, v0 = blockIdx.x * kChunk;
    const Decision d = decide<T, kWaves>(a, parts, request);
    if (d.kind != kRest) return;
    const float temperature = temperature_of(a, request);
    const float* q = a.draft_probs + static_cast<int64_t>(d.row) * a.draft_row;
    double sum = 0.0;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
        const uint32_t v = v0 + i * kThreads + threadIdx.x;
        if (v < a.vocab) {
            const double rest = weight_at<T>(a, d.row, d.whole, temperature, v) / d.whole.sum - static_cast<double>(q[v]);
            sum += rest > 0.0 ? rest : 0.0;
        }
    }
    sum = block_sum<kWaves>(sum, sums);
    if (threadIdx.x == 0) rests[static_cast<uint64_t>(request) * gridDim.x + blockIdx.x] = sum;
}

// The next token of a request: the chunk in which the sum of weights passes
// the wanted share of all, then the token in it.
template <typename T>
__global__ __launch_bounds__(kPickThreads)
void nz_verify_pick_kernel(nz_verify_args a, const Part* __restrict__ parts, const double* __restrict__ rests) {
    __shared__ double sums[kPickWaves], before_chunk, chunk_total;
    __shared__ uint32_t found, last;
    const uint32_t request = blockIdx.x, chunks = chunks_of(a.vocab), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Decision d = decide<T, kPickWaves>(a, parts, request);
    const bool none = d.row == kNone || d.whole.sum == 0.0;
    if (threadIdx.x == 0) {
        a.accepted[request] = static_cast<int32_t>(d.accepted);
        if (none) a.next[request] = -1;
    }
    if (none) return;
    const float temperature = temperature_of(a, request);
    Kind kind = d.kind;
    const auto token_weight = [&](uint32_t v) {
        const double p = weight_at<T>(a, d.row, d.whole, temperature, v) / d.whole.sum;
        if (kind == kWhole) return p;
        if (kind == kWithout) return v == d.refused ? 0.0 : p;
        const double rest = p - static_cast<double>(a.draft_probs[static_cast<int64_t>(d.row) * a.draft_row + v]);
        return rest > 0.0 ? rest : 0.0;
    };
    // the weights of kPickEach neighbours of a chunk, and their sum
    double w[kPickEach];
    const auto chunk_weights = [&](uint32_t chunk) {
        double sum = 0.0;
#pragma unroll
        for (uint32_t i = 0; i < kPickEach; ++i) {
            const uint32_t v = chunk * kChunk + threadIdx.x * kPickEach + i;
            w[i] = v < a.vocab ? token_weight(v) : 0.0;
            sum += w[i];
        }
        return sum;
    };
    // inclusive prefix sums, in a fixed order
    const auto scan = [&](double v) {
#pragma unroll
        for (uint32_t s = 1; s < 64; s <<= 1) {
            const double below = __shfl_up(v, s);
            if (lane >= s) v += below;
        }
        __syncthreads();   // the last reads of the shared numbers
        if (lane == 63) sums[wave] = v;
        if (threadIdx.x == 0) found = kNone, last = 0;
        __syncthreads();
        double before = 0.0;
        for (uint32_t i = 0; i < wave; ++i) before += sums[i];
        return before + v;
    };
    const uint32_t hole = kind == kWithout ? d.refused / kChunk : kNone;   // its sum is taken anew
    double without = 0.0;
    if (kind == kWithout) without = block_sum<kPickWaves>(chunk_weights(hole), sums);
    // a thread per chunk: their weights; from the row itself if the refusal leaves nothing
    double mine = 0.0, upto = 0.0, total = 0.0;
    for (uint32_t turn = 0; turn < 2; ++turn) {
        mine = 0.0;
        const uint32_t c = threadIdx.x;
        if (c < chunks) {
            const Part part = parts[static_cast<uint64_t>(d.row) * chunks + c];
            if (kind == kRest) mine = rests[static_cast<uint64_t>(request) * chunks + c];
            else if (kind == kWithout && c == hole) mine = without;
            else if (!(temperature > 0.0f)) mine = c == d.whole.first / kChunk ? 1.0 : 0.0;
            else mine = part.sum * weight_of(part.top, d.whole.top, temperature) / d.whole.sum;
        }
        upto = scan(mine);
        if (threadIdx.x == kPickThreads - 1) chunk_total = upto;
        __syncthreads();
        total = chunk_total;
        if (total > 0.0) break;
        kind = kWhole;
    }
    const double wanted = a.sample[request] * total;
    if (mine > 0.0) {
        atomicMax(&last, threadIdx.x);
        if (upto > wanted) atomicMin(&found, threadIdx.x);
    }
    __syncthreads();
    const uint32_t chunk = found != kNone ? found : last;
    if (threadIdx.x == chunk) before_chunk = upto - mine;
    // the token: the first with a weight at which the sum passes what is wanted, or the chunk's last
    mine = chunk_weights(chunk);
    upto = scan(mine);
    double sum = before_chunk + upto - mine;
#pragma unroll
    for (uint32_t i = 0; i < kPickEach; ++i) {
        sum += w[i];
        const uint32_t v = chunk * kChunk + threadIdx.x * kPickEach + i;
        if (w[i] > 0.0) {
            atomicMax(&last, v);
            if (sum > wanted) atomicMin(&found, v);
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) a.next[request] = found != kNone ? found : last;
}

template <typename T>
void launch_verify(const nz_verify_args& a, hipStream_t stream) {
    const uint32_t chunks = chunks_of(a.vocab);
    Part* const parts = static_cast<Part*>(a.scratch);
    double* const rests = reinterpret_cast<double*>(parts + static_cast<uint64_t>(a.n_rows) * chunks);
    if (a.n_rows) hipLaunchKernelGGL(nz_verify_rows_kernel<T>, dim3(chunks, a.n_rows), dim3(kThreads), 0, stream, a, parts);
    if (a.n_rows && a.draft_probs)
        hipLaunchKernelGGL(nz_verify_rest_kernel<T>, dim3(chunks, a.n_requests), dim3(kThreads), 0, stream, a, parts, rests);
    hipLaunchKernelGGL(nz_verify_pick_kernel<T>, dim3(a.n_requests), dim3(kPickThreads), 0, stream, a, parts, rests);
}

}  // namespace

// The callers (capi_serving.cpp) have checked the arguments.

extern "C" uint64_t nz_hip_verify_scratch(uint32_t n_rows, uint32_t n_requests, uint32_t vocab) {
    return (static_cast<uint64_t>(n_rows) * sizeof(Part) + static_cast<uint64_t>(n_requests) * 8) * chunks_of(vocab);
}

extern "C" int nz_hip_verify_drafts(const nz_verify_args* args, void* stream, char* message, size_t message_size) {
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (args->type == NZ_BF16) launch_verify<bf16_t>(*args, st);
    else if (args->type == NZ_FP16) launch_verify<_Float16>(*args, st);
    else launch_verify<float>(*args, st);
    return launched("verification", message, message_size);
}
