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
// Of workgroups that decide on a request's drafts, a wavefront per row.
constexpr uint32_t kPickThreads = 512, kPickWaves = kPickThreads / 64, kPickEach = kChunk / kPickThreads;
// Chunks of a row that a thread weighs, at most.
constexpr uint32_t kMaxChunks = NZ_VERIFY_MAX_VOCAB / kChunk, kChunksEach = kMaxChunks / kPickThreads;
constexpr uint32_t kNone = 0xFFFFFFFFu;

// What is known of a chunk of a row: its largest logit, where that is first (of
// a greedy row), and the sum of the weights exp((x - top) / temperature).
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
    double weight;      // of the draft
};

__host__ __device__ __forceinline__ uint32_t chunks_of(uint32_t vocab) { return (vocab + kChunk - 1) / kChunk; }

// Weights are held times 2^60, so that the smallest that 64 bits hold beside a
// largest of 1 are normal numbers. Those of 2^-kReach and less are 0, as 64
// bits would round them.
constexpr double kUnit = 0x1p60;
constexpr double kReach = 1075.0;

// How a row's logits are weighed: exp((x - top) / temperature) where `top` is
// the largest, and the first of the largest alone where the temperature is not
// above 0.
struct Scale {
    double rate;        // log2(e) / temperature (an infinite one: so small that every number weighs as much); 0: greedy
    // The Taylor series of 2^f, (ln 2)^k / k!, kept in scalar registers (as
    // literals each takes two moves into vector registers).
    static constexpr uint32_t kTerms = 13;
    double series[kTerms];

    __device__ __forceinline__ explicit Scale(float temperature)
        : rate(temperature > 0.0f ? 1.44269504088896340736 / fmin(static_cast<double>(temperature), 1e300) : 0.0) {
        double term = kUnit;
#pragma unroll
        for (uint32_t k = 0; k < kTerms; ++k) {
            series[k] = term;
            term = term * 0.693147180559945309417 / (k + 1);
            asm("" : "+s"(series[k]));
        }
    }
    __device__ __forceinline__ bool greedy() const { return rate == 0.0; }
    // 2^y, y = (x - top) rate <= 0, to 2 units of the last place: y's whole
    // part, the low bits of a sum with 1.5 * 2^52, as the exponent, and the
    // series for the rest, |f| <= 1/2, whose next term is below 2^-52. The
    // library's exp takes four times as long, and most of the call's time was
    // spent in it. The cut is by y itself: past it the whole part would not
    // stay inside the exponent, however near x is to top.
    __device__ __forceinline__ double finite(float x, float top) const {
        const double y = (static_cast<double>(x) - static_cast<double>(top)) * rate;
        const double shifted = y + 0x1.8p52, f = y - (shifted - 0x1.8p52);
        double p = series[kTerms - 1];
#pragma unroll
        for (uint32_t k = kTerms - 1; k-- > 0;) p = fma(p, f, series[k]);
        vec<uint32_t, 2> bits = __builtin_bit_cast(vec<uint32_t, 2>, p);
        bits.y += __builtin_bit_cast(vec<uint32_t, 2>, shifted).x << 20;
        return y > -kReach ? __builtin_bit_cast(double, bits) : 0.0;
    }
    // the weights of some logits (NaN has none)
    template <uint32_t N>
    __device__ __forceinline__ void weigh(const float (&x)[N], float top, double (&w)[N]) const {
        if (top == __builtin_inff()) {
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) w[i] = x[i] == top ? kUnit : 0.0;
        } else {
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) w[i] = finite(x[i], top);
        }
    }
    __device__ __forceinline__ double operator()(float x, float top) const {
        double w[1];
        weigh({x}, top, w);
        return w[0];
    }
};

// NaN is no token's logit.
template <typename T>
__device__ __forceinline__ float logit(T x) {
    const float y = to_float(x);
    return y == y ? y : -__builtin_inff();
}

// Largest of a wavefront's values, NaN aside; the same in every lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_max(float v) {
    const int low = __float_as_int(-__builtin_inff());
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(low, __float_as_int(v), CTRL, ROWS, 0xF, false)));
}

__device__ __forceinline__ float wave_max(float v) {
    v = dpp_max<0x111, 0xF>(v);
    v = dpp_max<0x112, 0xF>(v);
    v = dpp_max<0x114, 0xF>(v);
    v = dpp_max<0x118, 0xF>(v);
    v = dpp_max<0x142, 0xA>(v);
    v = dpp_max<0x143, 0xC>(v);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Neighbouring elements from `v` on, wherever they lie in memory, with
// `none` past the end.
template <uint32_t N, typename T>
__device__ __forceinline__ void load_each(const T* src, uint32_t v, uint32_t end, T none, T (&x)[N]) {
    if (v + N <= end) {
        __builtin_memcpy(x, src + v, sizeof x);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) x[i] = v + i < end ? src[v + i] : none;
    }
}

template <typename T, uint32_t N>
__device__ __forceinline__ void load_logits(const nz_verify_args& a, uint32_t row, uint32_t v, float (&x)[N]) {
    T raw[N];
    load_each(static_cast<const T*>(a.logits) + static_cast<int64_t>(row) * a.logits_row, v, a.vocab,
              static_cast<T>(-__builtin_inff()), raw);
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) x[i] = logit(raw[i]);
}

__device__ __forceinline__ float temperature_of(const nz_verify_args& a, uint32_t request) {
    return a.temperature ? a.temperature[request] : 1.0f;
}

__device__ __forceinline__ uint32_t row_limit(const nz_verify_args& a, uint32_t request) {
    return min(static_cast<uint32_t>(max(a.starts[request], 0)), a.n_rows);
}

// The request whose rows hold `row` (kNone: none does) and its temperature, by
// a wavefront: 64 requests at a time, all of what is needed of them read at
// once, after a search among every 64th start where there are more.
__device__ __forceinline__ uint32_t request_of(const nz_verify_args& a, uint32_t row, float& temperature) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t low = 0, count = a.n_requests;
    while (count > 64) {
        const uint32_t step = (count + 63) / 64, at = lane * step;
        const uint64_t bits = __ballot(at < count && row_limit(a, low + at) <= row);
        if (bits == 0) return kNone;
        const uint32_t last = 63 - __builtin_clzll(bits);
        low += last * step;
        count = min(step, count - last * step);
    }
    const uint32_t request = low + min(lane, count - 1);
    const uint32_t begin = row_limit(a, request), end = row_limit(a, request + 1);
    const float mine = temperature_of(a, request);
    const uint64_t bits = __ballot(lane < count && begin <= row && row < end);
    if (bits == 0) return kNone;
    temperature = __shfl(mine, __builtin_ctzll(bits));
    return low + __builtin_ctzll(bits);
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// Sum over the workgroup, in a fixed order.
template <uint32_t WAVES>
__device__ __forceinline__ double block_sum(double v, double* lds) {
    v = wave_sum(v);
    __syncthreads();   // the last call's reads
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double sum = 0.0;
#pragma unroll
    for (uint32_t w = 0; w < WAVES; ++w) sum += lds[w];
    return sum;
}

// Largest logit, and where it is first, of two parts.
__device__ __forceinline__ void take_larger(Part& a, float top, uint32_t first) {
    if (top > a.top || (top == a.top && first < a.first)) a.top = top, a.first = first;
}

__device__ __forceinline__ void wave_largest(Part& a) {
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) take_larger(a, __shfl_xor(a.top, d), __shfl_xor(a.first, d));
}

// One chunk of one row. Bound by the vector units, some 20 instructions of 64
// bits a logit: 240 rows of 128256 fp32 logits in 38 us (3.3 TB/s; the units
// are busy 63 % of the time), 104 in bf16 in 16. Several chunks a workgroup,
// each read ahead, took as long, as did registers for eight wavefronts a SIMD.
template <typename T>
__global__ __launch_bounds__(kThreads) void nz_verify_rows_kernel(nz_verify_args a, Part* __restrict__ parts) {
    __shared__ float tops[kWaves];
    __shared__ uint32_t firsts[kWaves];
    __shared__ double sums[kWaves];
    const uint32_t row = blockIdx.y, v = blockIdx.x * kChunk + threadIdx.x * kEach;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T raw[kEach];
    load_each(static_cast<const T*>(a.logits) + static_cast<int64_t>(row) * a.logits_row, v, a.vocab,
              static_cast<T>(-__builtin_inff()), raw);
    float temperature;
    if (request_of(a, row, temperature) == kNone) return;
    const Scale scale(temperature);
    float x[kEach], top = -__builtin_inff();
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
        x[i] = to_float(raw[i]);
        top = fmaxf(top, x[i]);
    }
    top = wave_max(top);
    if (lane == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) top = fmaxf(top, tops[w]);
    Part part = {top, kNone, 0.0};
    if (scale.greedy()) {
#pragma unroll
        for (uint32_t i = kEach; i-- > 0;)
            if (x[i] == top && v + i < a.vocab) part.first = v + i;
        // (lanes hold rising tokens)
        const uint64_t bits = __ballot(part.first != kNone);
        const uint32_t first = __shfl(part.first, bits ? __builtin_ctzll(bits) : 0);
        if (lane == 0) firsts[wave] = first;
        __syncthreads();
        part.first = kNone;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) part.first = min(part.first, firsts[w]);
    } else if (top > -__builtin_inff()) {
        double w[kEach];
        scale.weigh(x, top, w);
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) part.sum += w[i];
        part.sum = block_sum<kWaves>(part.sum, sums);
    }
    if (threadIdx.x == 0) parts[static_cast<uint64_t>(row) * gridDim.x + blockIdx.x] = part;
}

// A row's largest logit, its first token and the sum of weights (of a greedy
// row: 1), by a wavefront; the same in every lane.
__device__ __forceinline__ Part row_of(const Part* parts, uint32_t chunks, const Scale& scale) {
    const uint32_t lane = threadIdx.x & 63;
    Part mine = {-__builtin_inff(), kNone, 0.0};
    if (lane < chunks) mine = parts[lane];
    Part row = mine;
    for (uint32_t c = lane + 64; c < chunks; c += 64) take_larger(row, parts[c].top, parts[c].first);
    wave_largest(row);
    row.sum = 0.0;
    if (row.top == -__builtin_inff()) return row;
    if (scale.greedy()) {
        row.sum = 1.0;
        return row;
    }
    row.sum = mine.sum * (scale(mine.top, row.top) / kUnit);
    for (uint32_t c = lane + 64; c < chunks; c += 64) row.sum += parts[c].sum * (scale(parts[c].top, row.top) / kUnit);
    row.sum = wave_sum(row.sum);
    return row;
}

// Accepts a request's drafts in turn, a wavefront per row; the result is the
// same in every thread. Probabilities are compared and subtracted times the
// row's sum of weights.
template <typename T, uint32_t WAVES>
__device__ Decision decide(const nz_verify_args& a, const Part* parts, uint32_t request, const Scale& scale) {
    __shared__ Decision rows[WAVES];
    __shared__ bool stops[WAVES];
    const uint32_t chunks = chunks_of(a.vocab), wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint32_t begin = row_limit(a, request), end = row_limit(a, request + 1);
    for (uint32_t r0 = begin; r0 < end; r0 += WAVES) {
        const uint32_t row = r0 + wave;
        __syncthreads();   // the last rows' reads
        if (row < end) {
            const int64_t draft = row + 1 < end ? a.tokens[row + 1] : -1;
            const bool known = static_cast<uint64_t>(draft) < a.vocab;
            float x = -__builtin_inff();
            double limit = 0.0;
            if (known) {
                x = logit(static_cast<const T*>(a.logits)[static_cast<int64_t>(row) * a.logits_row + draft]);
                limit = a.accept[row];
                if (a.draft_probs) limit *= static_cast<double>(a.draft_probs[static_cast<int64_t>(row) * a.draft_row + draft]);
            }
            Decision here = {row, row - begin, 0, kWhole, row_of(parts + static_cast<uint64_t>(row) * chunks, chunks, scale), 0.0};
            bool stop = true;
            if (known && here.whole.sum > 0.0) {
                here.refused = static_cast<uint32_t>(draft);
                here.kind = a.draft_probs ? kRest : kWithout;
                here.weight = scale.greedy() ? here.refused == here.whole.first : scale(x, here.whole.top);
                stop = !(limit * here.whole.sum < here.weight);
            }
            if (lane == 0) rows[wave] = here, stops[wave] = stop;
        }
        __syncthreads();
        for (uint32_t w = 0; w < WAVES && r0 + w < end; ++w)
            if (stops[w]) return rows[w];
    }
    return Decision{kNone, 0, 0, kWhole, {-__builtin_inff(), kNone, 0.0}, 0.0};
}

// The weights of neighbouring tokens of a decision's row, from `v` on;
// returns their sum.
template <typename T, uint32_t N>
__device__ __forceinline__ double weigh(const nz_verify_args& a, const Decision& d, Kind kind, const Scale& scale,
                                        uint32_t v, double (&w)[N]) {
    float x[N], q[N] = {};
    load_logits<T>(a, d.row, v, x);
    if (kind == kRest)
        load_each(a.draft_probs + static_cast<int64_t>(d.row) * a.draft_row, v, a.vocab, __builtin_inff(), q);
    if (!scale.greedy()) scale.weigh(x, d.whole.top, w);
    double sum = 0.0;
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
        if (scale.greedy()) w[i] = v + i == d.whole.first;
        if (kind == kWithout && v + i == d.refused) w[i] = 0.0;
        if (kind == kRest) {
            const double rest = w[i] - static_cast<double>(q[i]) * d.whole.sum;
            w[i] = rest > 0.0 ? rest : 0.0;
        }
        sum += w[i];
    }
    return sum;
}

// With draft probabilities, the decisions are made first: 5.3 us for 48
// requests of four drafts, latencies of the chunks' parts and of two
// reductions.
template <typename T>
__global__ __launch_bounds__(kPickThreads)
void nz_verify_decide_kernel(nz_verify_args a, const Part* __restrict__ parts, Decision* __restrict__ decisions) {
    const uint32_t request = blockIdx.x;
    const Scale scale(temperature_of(a, request));
    const Decision d = decide<T, kPickWaves>(a, parts, request, scale);
    if (threadIdx.x == 0) decisions[request] = d;
}

// Then the sums of max(p - q, 0) over the chunks of the row that a request's
// next token is picked from. Bound by memory: 48 rows of 128256 fp32 logits and
// as many probabilities in 11.5 us (4.3 TB/s). (When its workgroups decided
// each for itself, 17.)
template <typename T>
__global__ __launch_bounds__(kThreads)
void nz_verify_rest_kernel(nz_verify_args a, const Decision* __restrict__ decisions, double* __restrict__ rests) {
    __shared__ double sums[kWaves];
    const uint32_t request = blockIdx.y;
    const Decision d = decisions[request];
    if (d.kind != kRest) return;
    const Scale scale(temperature_of(a, request));
    double w[kEach];
    const double sum = block_sum<kWaves>(weigh<T>(a, d, kRest, scale, blockIdx.x * kChunk + threadIdx.x * kEach, w), sums);
    if (threadIdx.x == 0) rests[static_cast<uint64_t>(request) * gridDim.x + blockIdx.x] = sum;
}

// The next token of a request: the chunk in which the sum of weights passes
// the wanted share of all, then the token in it. Bound by latencies, the
// decision's among them: 7.6 us for one row, 10.7 for 32 requests of up to five
// drafts, 7.4 for 48 that are decided already.
template <typename T>
__global__ __launch_bounds__(kPickThreads)
void nz_verify_pick_kernel(nz_verify_args a, const Part* __restrict__ parts, const Decision* __restrict__ decisions,
                           const double* __restrict__ rests) {
    __shared__ double sums[kPickWaves], before_chunk, all_chunks;
    __shared__ uint32_t found, last;
    const uint32_t request = blockIdx.x, chunks = chunks_of(a.vocab), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Scale scale(temperature_of(a, request));
    const double share = a.sample[request];
    const Decision d = decisions ? decisions[request] : decide<T, kPickWaves>(a, parts, request, scale);
    const bool none = d.row == kNone || d.whole.sum == 0.0;
    if (threadIdx.x == 0) {
        a.accepted[request] = static_cast<int32_t>(d.accepted);
        if (none) a.next[request] = -1;
    }
    if (none) return;
    Kind kind = d.kind;
    double w[kPickEach];
    // sums of the threads before this one, in a fixed order
    const auto scan = [&](double v) {
        const double mine = v;
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
#pragma unroll
        for (uint32_t i = 0; i < kPickWaves; ++i)
            if (i < wave) before += sums[i];
        return before + v - mine;
    };
    const auto chunk_weight = [&](uint32_t c) -> double {
        if (scale.greedy()) return c == d.whole.first / kChunk;
        const Part part = parts[static_cast<uint64_t>(d.row) * chunks + c];
        return part.sum * (scale(part.top, d.whole.top) / kUnit);
    };
    // the first and the last of what the threads found (a wavefront's one atomic each: 4096 of them took 60 us)
    const auto note = [&](uint32_t first, uint32_t most) {
#pragma unroll
        for (uint32_t s = 1; s < 64; s <<= 1) {
            first = min(first, static_cast<uint32_t>(__shfl_xor(first, s)));
            most = max(most, static_cast<uint32_t>(__shfl_xor(most, s)));
        }
        if (lane == 0) atomicMin(&found, first), atomicMax(&last, most);
    };
    // without the draft refused: its chunk's sum less its weight, or, where that would cancel, anew
    const uint32_t hole = kind == kWithout ? d.refused / kChunk : kNone;
    double without = 0.0;
    if (kind == kWithout) {
        const double all = chunk_weight(hole), less = all - d.weight;
        without = 2.0 * less >= all
                      ? less
                      : block_sum<kPickWaves>(weigh<T>(a, d, kind, scale, hole * kChunk + threadIdx.x * kPickEach, w), sums);
    }
    // some neighbouring chunks a thread: their weights; from the row itself if the refusal leaves nothing
    const uint32_t each = (chunks + kPickThreads - 1) / kPickThreads, c0 = threadIdx.x * each;
    double weights[kChunksEach], before = 0.0;
    for (uint32_t turn = 0; turn < 2; ++turn) {
        double mine = 0.0;
#pragma unroll
        for (uint32_t i = 0; i < kChunksEach; ++i) {
            const uint32_t c = c0 + i;
            weights[i] = 0.0;
            if (i < each && c < chunks) {
                if (kind == kRest) {
                    weights[i] = rests[static_cast<uint64_t>(request) * chunks + c];
                } else if (kind == kWithout && c == hole) {
                    weights[i] = without;
                } else {
                    weights[i] = chunk_weight(c);
                }
            }
            mine += weights[i];
        }
        before = scan(mine);
        if (threadIdx.x == kPickThreads - 1) all_chunks = before + mine;
        __syncthreads();
        if (all_chunks > 0.0) break;
        kind = kWhole;
    }
    const double wanted = share * all_chunks;
    double upto = before;
    uint32_t mine_first = kNone, mine_last = 0;
#pragma unroll
    for (uint32_t i = 0; i < kChunksEach; ++i) {
        upto += weights[i];
        if (weights[i] > 0.0) {
            mine_last = c0 + i;
            if (upto > wanted) mine_first = min(mine_first, c0 + i);
        }
    }
    note(mine_first, mine_last);
    __syncthreads();
    const uint32_t chunk = found != kNone ? found : last;
#pragma unroll
    for (uint32_t i = 0; i < kChunksEach; ++i) {
        if (i < each && c0 + i == chunk) before_chunk = before;
        before += weights[i];
    }
    // the token: the first with a weight at which the sum passes what is wanted, or the chunk's last
    const uint32_t v = chunk * kChunk + threadIdx.x * kPickEach;
    double sum = scan(weigh<T>(a, d, kind, scale, v, w));   // its barriers come before before_chunk is read
    sum += before_chunk;
    mine_first = kNone, mine_last = 0;
#pragma unroll
    for (uint32_t i = 0; i < kPickEach; ++i) {
        sum += w[i];
        if (w[i] > 0.0) {
            mine_last = v + i;
            if (sum > wanted) mine_first = min(mine_first, v + i);
        }
    }
    note(mine_first, mine_last);
    __syncthreads();
    if (threadIdx.x == 0) a.next[request] = found != kNone ? found : last;
}

template <typename T>
void launch_verify(const nz_verify_args& a, hipStream_t stream) {
    const uint32_t chunks = chunks_of(a.vocab);
    Part* const parts = static_cast<Part*>(a.scratch);
    Decision* const decisions = reinterpret_cast<Decision*>(parts + static_cast<uint64_t>(a.n_rows) * chunks);
    double* const rests = reinterpret_cast<double*>(decisions + a.n_requests);
    const bool decided = a.draft_probs && a.n_rows;
    if (a.n_rows) hipLaunchKernelGGL(nz_verify_rows_kernel<T>, dim3(chunks, a.n_rows), dim3(kThreads), 0, stream, a, parts);
    if (decided) {
        hipLaunchKernelGGL(nz_verify_decide_kernel<T>, dim3(a.n_requests), dim3(kPickThreads), 0, stream, a, parts, decisions);
        hipLaunchKernelGGL(nz_verify_rest_kernel<T>, dim3(chunks, a.n_requests), dim3(kThreads), 0, stream, a, decisions, rests);
    }
    hipLaunchKernelGGL(nz_verify_pick_kernel<T>, dim3(a.n_requests), dim3(kPickThreads), 0, stream, a, parts,
                       decided ? decisions : nullptr, rests);
}

}  // namespace

// The callers (capi_serving.cpp) have checked the arguments.

extern "C" uint64_t nz_hip_verify_scratch(uint32_t n_rows, uint32_t n_requests, uint32_t vocab) {
    static_assert(sizeof(Part) == 16 && sizeof(Decision) % 8 == 0, "scratch of 8-byte numbers");
    return static_cast<uint64_t>(n_rows) * chunks_of(vocab) * sizeof(Part) +
           n_requests * (sizeof(Decision) + static_cast<uint64_t>(chunks_of(vocab)) * sizeof(double));
}

extern "C" int nz_hip_verify_drafts(const nz_verify_args* args, void* stream, char* message, size_t message_size) {
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (args->type == NZ_BF16) launch_verify<bf16_t>(*args, st);
    else if (args->type == NZ_FP16) launch_verify<_Float16>(*args, st);
    else launch_verify<float>(*args, st);
    return launched("verification", message, message_size);
}
