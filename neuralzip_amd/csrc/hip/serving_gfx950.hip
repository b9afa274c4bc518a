// serving_gfx950.hip -- gfx950 kernels of a serving step around the decoded
// weights: pages of the step's tokens (nz_pages_*), head norms, rotation and
// the store into the pages (nz_rotary_store), and the logits' adjustments
// (nz_adjust_logits). The attention over the pages is in attention_gfx950.hip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdint.h>
#include <stdio.h>

#include "neuralzip_hip.h"
#include "serving_types.h"

namespace {

// ------------------------------------------------------------------ pages

// Workgroups are as wide as a step of so many requests needs (a strip of
// requests at a time): one wavefront needs no barriers between wavefronts.
constexpr uint32_t kPagesThreads = 1024;
// Tokens (or pages to release) that one workgroup writes before the work is
// shared among several.
constexpr uint32_t kPagesShare = 2048, kPagesGroups = 128;

// Inclusive saturating prefix sums over the workgroup of N values at once;
// total receives the sums.
template <uint32_t THREADS, int N>
__device__ __forceinline__ void block_scan(uint32_t (&v)[N], uint32_t (&total)[N], uint32_t (*lds)[THREADS / 64]) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_scan(v[i]);
    if (THREADS == 64) {
#pragma unroll
        for (int i = 0; i < N; ++i) total[i] = last_lane(v[i]);
        return;
    }
    __syncthreads();   // the last call's reads
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (lane == 63) lds[i][wave] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        uint32_t before = 0, sum = 0;
#pragma unroll
        for (uint32_t w = 0; w < THREADS / 64; ++w) {
            if (w < wave) before = add_sat(before, lds[i][w]);
            sum = add_sat(sum, lds[i][w]);
        }
        v[i] = add_sat(before, v[i]);
        total[i] = sum;
    }
}

// Prefix sums over the requests of the tokens asked and the pages wanted; if
// that refuses some, of the pages wanted by the rest, the tokens granted and
// the pages granted; then the new pages and tokens, each found by a search in
// the sums. Every workgroup computes the sums for itself and writes its share
// of the tokens and pages, 20 bytes a token. Bound by latency: the sums and two
// dependent reads. 32 requests' single tokens take 3.3 us (one wavefront, no
// barriers; 6.3 by 1024 threads), 256 requests' 100606 prompt tokens, the last
// of which are refused, 6.6 us (one workgroup alone 96).
template <uint32_t THREADS>
__global__ __launch_bounds__(THREADS) void nz_pages_extend_kernel(nz_pages_extend_args a) {
    __shared__ uint32_t waves[2][THREADS / 64];
    __shared__ uint32_t page_first[THREADS], token_first[THREADS];
    __shared__ int32_t lens[THREADS];
    const uint32_t page = a.page_size, shift = 31 - __clz(page);
    const uint32_t stride = gridDim.x * THREADS, at = blockIdx.x * THREADS + threadIdx.x;
    const uint64_t limit = static_cast<uint64_t>(a.max_pages) << shift;
    const uint32_t n_free = min(static_cast<uint32_t>(max(a.n_free[0], 0)), a.n_pages);
    uint32_t asked_before = 0, pages_before = 0, tokens_before = 0, taken = 0;
    for (uint32_t r0 = 0; r0 < a.n_requests; r0 += THREADS) {
        const uint32_t r = r0 + threadIdx.x;
        const bool live = r < a.n_requests;
        const int32_t length = live ? a.lengths[r] : 0, asks = live ? a.new_tokens[r] : 0;
        const bool fits = asks >= 0 && length >= 0 &&
                          static_cast<uint64_t>(length) + static_cast<uint64_t>(asks) <= limit;
        const uint32_t old = fits ? (static_cast<uint32_t>(length) + page - 1) >> shift : 0;
        uint32_t n = fits ? asks : 0;
        uint32_t want = fits ? ((static_cast<uint32_t>(length) + n + page - 1) >> shift) - old : 0;
        uint32_t sums[2] = {n, want}, totals[2];
        block_scan<THREADS, 2>(sums, totals, waves);
        bool room = true, have = true;
        if (add_sat(asked_before, totals[0]) > a.max_tokens || add_sat(pages_before, totals[1]) > n_free) {
            room = n == 0 || add_sat(asked_before, sums[0]) <= a.max_tokens;
            if (!room) n = 0, want = 0;
            uint32_t wanted[1] = {want}, total[1];
            block_scan<THREADS, 1>(wanted, total, waves);
            have = want == 0 || add_sat(pages_before, wanted[0]) <= n_free;
            asked_before = add_sat(asked_before, totals[0]);
            pages_before = add_sat(pages_before, total[0]);
            if (!have) n = 0, want = 0;
            sums[0] = n, sums[1] = want;
            block_scan<THREADS, 2>(sums, totals, waves);
        } else {
            asked_before = add_sat(asked_before, totals[0]);
            pages_before = add_sat(pages_before, totals[1]);
        }
        const uint32_t tokens = tokens_before + sums[0] - n;
        page_first[threadIdx.x] = taken + sums[1] - want;
        token_first[threadIdx.x] = tokens;
        lens[threadIdx.x] = length;
        if (live && blockIdx.x == 0) {
            a.status[r] = !fits ? NZ_PAGES_TOO_LONG : !room ? NZ_PAGES_NO_ROOM : !have ? NZ_PAGES_NO_PAGE : NZ_PAGES_OK;
            a.starts[r] = static_cast<int32_t>(tokens);
            a.lengths_after[r] = length + static_cast<int32_t>(n);
            // a single workgroup advances the state itself: no other reads it
            if (a.advance && gridDim.x == 1) const_cast<int32_t*>(a.lengths)[r] = length + static_cast<int32_t>(n);
        }
        __syncthreads();
        for (uint32_t j = at; j < totals[1]; j += stride) {
            const uint32_t i = owner(page_first, THREADS, taken + j);
            const uint32_t entry = ((static_cast<uint32_t>(lens[i]) + page - 1) >> shift) + taken + j - page_first[i];
            a.tables[static_cast<uint64_t>(r0 + i) * a.max_pages + entry] = a.free_pages[n_free - 1 - (taken + j)];
        }
        for (uint32_t j = at; j < totals[0]; j += stride) {
            const uint32_t t = tokens_before + j, i = owner(token_first, THREADS, t);
            const uint32_t len = lens[i], position = len + t - token_first[i], entry = position >> shift;
            const uint32_t old_pages = (len + page - 1) >> shift;
            const int32_t p = entry < old_pages ? a.tables[static_cast<uint64_t>(r0 + i) * a.max_pages + entry]
                                                : a.free_pages[n_free - 1 - (page_first[i] + entry - old_pages)];
            a.slots[t] = static_cast<uint32_t>(p) < a.n_pages
                             ? (static_cast<int64_t>(p) << shift) + (position & (page - 1)) : -1;
            a.positions[t] = static_cast<int32_t>(position);
            a.requests[t] = static_cast<int32_t>(r0 + i);
            a.contexts[t] = static_cast<int32_t>(position) + 1;
        }
        tokens_before += totals[0];
        taken += totals[1];
        __syncthreads();   // the searches above, before the next strip's sums
    }
    for (uint32_t t = tokens_before + at; t < a.max_tokens; t += stride) {
        a.slots[t] = -1;
        a.positions[t] = 0;
        a.requests[t] = -1;
        a.contexts[t] = 0;
    }
    if (at == 0) {
        a.starts[a.n_requests] = static_cast<int32_t>(tokens_before);
        a.n_free_after[0] = static_cast<int32_t>(n_free - taken);
        if (a.advance && gridDim.x == 1) const_cast<int32_t*>(a.n_free)[0] = static_cast<int32_t>(n_free - taken);
    }
}

// Prefix sums over the requests of the pages they give back, then the pages,
// each found by a search in the sums: 22131 pages of 250 of 1000 requests take
// 3.7 us, and 20 by one workgroup alone.
template <uint32_t THREADS>
__global__ __launch_bounds__(THREADS) void nz_pages_release_kernel(nz_pages_release_args a) {
    __shared__ uint32_t waves[1][THREADS / 64];
    __shared__ uint32_t first[THREADS];
    const uint32_t page = a.page_size, shift = 31 - __clz(page);
    const uint32_t stride = gridDim.x * THREADS, at = blockIdx.x * THREADS + threadIdx.x;
    uint32_t top = min(static_cast<uint32_t>(max(a.n_free[0], 0)), a.n_pages);
    for (uint32_t r0 = 0; r0 < a.n_requests; r0 += THREADS) {
        const uint32_t r = r0 + threadIdx.x;
        const bool live = r < a.n_requests, done = live && a.done[r] != 0;
        const int32_t length = live ? max(a.lengths[r], 0) : 0;
        const uint32_t back = done ? min((static_cast<uint32_t>(length) + page - 1) >> shift, a.max_pages) : 0;
        uint32_t sum[1] = {back}, total[1];
        block_scan<THREADS, 1>(sum, total, waves);
        first[threadIdx.x] = sum[0] - back;
        if (live && blockIdx.x == 0) {
            a.lengths_after[r] = done ? 0 : length;
            if (a.advance && gridDim.x == 1) const_cast<int32_t*>(a.lengths)[r] = done ? 0 : length;
        }
        __syncthreads();
        const uint32_t kept = min(total[0], a.n_pages - top);
        for (uint32_t j = at; j < kept; j += stride) {
            const uint32_t i = owner(first, THREADS, j);
            a.free_pages[top + j] = a.tables[static_cast<uint64_t>(r0 + i) * a.max_pages + j - first[i]];
        }
        top += kept;
        __syncthreads();
    }
    if (at == 0) {
        a.n_free_after[0] = static_cast<int32_t>(top);
        if (a.advance && gridDim.x == 1) const_cast<int32_t*>(a.n_free)[0] = static_cast<int32_t>(top);
    }
}

// The state after a call of several workgroups, which read the old one until
// the last of them ends.
__global__ __launch_bounds__(kPagesThreads)
void nz_pages_advance_kernel(const int32_t* __restrict__ lengths_after, const int32_t* __restrict__ n_free_after,
                             int32_t* lengths, int32_t* n_free, uint32_t n) {
    const uint32_t r = blockIdx.x * kPagesThreads + threadIdx.x;
    if (r < n) lengths[r] = lengths_after[r];
    if (r == 0) n_free[0] = n_free_after[0];
}

// ------------------------------------------------- norm, rotation and store

constexpr uint32_t kRotaryThreads = 256;

// A head is held by a group of `LANES` lanes (a power of two), 16 elements
// each, in runs of 16 bytes: the first rotary_dim elements, and apart from
// them the rest, are cut into as many stretches as a lane has runs, and a
// lane's runs lie at the same place of each, so that the group's accesses are
// whole stretches. Pairs (i, i + rotary_dim / 2) are then in one lane, in x
// and y; neighbouring pairs are inside a run. Bound by memory: 8191 tokens of
// 64 bf16 heads over 8, normed (340 MB), take 64 to 67 us, 5.1 to 5.3 TB/s,
// with streaming stores and 72 with ordinary ones, which gain nothing for the
// attention that reads the results (a layer of 32 tokens over 500 keys 17.6 us
// with either).
template <typename T, uint32_t LANES>
__global__ __launch_bounds__(kRotaryThreads) void nz_rotary_kernel(nz_rotary_args a) {
    constexpr uint32_t kRun = run_of<T>(), kRuns = 8 / kRun;   // of x and of y
    // (the caller keeps the heads of a call below 2^31)
    const uint32_t index = blockIdx.x * (kRotaryThreads / LANES) + threadIdx.x / LANES;
    const uint32_t per_token = a.heads + 2 * a.kv_heads;
    if (index >= a.tokens * per_token) return;   // whole groups leave together
    const uint32_t token = index / per_token, head = index % per_token;
    const bool is_q = head < a.heads, is_v = head >= a.heads + a.kv_heads;
    const uint32_t h = is_q ? head : is_v ? head - a.heads - a.kv_heads : head - a.heads;
    const uint32_t lane = threadIdx.x % LANES, turned = is_v ? 0 : a.rotary_dim;
    const bool live = lane < a.head_dim / 16, turns = lane < turned / 16;
    const uint32_t start = turns ? 0 : turned, half = (turns ? turned : a.head_dim - turned) / 2;
    const uint32_t apart = half / kRuns, xt = start + kRun * (turns ? lane : lane - turned / 16), yt = xt + half;
    T* dst = nullptr;
    if (is_q) {
        dst = static_cast<T*>(a.out) + token * a.out_token + h * a.out_head;
    } else if (a.key_cache != nullptr) {
        const int64_t slot = a.slots[token];
        const uint32_t shift = 31 - __clz(a.page_size);
        if (static_cast<uint64_t>(slot) < static_cast<uint64_t>(a.n_pages) << shift) {
            const int64_t p = slot >> shift, place = slot & (a.page_size - 1);
            dst = is_v ? static_cast<T*>(a.value_cache) + p * a.value_page + place * a.value_slot + h * a.value_head
                       : static_cast<T*>(a.key_cache) + p * a.key_page + place * a.key_slot + h * a.key_head;
        }
    }
    const T* src = is_q   ? static_cast<const T*>(a.q) + token * a.q_token + h * a.q_head
                   : is_v ? static_cast<const T*>(a.v) + token * a.v_token + h * a.v_head
                          : static_cast<const T*>(a.k) + token * a.k_token + h * a.k_head;
    const bool works = live && dst != nullptr;
    float x[8] = {}, y[8] = {};
    if (works) {
        load_runs(src + xt, apart, x);
        load_runs(src + yt, apart, y);
    }
    const void* weight = is_q ? a.q_weight : is_v ? nullptr : a.k_weight;
    if (weight != nullptr) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += x[i] * x[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += y[i] * y[i];
#pragma unroll
        for (uint32_t d = 1; d < LANES; d <<= 1) sum += __shfl_xor(sum, d);
        const float scale = rsqrtf(sum / static_cast<float>(a.head_dim) + a.eps);
        if (live) {
            float wx[8], wy[8];
            if (a.weight_type == NZ_FP32) {
#pragma unroll
                for (uint32_t r = 0; r < kRuns; ++r) {
                    load_floats<kRun>(static_cast<const float*>(weight) + xt + r * apart, wx + r * kRun);
                    load_floats<kRun>(static_cast<const float*>(weight) + yt + r * apart, wy + r * kRun);
                }
            } else {
                load_runs(static_cast<const T*>(weight) + xt, apart, wx);
                load_runs(static_cast<const T*>(weight) + yt, apart, wy);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * scale * wx[i], y[i] = y[i] * scale * wy[i];
        }
    }
    if (turns) {
        const uint32_t position = static_cast<uint32_t>(a.positions[token]);
        const bool known = position < a.n_positions;
        const uint64_t angles = static_cast<uint64_t>(known ? position : 0) * (a.rotary_dim / 2);
        float c[8], s[8];
        if (a.interleaved) {   // of the pairs in x's runs, then in y's
#pragma unroll
            for (uint32_t r = 0; r < 2 * kRuns; ++r) {
                const uint32_t at = ((r < kRuns ? xt : yt) + r % kRuns * apart) / 2;
#pragma unroll
                for (uint32_t i = 0; i < kRun / 2; ++i)
                    c[r * kRun / 2 + i] = a.cos[angles + at + i], s[r * kRun / 2 + i] = a.sin[angles + at + i];
            }
        } else {
#pragma unroll
            for (uint32_t r = 0; r < kRuns; ++r) {
                load_floats<kRun>(a.cos + angles + xt + r * apart, c + r * kRun);
                load_floats<kRun>(a.sin + angles + xt + r * apart, s + r * kRun);
            }
        }
        if (!known) {
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] = s[i] = __builtin_nanf("");
        }
        if (a.interleaved) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                turn(x[2 * i], x[2 * i + 1], c[i], s[i]);
                turn(y[2 * i], y[2 * i + 1], c[4 + i], s[4 + i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) turn(x[i], y[i], c[i], s[i]);
        }
    }
    if (works) {
        store_runs(dst + xt, apart, x);
        store_runs(dst + yt, apart, y);
    }
}

// -------------------------------------------------------------- the logits

constexpr uint32_t kLogitsThreads = 1024;
// Tokens of the vocabulary that a workgroup takes and counts in LDS.
constexpr uint32_t kLogitsChunk = 8192;

// Calls note(i, id) for the ids 0 .. length - 1 at `ids`: 16 bytes at a time
// where they lie on such boundaries, one by one at the ends.
template <typename ID, typename Note>
__device__ __forceinline__ void for_history(const ID* ids, uint32_t length, const Note& note) {
    constexpr uint32_t kRun = run_of<ID>();
    const uint32_t skip = min(static_cast<uint32_t>(-reinterpret_cast<uintptr_t>(ids) % 16 / sizeof(ID)), length);
    const uint32_t runs = (length - skip) / kRun, rest = length - runs * kRun;
#pragma unroll 4
    for (uint32_t j = threadIdx.x; j < runs; j += kLogitsThreads) {
        const vec<ID, kRun> v = *reinterpret_cast<const vec<ID, kRun>*>(ids + skip + j * kRun);
#pragma unroll
        for (uint32_t e = 0; e < kRun; ++e) note(skip + j * kRun + e, static_cast<int64_t>(v[e]));
    }
    for (uint32_t e = threadIdx.x; e < rest; e += kLogitsThreads) {
        const uint32_t i = e < skip ? e : e + runs * kRun;
        note(i, static_cast<int64_t>(ids[i]));
    }
}

// One workgroup: kLogitsChunk neighbouring tokens of a row, the first on a
// 16-byte boundary of the row's memory (in the row's first chunk that may lie
// before the row). It requests its logits, counts the row's history that
// falls into the chunk meanwhile (answer tokens in the low 31 bits, a prompt
// token in the top bit) and notes each token's last bias entry, and then adjusts
// and stores the logits. Integer LDS atomics only: the order of arrival does
// not show. Every chunk's workgroup reads the row's whole history, out of the
// L2. Bound by memory, once the history is short against the vocabulary: 32
// rows of 128256 fp32 logits with everything on (33 MB) take 9.6 us, one row of
// 151936 bf16 logits 4.1; the first were 12.8 us with chunks of 2048, 11.3 of
// 4096 and 10.6 of 8192 tokens (64 rows with up to 8000 ids 27, 21 and 18, and
// 16 with ids read 16 bytes at a time, which costs short histories 0.1 to 0.5).
// VECTOR: logits and out lie alike on 16-byte boundaries.
template <typename T, bool VECTOR>
__global__ __launch_bounds__(kLogitsThreads) void nz_logits_kernel(nz_logits_args a) {
    constexpr uint32_t kRun = VECTOR ? 16 / sizeof(T) : 1, kRuns = kLogitsChunk / (kLogitsThreads * kRun);
    using run = vec<T, kRun>;
    __shared__ uint32_t counts[kLogitsChunk], entries[kLogitsChunk];
    const uint32_t row = blockIdx.y;
    const T* const src = static_cast<const T*>(a.logits) + row * a.logits_row;
    T* const dst = static_cast<T*>(a.out) + row * a.out_row;
    const uint32_t before = VECTOR ? static_cast<uint32_t>(reinterpret_cast<uintptr_t>(src) % 16 / sizeof(T)) : 0;
    const int64_t v0 = static_cast<int64_t>(blockIdx.x) * kLogitsChunk - before;
    if (v0 >= static_cast<int64_t>(a.vocab)) return;
    const uint32_t* mask = nullptr;
    const uint32_t words = (a.vocab + 31) / 32;
    if (a.masks != nullptr) {
        const int64_t m = a.mask_rows ? a.mask_rows[row] : static_cast<int64_t>(row);
        if (static_cast<uint64_t>(m) < a.n_masks) mask = a.masks + static_cast<uint64_t>(m) * words;
    }
    // a run inside the row as one access, one at its ends by elements; its
    // mask bits are in one word or two
    run x[kRuns];
    uint32_t bits[kRuns];
#pragma unroll
    for (uint32_t k = 0; k < kRuns; ++k) {
        const int64_t v = v0 + (k * kLogitsThreads + threadIdx.x) * kRun;
        if (v >= 0 && v + kRun <= a.vocab) {
            x[k] = *reinterpret_cast<const run*>(src + v);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kRun; ++i)
                x[k][i] = v + i >= 0 && v + i < a.vocab ? src[v + i] : static_cast<T>(0.0f);
        }
        bits[k] = ~0u;
        if (mask != nullptr && v + kRun > 0 && v < a.vocab) {
            const uint32_t first = v > 0 ? static_cast<uint32_t>(v) : 0, word = first >> 5;
            uint64_t two = mask[word];
            if (kRun > 1 && (first & 31) + kRun > 32 && word + 1 < words)
                two |= static_cast<uint64_t>(mask[word + 1]) << 32;
            bits[k] = static_cast<uint32_t>(two >> (first & 31)) << (first - v);
        }
    }
    const float repetition = a.repetition ? a.repetition[row] : 1.0f, frequency = a.frequency ? a.frequency[row] : 0.0f;
    const float presence = a.presence ? a.presence[row] : 0.0f;
    for (uint32_t i = threadIdx.x; i < kLogitsChunk; i += kLogitsThreads) counts[i] = 0;
    if (a.bias_starts != nullptr)
        for (uint32_t i = threadIdx.x; i < kLogitsChunk; i += kLogitsThreads) entries[i] = 0;
    __syncthreads();
    if (a.history != nullptr) {
        const uint32_t length = min(static_cast<uint32_t>(max(a.lengths[row], 0)), a.history_capacity);
        const uint32_t prompt = a.prompt_lengths ? static_cast<uint32_t>(max(a.prompt_lengths[row], 0)) : 0;
        const uint64_t first = static_cast<uint64_t>(row) * static_cast<uint64_t>(a.history_row);
        const auto note = [&](uint32_t i, int64_t id) {
            const uint64_t v = static_cast<uint64_t>(id - v0);
            if (v < kLogitsChunk) {
                if (i < prompt) atomicOr(&counts[v], 0x80000000u);
                else atomicAdd(&counts[v], 1u);
            }
        };
        if (a.history_bytes == 8) for_history(static_cast<const int64_t*>(a.history) + first, length, note);
        else for_history(static_cast<const int32_t*>(a.history) + first, length, note);
    }
    if (a.bias_starts != nullptr) {
        const uint32_t e0 = min(static_cast<uint32_t>(max(a.bias_starts[row], 0)), a.n_bias);
        const uint32_t e1 = min(static_cast<uint32_t>(max(a.bias_starts[row + 1], 0)), a.n_bias);
        for (uint32_t e = e0 + threadIdx.x; e < e1; e += kLogitsThreads) {
            const uint64_t v = static_cast<uint64_t>(static_cast<int64_t>(a.bias_tokens[e]) - v0);
            if (v < kLogitsChunk) atomicMax(&entries[v], e + 1);
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < kRuns; ++k) {
        const uint32_t at = (k * kLogitsThreads + threadIdx.x) * kRun;
        const int64_t v = v0 + at;
#pragma unroll
        for (uint32_t i = 0; i < kRun; ++i) {
            float y = to_float(static_cast<T>(x[k][i]));
            const uint32_t count = counts[at + i], entry = a.bias_starts != nullptr ? entries[at + i] : 0;
            if (count) {
                y = y > 0.0f ? y / repetition : y * repetition;
                const uint32_t answers = count & 0x7FFFFFFFu;
                if (answers) y = y - frequency * static_cast<float>(answers) - presence;
            }
            if (entry) y += a.bias_values[entry - 1];
            if (!(bits[k] >> i & 1u)) y = -__builtin_inff();
            x[k][i] = from_float<T>(y);
        }
        if (v >= 0 && v + kRun <= a.vocab) {
            *reinterpret_cast<run*>(dst + v) = x[k];
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kRun; ++i)
                if (v + i >= 0 && v + i < a.vocab) dst[v + i] = x[k][i];
        }
    }
}

int launched(const char* what, char* message, size_t message_size) {
    const hipError_t rc = hipGetLastError();
    if (rc == hipSuccess) return 0;
    snprintf(message, message_size, "%s launch failed: %s", what, hipGetErrorString(rc));
    return -6;
}

template <typename T>
void launch_rotary(const nz_rotary_args& a, hipStream_t stream) {
    uint32_t lanes = 1;
    while (lanes * 16 < a.head_dim) lanes *= 2;
    const uint64_t threads = static_cast<uint64_t>(a.tokens) * (a.heads + 2 * a.kv_heads) * lanes;
    const dim3 grid(static_cast<uint32_t>((threads + kRotaryThreads - 1) / kRotaryThreads));
#define NZ_ROTARY(L) hipLaunchKernelGGL((nz_rotary_kernel<T, L>), grid, dim3(kRotaryThreads), 0, stream, a)
    switch (lanes) {
        case 1: NZ_ROTARY(1); break;
        case 2: NZ_ROTARY(2); break;
        case 4: NZ_ROTARY(4); break;
        case 8: NZ_ROTARY(8); break;
        default: NZ_ROTARY(16); break;
    }
#undef NZ_ROTARY
}

}  // namespace

// The callers (capi_serving.cpp) have checked the arguments.

// `work` tokens or pages by workgroups of 64, 256 or 1024 threads, several
// where one would write more than kPagesShare; then the state's advance.
#define NZ_PAGES(kernel, work)                                                                                    \
    const hipStream_t st = static_cast<hipStream_t>(stream);                                                      \
    const uint64_t amount = (work);                                                                               \
    const uint32_t groups = amount <= kPagesShare                                                                 \
                                ? 1 : static_cast<uint32_t>(std::min<uint64_t>((amount + 1023) / 1024, kPagesGroups)); \
    if (groups == 1 && args->n_requests <= 64 && amount <= 128)                                                   \
        hipLaunchKernelGGL(kernel<64>, dim3(1), dim3(64), 0, st, *args);                                          \
    else if (groups == 1 && args->n_requests <= 256 && amount <= 1024)                                            \
        hipLaunchKernelGGL(kernel<256>, dim3(1), dim3(256), 0, st, *args);                                        \
    else                                                                                                          \
        hipLaunchKernelGGL(kernel<kPagesThreads>, dim3(groups), dim3(kPagesThreads), 0, st, *args);               \
    if (args->advance && groups > 1)                                                                              \
        hipLaunchKernelGGL(nz_pages_advance_kernel, dim3((args->n_requests + kPagesThreads) / kPagesThreads),     \
                           dim3(kPagesThreads), 0, st, args->lengths_after, args->n_free_after,                   \
                           const_cast<int32_t*>(args->lengths), const_cast<int32_t*>(args->n_free), args->n_requests)

extern "C" int nz_hip_pages_extend(const nz_pages_extend_args* args, void* stream, char* message, size_t message_size) {
    NZ_PAGES(nz_pages_extend_kernel, args->max_tokens);
    return launched("pages extend", message, message_size);
}

extern "C" int nz_hip_pages_release(const nz_pages_release_args* args, void* stream, char* message,
                                    size_t message_size) {
    // no more pages come back than there are, or than the tables hold
    NZ_PAGES(nz_pages_release_kernel,
             std::min<uint64_t>(args->n_pages, static_cast<uint64_t>(args->n_requests) * args->max_pages));
    return launched("pages release", message, message_size);
}

extern "C" int nz_hip_rotary_store(const nz_rotary_args* args, void* stream, char* message, size_t message_size) {
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (args->type == NZ_BF16) launch_rotary<bf16_t>(*args, st);
    else if (args->type == NZ_FP16) launch_rotary<_Float16>(*args, st);
    else launch_rotary<float>(*args, st);
    return launched("rotary", message, message_size);
}

extern "C" int nz_hip_adjust_logits(const nz_logits_args* args, void* stream, char* message, size_t message_size) {
    const hipStream_t st = static_cast<hipStream_t>(stream);
    // every row of the two must start alike on 16-byte boundaries; one more
    // chunk holds what the first one's tokens before the row push out
    const uint32_t size = args->type == NZ_FP32 ? 4 : 2;
    const uintptr_t apart = reinterpret_cast<uintptr_t>(args->logits) - reinterpret_cast<uintptr_t>(args->out);
    const bool vector = apart % 16 == 0 && (args->rows == 1 || (args->logits_row - args->out_row) * size % 16 == 0);
    const dim3 grid((args->vocab + 16 / size - 1 + kLogitsChunk - 1) / kLogitsChunk, args->rows), block(kLogitsThreads);
#define NZ_LOGITS(T)                                                                                   \
    do {                                                                                               \
        if (vector) hipLaunchKernelGGL((nz_logits_kernel<T, true>), grid, block, 0, st, *args);        \
        else hipLaunchKernelGGL((nz_logits_kernel<T, false>), grid, block, 0, st, *args);              \
    } while (0)
    if (args->type == NZ_BF16) NZ_LOGITS(bf16_t);
    else if (args->type == NZ_FP16) NZ_LOGITS(_Float16);
    else NZ_LOGITS(float);
#undef NZ_LOGITS
    return launched("logits", message, message_size);
}
