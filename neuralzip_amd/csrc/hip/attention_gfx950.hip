// attention_gfx950.hip -- attention of single tokens over a paged key-value
// cache: the plan that cuts the rows' contexts into items (nz_attention_plan)
// and the kernels that run it (nz_attention).
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <type_traits>

#include "attention_types.h"
#include "neuralzip_hip.h"
#include "serving_types.h"

namespace {

// ------------------------------------------------------------------- plan

constexpr uint32_t kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
// Items start at multiples of kTile keys. The length that they may have is no
// shorter than gives each wavefront of a workgroup one such tile, or, up to
// kLeastLong, than a sixteenth of the longest context: more items than that
// take longer to join than they save (one row over 8 heads of 8000 keys 13.2
// us with items of 512 keys and 14.6 of 256; of 2001 keys 11.1 of 512 and 8.8
// of 128). A row is then cut into equal parts, which may be little more than
// half as long.
constexpr uint32_t kTile = 32, kLeastItem = 128, kLeastLong = 512;

struct PlanLds {
    uint64_t keys[kPlanWaves];
    uint32_t most[kPlanWaves], counts[kPlanWaves];
    uint32_t contexts[kPlanThreads];                     // of up to as many rows
    uint32_t first[kPlanThreads], each[kPlanThreads];    // per row of a strip: first item, its items' length
};

__device__ __forceinline__ uint32_t context_of(const int32_t* contexts, uint32_t r) {
    return static_cast<uint32_t>(max(contexts[r], 0));
}

// Items of all rows when none is longer than `share` (a wavefront's sum).
__device__ __forceinline__ uint32_t count_items(const int32_t* contexts, uint32_t n_rows, uint32_t share,
                                                const PlanLds& lds) {
    uint32_t n = 0;
    if (n_rows <= kPlanThreads) {
        for (uint32_t r = threadIdx.x & 63; r < n_rows; r += 64) n += max((lds.contexts[r] + share - 1) / share, 1u);
    } else {
#pragma unroll 4
        for (uint32_t r = threadIdx.x & 63; r < n_rows; r += 64)
            n += max((context_of(contexts, r) + share - 1) / share, 1u);
    }
    return last_lane(wave_scan(n));
}

// The shortest item length, in tiles and from `least` on, of which there are
// at most `limit` (n_rows or more) items; `longest` tiles is one. Every
// wavefront tries another length.
__device__ uint32_t shortest_share(const int32_t* contexts, uint32_t n_rows, uint32_t limit, uint64_t keys,
                                   uint32_t least, uint32_t longest, PlanLds& lds) {
    const uint32_t wave = threadIdx.x >> 6;
    // keys / share <= items < n_rows + keys / share
    const uint64_t below_all = keys / (static_cast<uint64_t>(limit) * kTile);
    uint32_t lo = static_cast<uint32_t>(std::max<uint64_t>(least, std::min<uint64_t>(below_all, longest)));
    uint32_t hi = max(longest, lo);
    if (limit > n_rows) {
        const uint64_t enough = keys / (static_cast<uint64_t>(limit - n_rows) * kTile) + 1;
        hi = max(static_cast<uint32_t>(min<uint64_t>(enough, hi)), lo);
    }
    while (lo < hi) {
        const uint32_t step = (hi - lo + kPlanWaves) / (kPlanWaves + 1);
        const uint32_t tried = min(lo + wave * step, hi);
        const uint32_t n = count_items(contexts, n_rows, tried * kTile, lds);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds.counts[wave] = n;
        __syncthreads();
        // longer items are fewer: the first length tried that gives few enough
        const uint32_t lane = threadIdx.x & 63;
        const uint64_t few = __ballot(lane < kPlanWaves && lds.counts[min(lane, kPlanWaves - 1)] <= limit);
        const uint32_t at = few ? __builtin_ctzll(few) : kPlanWaves;
        const uint32_t below = lo + at * step;   // the length itself, or one past those tried
        if (at > 0) lo = min(below - step, hi) + 1;
        if (few) hi = min(below, hi);
    }
    return lo;
}

// One workgroup. Items are as short as the number wanted allows, so that they
// take about the same time: one per compute unit and row's heads while that
// cuts no row far shorter than its share, since rows of one item need no
// join; one more per compute unit where some rows are much longer than others
// (in whole rounds of the units: 32 rows of up to 8191 keys over 8 heads 98 us
// with 64 items and 111 with 48). Latency bound: 5 us for one row of 2001
// keys, 9 for 64 ragged rows, once a step.
__global__ __launch_bounds__(kPlanThreads)
void nz_attention_plan_kernel(const int32_t* __restrict__ contexts, const int32_t* __restrict__ requests,
                              uint32_t n_rows, uint32_t target, uint32_t parts, nz_attention_item* __restrict__ items,
                              uint32_t* __restrict__ counters) {
    __shared__ PlanLds lds;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t keys = 0;
    uint32_t longest = 0;
    for (uint32_t r = threadIdx.x; r < n_rows; r += kPlanThreads) {
        const uint32_t context = context_of(contexts, r);
        if (r < kPlanThreads) lds.contexts[r] = context;
        keys += context;
        longest = max(longest, context);
    }
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        keys += __shfl_xor(keys, d);
        longest = max(longest, static_cast<uint32_t>(__shfl_xor(longest, d)));
    }
    if (lane == 0) lds.keys[wave] = keys, lds.most[wave] = longest;
    __syncthreads();
    keys = 0;
#pragma unroll
    for (uint32_t w = 0; w < kPlanWaves; ++w) keys += lds.keys[w], longest = max(longest, lds.most[w]);
    const uint32_t fewest = (max(target, n_rows) + target - 1) / target * target, tiles = (longest + kTile - 1) / kTile;
    const uint32_t least = min(max((tiles + 15) / 16, kLeastItem / kTile), kLeastLong / kTile);
    uint32_t share = least;
    if (tiles > least) {
        share = shortest_share(contexts, n_rows, fewest, keys, least, tiles, lds);
        const uint64_t length = static_cast<uint64_t>(share) * kTile;
        if (length * fewest * 2 > keys * 3 && length * target * 2 > keys)
            share = shortest_share(contexts, n_rows, fewest + target, keys, least, share, lds);
    }
    const uint32_t most = share * kTile;
    const int32_t total_keys = static_cast<int32_t>(min<uint64_t>((keys + 1023) / 1024, 0x7FFFFFFFu));
    uint32_t first = 0;
    for (uint32_t r0 = 0; r0 < n_rows; r0 += kPlanThreads) {
        const uint32_t r = r0 + threadIdx.x;
        const bool live = r < n_rows;
        const uint32_t context = live ? context_of(contexts, r) : 0;
        // a row's items are of equal length, in whole tiles
        uint32_t n = max((context + most - 1) / most, 1u);
        const uint32_t each = max(((context + n - 1) / n + kTile - 1) / kTile * kTile, kTile);
        n = live ? max((context + each - 1) / each, 1u) : 0;
        const uint32_t scan = wave_scan(n);
        __syncthreads();   // the last reads of `counts`, `first` and `each`
        if (lane == 63) lds.counts[wave] = scan;
        __syncthreads();
        uint32_t before = 0, total = 0;
#pragma unroll
        for (uint32_t w = 0; w < kPlanWaves; ++w) {
            if (w < wave) before += lds.counts[w];
            total += lds.counts[w];
        }
        lds.first[threadIdx.x] = before + scan - n;
        lds.each[threadIdx.x] = each;
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < total; j += kPlanThreads) {
            const uint32_t i = owner(lds.first, min(n_rows - r0, kPlanThreads), j), index = j - lds.first[i];
            const uint32_t end_of_row = i + 1 < min(n_rows - r0, kPlanThreads) ? lds.first[i + 1] : total;
            const uint32_t length = n_rows <= kPlanThreads ? lds.contexts[i] : context_of(contexts, r0 + i);
            nz_attention_item item;
            item.row = static_cast<int32_t>(r0 + i);
            item.request = requests ? requests[r0 + i] : static_cast<int32_t>(r0 + i);
            item.begin = static_cast<int32_t>(index * lds.each[i]);
            item.end = static_cast<int32_t>(min(length, (index + 1) * lds.each[i]));
            item.index = static_cast<int32_t>(index);
            item.count = static_cast<int32_t>(end_of_row - lds.first[i]);
            item.first = static_cast<int32_t>(first + lds.first[i]);
            item.keys = total_keys;
            items[first + j] = item;
        }
        first += total;
    }
    const nz_attention_item none = {-1, -1, 0, 0, 0, 0, 0, 0};
    for (uint32_t i = first + threadIdx.x; i < fewest + target; i += kPlanThreads) items[i] = none;
    for (uint64_t i = threadIdx.x; i < static_cast<uint64_t>(first) * parts; i += kPlanThreads) counters[i] = 0;
}

// -------------------------------------------------------------- attention

constexpr uint32_t kWaves = 4, kThreads = 64 * kWaves;
// Query heads of one key-value head that a workgroup takes: the columns of a
// matrix instruction.
constexpr uint32_t kHeads = 16;
// What the Infinity Cache holds.
constexpr uint64_t kCacheBytes = 256ull << 20;
// One item: 16 query heads' softmax over the keys begin .. end - 1 of one
// key-value head, tile by tile with a running maximum and sum:
//   m' = max(m, s_j), l' = l 2^(m - m') + sum_j 2^(s_j - m'),
//   o' = o 2^(m - m') + sum_j 2^(s_j - m') v_j, s_j = scale log2(e) q . k_j.
// Bound by HBM: 4 or 8 query heads read each key, a sixteenth of what the
// matrix instructions could do with it, so they may have idle columns and
// multiply by split weights. 64 rows of 100 to 16384 keys, 64 heads over 8 of
// 128 fp16 elements (2.16 GB), take 370 to 394 us by the rows' order, 5.5 to
// 5.8 TB/s; 32 rows of up to 8191 keys, 32 heads over 8 in bf16 (488 MB), 96
// us; one row of 2001 keys 8.7 us, of which starting takes 2.7 and the join
// of the items 2.7.
// Scores are computed transposed (keys are rows, heads columns), so that a
// lane's scores of a tile are the very elements it needs as the second
// operand of the product with the values: its four rows of each 16 keys. The
// values are loaded whole rows at a time, each lane some neighbours of the
// keys its scores belong to, and transposed in registers; no LDS until the
// wavefronts' sums are joined. Four wavefronts take every fourth tile of 32
// keys, each with the next tile's keys under way: three such workgroups a
// compute unit (two-byte types, up to 128 elements) keep 190 KB in flight.
// 16-bit types of up to 128 elements are held to the registers of three
// wavefronts a SIMD: 483 us for the 2.16 GB, 491 without, before the join
// was part of this kernel.
template <typename T, uint32_t DP, bool FULL>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(DP <= 128 && sizeof(T) == 2 ? 3 : 1)))
void nz_attention_kernel(nz_attention_args a) {
    using S = Shape<T, DP>;
    using P = Piece<T>;
    using piece = typename P::type;
    using value_run = vec<T, S::kValueRun>;
    __shared__ float lds_m[kWaves][kHeads], lds_l[kWaves][kHeads];
    __shared__ __align__(16) float lds_o[kWaves][kHeads][DP + 4];
    __shared__ uint32_t last;

    const uint32_t group = a.heads / a.kv_heads, blocks = (group + kHeads - 1) / kHeads;
    // Workgroups that read the same keys, for different blocks of heads, lie
    // kXcds apart: they run on one XCD and share its L2.
    const uint32_t turn = blockIdx.x / kXcds, unit = turn / blocks * kXcds + blockIdx.x % kXcds, block = turn % blocks;
    const uint32_t which = unit / a.kv_heads, kv_head = unit % a.kv_heads;
    if (which >= a.n_items) return;
    const nz_attention_item item = a.items[which];
    if (static_cast<uint32_t>(item.row) >= a.n_rows) return;
    const uint32_t per_item = a.kv_heads * blocks, part = kv_head * blocks + block;
    const uint32_t head0 = kv_head * group + block * kHeads;
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
    const T* const key_base = static_cast<const T*>(a.key_cache) + kv_head * a.key_head;
    const T* const value_base = static_cast<const T*>(a.value_cache) + kv_head * a.value_head;
    f32x4 o[S::kValueSteps][S::kValueRun] = {};
    float m = -__builtin_inff(), l = 0.0f;

    // The pages of a tile's runs of 16 keys (a run lies in one page).
    // Entries are read a tile ahead of the keys, and keys a tile ahead of
    // their products. Past the end, and where there is no page, page 0
    // is read and everything masked.
    auto entries = [&](uint32_t t0, int32_t (&page)[S::kHalves]) {
#pragma unroll
        for (uint32_t h = 0; h < S::kHalves; ++h) {
            const uint32_t t = t0 + 16 * h, entry = t >> shift;
            page[h] = table[min(entry, a.max_pages - 1)];
            if (!known || t >= end || entry >= a.max_pages) page[h] = -1;
        }
    };
    auto run_tiles = [&](auto past) {
        constexpr bool PAST = decltype(past)::value;
        piece keys[S::kHalves][S::kKeySteps];
        auto load_keys = [&](uint32_t t0, const int32_t (&page)[S::kHalves]) {
#pragma unroll
            for (uint32_t h = 0; h < S::kHalves; ++h) {
                const int64_t p = static_cast<uint32_t>(page[h]) < a.n_pages ? page[h] : 0;
                const int64_t place = (t0 + 16 * h) & place_mask;
                const T* src = key_base + p * a.key_page + place * a.key_slot;
#pragma unroll
                for (uint32_t s = 0; s < S::kKeySteps; ++s) {
                    const uint32_t d = s * 4 * S::kRun + quad * S::kRun;
                    keys[h][s] = piece{};
                    if (FULL || d < a.head_dim) keys[h][s] = fetch<PAST, piece>(src + col * a.key_slot + d);
                }
            }
        };
        constexpr uint32_t kStep = kWaves * S::kKeys;
        uint32_t t0 = static_cast<uint32_t>(item.begin) / 16 * 16 + wave * S::kKeys;
        int32_t page[S::kHalves], next[S::kHalves];
        if (t0 < end) {
            entries(t0, page);
            load_keys(t0, page);
            entries(t0 + kStep, next);
        }
        for (; t0 < end; t0 += kStep) {
            const T* values[S::kHalves];
            uint32_t limit[S::kHalves];
#pragma unroll
            for (uint32_t h = 0; h < S::kHalves; ++h) {
                const bool valid = static_cast<uint32_t>(page[h]) < a.n_pages;
                const int64_t p = valid ? page[h] : 0;
                limit[h] = valid ? end : 0;
                const int64_t place = (t0 + 16 * h) & place_mask;
                values[h] = value_base + p * a.value_page + place * a.value_slot;
            }
            value_run v[S::kGroups][S::kValueSteps][S::kRun];
#pragma unroll
            for (uint32_t w = 0; w < S::kGroups; ++w)
#pragma unroll
                for (uint32_t s = 0; s < S::kValueSteps; ++s)
#pragma unroll
                    for (uint32_t k = 0; k < S::kRun; ++k) {
                        const uint32_t d = (s * 16 + col) * S::kValueRun;
                        const uint32_t h = S::kRun == 8 ? k / 4 : w, place = 4 * quad + k % 4;
                        v[w][s][k] = value_run{};
                        if (FULL || d < a.head_dim)
                            v[w][s][k] = fetch<PAST, value_run>(values[h] + place * a.value_slot + d);
                    }
            float score[S::kHalves][4];
#pragma unroll
            for (uint32_t h = 0; h < S::kHalves; ++h) {
                f32x4 acc = {};
#pragma unroll
                for (uint32_t s = 0; s < S::kKeySteps; ++s) acc = P::mma(keys[h][s], q[s], acc);
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
                    score[h][i] = t0 + 16 * h + 4 * quad + i < limit[h] ? acc[i] * scale : -__builtin_inff();
            }
            if (t0 + kStep < end) {
                load_keys(t0 + kStep, next);
#pragma unroll
                for (uint32_t h = 0; h < S::kHalves; ++h) page[h] = next[h];
                entries(t0 + 2 * kStep, next);
            }
            float top = m;
#pragma unroll
            for (uint32_t h = 0; h < S::kHalves; ++h)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) top = fmaxf(top, score[h][i]);
            top = column_max(top);
            const float base = finite_base(top);
            const float fade = __builtin_amdgcn_exp2f(m - base);
            m = top;
            l *= fade;
#pragma unroll
            for (uint32_t s = 0; s < S::kValueSteps; ++s)
#pragma unroll
                for (uint32_t e = 0; e < S::kValueRun; ++e) o[s][e] *= fade;
#pragma unroll
            for (uint32_t h = 0; h < S::kHalves; ++h)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    score[h][i] = __builtin_amdgcn_exp2f(score[h][i] - (base - P::kLift));
                    l += score[h][i];
                }
            // values of masked keys may be anything, NaN among it
            if (t0 + S::kKeys > min(limit[0], limit[S::kHalves - 1])) {
#pragma unroll
                for (uint32_t w = 0; w < S::kGroups; ++w)
#pragma unroll
                    for (uint32_t s = 0; s < S::kValueSteps; ++s)
#pragma unroll
                        for (uint32_t k = 0; k < S::kRun; ++k) {
                            const uint32_t h = S::kRun == 8 ? k / 4 : w;
                            if (t0 + 16 * h + 4 * quad + k % 4 >= limit[h]) v[w][s][k] = value_run{};
                        }
            }
            // the products with the values, 4 * kRun keys at a time
#pragma unroll
            for (uint32_t w = 0; w < S::kGroups; ++w) {
                piece p_hi, p_lo;
#pragma unroll
                for (uint32_t k = 0; k < S::kRun; ++k) {
                    const float p = S::kRun == 8 ? score[k / 4][k % 4] : score[w][k];
                    p_hi[k] = P::head(p);
                    // the larger of the rest (no larger than the head, unless that is 0) and kLeast; without
                    // a head the rest itself
                    const float head = static_cast<float>(p_hi[k]);
                    p_lo[k] = static_cast<T>(__builtin_amdgcn_fmed3f(p - head, head, P::kLeast));
                }
#pragma unroll
                for (uint32_t s = 0; s < S::kValueSteps; ++s)
#pragma unroll
                    for (uint32_t e = 0; e < S::kValueRun; ++e) {
                        piece x;
#pragma unroll
                        for (uint32_t k = 0; k < S::kRun; ++k) x[k] = v[w][s][k][e];
                        o[s][e] = P::mma(x, p_hi, o[s][e]);
                        if (S::kRun == 8) o[s][e] = P::mma(x, p_lo, o[s][e]);
                    }
            }
        }
    };
    // Keys and values that no cache holds until the next step, and that no
    // other workgroup reads, are streamed (64 rows of 70B's heads over up to
    // 16384 keys: 378 us, 391 without).
    const uint64_t cache_bytes = static_cast<uint64_t>(item.keys) * 1024 * a.kv_heads * a.head_dim * 2 * sizeof(T);
    if (FULL && blocks == 1 && cache_bytes > kCacheBytes) run_tiles(std::true_type());
    else run_tiles(std::false_type());

    l = column_sum(l);
    if (quad == 0) {
        lds_m[wave][col] = m;
        lds_l[wave][col] = l;
    }
    if (col < heads) {
#pragma unroll
        for (uint32_t s = 0; s < S::kValueSteps; ++s)
#pragma unroll
            for (uint32_t e = 0; e < S::kValueRun; ++e)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
                    lds_o[wave][col][(s * 16 + 4 * quad + i) * S::kValueRun + e] = o[s][e][i];
    }
    __syncthreads();
    // The item's sums over its wavefronts: the row itself, or, unnormalised
    // and with their maximum and weight, a part of it.
    const bool whole = item.count == 1;
    const uint64_t slot0 = static_cast<uint64_t>(item.first) * a.heads + head0;
    // the scratch: every item's and head's sums, then their maxima and weights
    const rsrc_t part_o = device_buffer(a.partials + slot0 * a.head_dim);
    const rsrc_t part_ml =
        device_buffer(a.partials + static_cast<uint64_t>(a.n_items) * a.heads * a.head_dim + 2 * slot0);
    const uint32_t step = a.heads;   // of an item's heads among the slots
    T* const out = static_cast<T*>(a.out) + item.row * a.out_row + head0 * a.out_head;
    const uint32_t quads = a.head_dim / 4;   // runs of 4 elements of a head
    for (uint32_t i = threadIdx.x; i < heads * quads; i += kThreads) {
        const uint32_t h = i / quads, d = i % quads * 4;
        float top = -__builtin_inff();
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) top = fmaxf(top, lds_m[w][h]);
        const float base = finite_base(top);
        float weight = 0.0f;
        f32x4 sum = {};
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) {
            const float share = __builtin_amdgcn_exp2f(lds_m[w][h] - base);
            weight += share * lds_l[w][h];
            sum += share * *reinterpret_cast<const f32x4*>(&lds_o[w][h][d]);
        }
        if (whole) {
            store_row(out + h * a.out_head + d, sum, weight);
        } else {
            const uint32_t slot = static_cast<uint32_t>(item.index) * step + h;
            if (d == 0) put_pair(part_ml, 8 * slot, top, weight);
            put_four(part_o, 4 * (slot * a.head_dim + d), sum);
        }
    }
    if (whole) return;
    // The last of the row's items to arrive joins them all, in their order (a
    // launch of its own for that took 118 us in all where one row's 2001 keys
    // now take 8.7, and an arrival with a release fence 19).
    uint32_t* const counter = a.counters + static_cast<uint64_t>(item.first) * per_item + part;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wavefront's stores have arrived
    __syncthreads();
    if (threadIdx.x == 0)
        last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 ==
               static_cast<uint32_t>(item.count);
    __syncthreads();
    if (!last) return;
    if (threadIdx.x == 0) *counter = 0;   // for the next call
    // Each run of 4 elements of a head is joined by `subs` threads, each over
    // a share of the items, kBatch of them in flight at a time.
    const uint32_t n = static_cast<uint32_t>(item.count);
    const uint32_t runs = heads * quads, subs = max(kThreads / runs, 1u);
    float* const lds_sum = &lds_o[0][0][0];
    for (uint32_t i = threadIdx.x; i < runs * subs; i += kThreads) {
        const uint32_t run = i % runs, sub = i / runs, h = run / quads, d = run % quads * 4;
        const uint32_t k0 = sub * n / subs, k1 = (sub + 1) * n / subs;
        float top = -__builtin_inff(), weight = 0.0f;
        f32x4 sum = {};
        constexpr uint32_t kBatch = 8;
        for (uint32_t k = k0; k < k1; k += kBatch) {
            vec<float, 2> ml[kBatch];
            f32x4 x[kBatch];
#pragma unroll
            for (uint32_t j = 0; j < kBatch; ++j) {
                const uint32_t slot = min(k + j, k1 - 1) * step + h;
                ml[j] = get_pair(part_ml, 8 * slot);
                x[j] = get_four(part_o, 4 * (slot * a.head_dim + d));
            }
            float higher = top;
#pragma unroll
            for (uint32_t j = 0; j < kBatch; ++j) higher = fmaxf(higher, ml[j].x);
            const float base = finite_base(higher), fade = __builtin_amdgcn_exp2f(top - base);
            top = higher;
            weight *= fade;
            sum *= fade;
#pragma unroll
            for (uint32_t j = 0; j < kBatch; ++j) {
                const float share = __builtin_amdgcn_exp2f(ml[j].x - base);
                if (k + j < k1) {
                    weight += share * ml[j].y;
                    sum += share * x[j];
                }
            }
        }
        if (subs == 1) {
            store_row(out + h * a.out_head + d, sum, weight);
        } else {
            *reinterpret_cast<f32x4*>(lds_sum + i * 8) = sum;
            lds_sum[i * 8 + 4] = top;
            lds_sum[i * 8 + 5] = weight;
        }
    }
    if (subs == 1) return;
    __syncthreads();
    if (threadIdx.x < runs) {
        const uint32_t h = threadIdx.x / quads, d = threadIdx.x % quads * 4;
        float top = -__builtin_inff(), weight = 0.0f;
        for (uint32_t sub = 0; sub < subs; ++sub) top = fmaxf(top, lds_sum[(sub * runs + threadIdx.x) * 8 + 4]);
        const float base = finite_base(top);
        f32x4 sum = {};
        for (uint32_t sub = 0; sub < subs; ++sub) {
            const float* src = lds_sum + (sub * runs + threadIdx.x) * 8;
            const float share = __builtin_amdgcn_exp2f(src[4] - base);
            weight += share * src[5];
            sum += share * *reinterpret_cast<const f32x4*>(src);
        }
        store_row(out + h * a.out_head + d, sum, weight);
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
    const uint32_t units = a.n_items * a.kv_heads;
    const dim3 grid((units + kXcds - 1) / kXcds * kXcds * ((group + kHeads - 1) / kHeads));
    if (a.head_dim <= 32) launch_attention_dim<T, 32>(a, grid, stream);
    else if (a.head_dim <= 64) launch_attention_dim<T, 64>(a, grid, stream);
    else if (a.head_dim <= 128) launch_attention_dim<T, 128>(a, grid, stream);
    else launch_attention_dim<T, 256>(a, grid, stream);
}

}  // namespace

// The callers (capi_serving.cpp) have checked the arguments.

extern "C" int nz_hip_attention_plan(const int32_t* contexts, const int32_t* requests, uint32_t n_rows, uint32_t target,
                                     uint32_t parts, nz_attention_item* items, uint32_t* counters, void* stream,
                                     char* message, size_t message_size) {
    hipLaunchKernelGGL(nz_attention_plan_kernel, dim3(1), dim3(kPlanThreads), 0, static_cast<hipStream_t>(stream),
                       contexts, requests, n_rows, target, parts, items, counters);
    return launched("attention plan", message, message_size);
}

extern "C" int nz_hip_attention(const nz_attention_args* args, void* stream, char* message, size_t message_size) {
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (args->type == NZ_BF16) launch_attention<bf16_t>(*args, st);
    else if (args->type == NZ_FP16) launch_attention<_Float16>(*args, st);
    else launch_attention<float>(*args, st);
    return launched("attention", message, message_size);
}
