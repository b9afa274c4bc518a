// shared_attention_gfx950.hip -- attention over a paged key-value cache for
// rows that see the same keys: requests that begin with the same pages, and
// several rows of one request. The plan that finds such rows and cuts their
// keys into items (nz_shared_plan), and the kernels that run it
// (nz_shared_attention).
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <type_traits>

#include "attention_types.h"
#include "neuralzip_hip.h"
#include "serving_types.h"

namespace {

// ------------------------------------------------------------------- plan

constexpr uint32_t kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr uint32_t kMaxRows = NZ_SHARED_MAX_ROWS, kMaxGroups = NZ_SHARED_MAX_GROUPS, kColumns = NZ_SHARED_COLUMNS;
// Items start at multiples of kTile keys and are no shorter than one such tile
// for each wavefront of a workgroup.
constexpr uint32_t kTile = 32, kLeastItem = 128;

// Tiles are numbered group by group, then row by row; their keys are cut alike
// within a group.
struct PlanLds {
    uint32_t waves[kPlanWaves], counts[kPlanWaves];
    uint64_t keys[kPlanWaves];
    int32_t context[kMaxRows], request[kMaxRows], group[kMaxRows];
    uint32_t start[kMaxRows];                 // of the run of rows of one request
    uint32_t rank[kMaxRows];                  // among the rows of its group
    uint32_t own_first[kMaxRows + 1];         // first item of the tile that begins at a row
    uint32_t members[kMaxGroups], base[kMaxGroups], shared[kMaxGroups];
    int32_t least[kMaxGroups], most[kMaxGroups];   // requests of its rows
    uint32_t longest[kMaxGroups];             // context of them
    uint32_t group_first[kMaxGroups + 1];     // a group's first item
    uint32_t order[kMaxRows];                 // rows by group
};

// Inclusive prefix sum over the workgroup; total receives the sum.
__device__ __forceinline__ uint32_t plan_scan(uint32_t v, uint32_t& total, PlanLds& lds) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads();   // the last call's reads
    if (lane == 63) lds.waves[wave] = v;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kPlanWaves; ++w) {
        if (w < wave) before += lds.waves[w];
        total += lds.waves[w];
    }
    return before + v;
}

// Items of `keys` keys when none is longer than `share`.
__device__ __forceinline__ uint32_t cuts(uint32_t keys, uint32_t share) { return (keys + share - 1) / share; }

// One workgroup. Groups of which several requests have rows are read by tiles
// of as many rows as fit kColumns columns; then each request's rows in such
// tiles, from where the group's keys end. Latency bound.
__global__ __launch_bounds__(kPlanThreads) void nz_shared_plan_kernel(nz_shared_plan_args a) {
    __shared__ PlanLds lds;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = a.n_rows;
    const uint32_t heads = a.heads / a.kv_heads, tile_rows = heads <= kColumns ? kColumns / heads : 1;
    const uint32_t parts = a.kv_heads * ((heads + kColumns - 1) / kColumns);

    for (uint32_t g = threadIdx.x; g < a.n_groups; g += kPlanThreads) {
        lds.shared[g] = static_cast<uint32_t>(max(a.shared[g], 0));
        lds.members[g] = 0;
        lds.least[g] = 0x7FFFFFFF;
        lds.most[g] = -1;
        lds.longest[g] = 0;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) {
        const int32_t request = a.requests ? a.requests[i] : static_cast<int32_t>(i);
        const bool known = static_cast<uint32_t>(request) < a.n_requests;
        int32_t group = known && a.n_groups ? a.groups[request] : -1;
        if (static_cast<uint32_t>(group) >= a.n_groups || lds.shared[group] == 0) group = -1;
        lds.context[i] = known ? max(a.contexts[i], 0) : 0;
        lds.request[i] = known ? request : -1;
        lds.group[i] = group;
        if (group >= 0) {
            atomicMin(&lds.least[group], request);
            atomicMax(&lds.most[group], request);
            atomicMax(&lds.longest[group], static_cast<uint32_t>(lds.context[i]));
        }
    }
    __syncthreads();
    for (uint32_t g = threadIdx.x; g < a.n_groups; g += kPlanThreads)
        lds.shared[g] = min(lds.shared[g], lds.longest[g]);
    // Rows' places in their groups, in row order: by one wavefront, 64 rows at a time.
    if (wave == 0 && a.n_groups) {
        for (uint32_t i0 = 0; i0 < n; i0 += 64) {
            const uint32_t i = i0 + lane;
            int32_t group = i < n ? lds.group[i] : -1;
            // a group of one request is read with its own keys
            if (group >= 0 && lds.least[group] == lds.most[group]) group = -1;
            if (i < n) lds.group[i] = group;
            uint64_t left = __ballot(group >= 0);
            while (left) {
                const int32_t g = __builtin_amdgcn_readlane(group, __builtin_ctzll(left));
                const uint64_t same = __ballot(group == g);
                const uint32_t before = lds.members[g];
                if (group == g) lds.rank[i] = before + __popcll(same & ((1ull << lane) - 1));
                lds.members[g] = before + __popcll(same);   // by every lane
                left &= ~same;
            }
        }
    }
    __syncthreads();
    uint32_t placed = 0;
    for (uint32_t g0 = 0; g0 < a.n_groups; g0 += kPlanThreads) {
        const uint32_t g = g0 + threadIdx.x, count = g < a.n_groups ? lds.members[g] : 0;
        uint32_t total;
        const uint32_t upto = plan_scan(count, total, lds);
        if (g < a.n_groups) lds.base[g] = placed + upto - count;
        placed += total;
    }
    __syncthreads();
    uint64_t keys = 0;
    uint32_t longest = 0, tiles = 0;
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) {
        const int32_t group = lds.group[i];
        if (group >= 0) lds.order[lds.base[group] + lds.rank[i]] = i;
    }
    // runs of rows of one request
    uint32_t runs_before = 0;
    for (uint32_t i0 = 0; i0 < n; i0 += kPlanThreads) {
        const uint32_t i = i0 + threadIdx.x;
        const bool begins_run = i < n && (i == 0 || lds.request[i] < 0 || lds.request[i - 1] != lds.request[i]);
        uint32_t total;
        const uint32_t upto = plan_scan(begins_run, total, lds);
        if (i < n) lds.start[i] = runs_before + upto - 1;   // the run's number, for now
        if (begins_run) lds.own_first[runs_before + upto - 1] = i;
        runs_before += total;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) lds.start[i] = lds.own_first[lds.start[i]];
    __syncthreads();
    // Keys of the tile of its request's rows that begins at row i (0: no tile).
    const auto own_keys = [&](uint32_t i) -> uint32_t {
        if ((i - lds.start[i]) % tile_rows) return 0;
        uint32_t most = 0;
        for (uint32_t j = i; j < min(i + tile_rows, n) && lds.start[j] == lds.start[i]; ++j)
            most = max(most, static_cast<uint32_t>(lds.context[j]));
        const uint32_t from = lds.group[i] >= 0 ? lds.shared[lds.group[i]] : 0;
        return most > from ? most - from : 0;
    };
    const auto begins = [&](uint32_t i) { return (i - lds.start[i]) % tile_rows == 0; };
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) {
        const uint32_t own = own_keys(i);
        lds.own_first[i] = own;
        keys += own;
        longest = max(longest, own);
        tiles += begins(i);
    }
    for (uint32_t g = threadIdx.x; g < a.n_groups; g += kPlanThreads) {
        const uint32_t count = cuts(lds.members[g], tile_rows);
        if (count) longest = max(longest, lds.shared[g]);
        keys += static_cast<uint64_t>(count) * lds.shared[g];
        tiles += count;
    }
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        keys += __shfl_xor(keys, d);
        longest = max(longest, static_cast<uint32_t>(__shfl_xor(longest, d)));
        tiles += __shfl_xor(tiles, d);
    }
    if (lane == 0) lds.keys[wave] = keys, lds.waves[wave] = longest, lds.counts[wave] = tiles;
    __syncthreads();
    keys = 0, tiles = 0;
#pragma unroll
    for (uint32_t w = 0; w < kPlanWaves; ++w) {
        keys += lds.keys[w];
        longest = max(longest, lds.waves[w]);
        tiles += lds.counts[w];
    }
    __syncthreads();
    // The shortest length of items, in tiles of keys, that gives few enough.
    const uint32_t limit = min(cuts(max(a.target, tiles), a.target) * a.target, a.n_items);
    uint32_t lo = kLeastItem / kTile, hi = max((longest + kTile - 1) / kTile, lo);
    const auto count_items = [&](uint32_t share) {   // a wavefront's sum
        uint32_t sum = 0;
        for (uint32_t i = lane; i < n; i += 64)
            if (begins(i)) sum += max(cuts(lds.own_first[i], share), lds.group[i] < 0 ? 1u : 0u);
        for (uint32_t g = lane; g < a.n_groups; g += 64)
            sum += cuts(lds.members[g], tile_rows) * cuts(lds.shared[g], share);
        return last_lane(wave_scan(sum));
    };
    while (lo < hi) {
        const uint32_t step = (hi - lo + kPlanWaves) / (kPlanWaves + 1);
        const uint32_t tried = min(lo + wave * step, hi);
        const uint32_t count = count_items(tried * kTile);
        __syncthreads();
        if (lane == 0) lds.counts[wave] = count;
        __syncthreads();
        const uint64_t few = __ballot(lane < kPlanWaves && lds.counts[min(lane, kPlanWaves - 1)] <= limit);
        const uint32_t at = few ? __builtin_ctzll(few) : kPlanWaves;
        const uint32_t below = lo + at * step;
        if (at > 0) lo = min(below - step, hi) + 1;
        if (few) hi = min(below, hi);
    }
    const uint32_t share = lo * kTile;
    // a tile's items are of equal length, in whole kTile keys
    const auto each_of = [&](uint32_t length) {
        const uint32_t count = max(cuts(length, share), 1u);
        return max((cuts(length, count) + kTile - 1) / kTile * kTile, kTile);
    };
    __syncthreads();
    // first items: the groups', then the tiles of requests' rows
    uint32_t first = 0;
    for (uint32_t g0 = 0; g0 < a.n_groups; g0 += kPlanThreads) {
        const uint32_t g = g0 + threadIdx.x;
        const uint32_t count = g < a.n_groups ? cuts(lds.members[g], tile_rows) * cuts(lds.shared[g], each_of(lds.shared[g])) : 0;
        uint32_t total;
        const uint32_t upto = plan_scan(count, total, lds);
        if (g < a.n_groups) lds.group_first[g] = first + upto - count;
        first += total;
    }
    const uint32_t grouped = first;
    for (uint32_t i0 = 0; i0 < n; i0 += kPlanThreads) {
        const uint32_t i = i0 + threadIdx.x;
        uint32_t count = 0;
        if (i < n && begins(i)) {
            count = cuts(lds.own_first[i], each_of(lds.own_first[i]));
            if (count == 0 && lds.group[i] < 0) count = 1;   // rows without keys are written too
        }
        uint32_t total;
        const uint32_t upto = plan_scan(count, total, lds);
        if (i < n) lds.own_first[i] = first + upto - count;
        first += total;
    }
    if (threadIdx.x == 0) lds.own_first[n] = first, lds.group_first[a.n_groups] = grouped;
    __syncthreads();
    const int32_t total_keys = static_cast<int32_t>(min<uint64_t>((keys + 1023) / 1024, 0x7FFFFFFFu));
    // the items of the groups: parts of the keys, and within them tiles of rows, so that those that read the
    // same keys are neighbours
    for (uint32_t j = threadIdx.x; j < first; j += kPlanThreads) {
        nz_shared_item item;
        if (j < grouped) {
            uint32_t g = 0;
            {   // the last group that begins at or before j (groups without items begin where the next one does)
                uint32_t low = 0, high = a.n_groups;
                while (high - low > 1) {
                    const uint32_t mid = (low + high) >> 1;
                    if (lds.group_first[mid] <= j) low = mid;
                    else high = mid;
                }
                g = low;
            }
            const uint32_t count = cuts(lds.members[g], tile_rows), k = j - lds.group_first[g];
            const uint32_t tile = k % count, part = k / count, each = each_of(lds.shared[g]);
            item.member = static_cast<int32_t>(lds.base[g] + tile * tile_rows);
            item.rows = static_cast<int32_t>(min(tile_rows, lds.members[g] - tile * tile_rows));
            item.request = lds.request[lds.order[lds.base[g]]];
            item.begin = static_cast<int32_t>(part * each);
            item.end = static_cast<int32_t>(min(lds.shared[g], (part + 1) * each));
        } else {
            const uint32_t i = owner(lds.own_first, n, j);
            const uint32_t from = lds.group[i] >= 0 ? lds.shared[lds.group[i]] : 0, own = own_keys(i);
            const uint32_t each = each_of(own), part = j - lds.own_first[i];
            uint32_t rows = 1;
            while (rows < tile_rows && i + rows < n && lds.start[i + rows] == lds.start[i]) ++rows;
            item.member = static_cast<int32_t>(n + i);
            item.rows = static_cast<int32_t>(rows);
            item.request = lds.request[i];
            item.begin = static_cast<int32_t>(from + part * each);
            item.end = static_cast<int32_t>(from + min(own, (part + 1) * each));
        }
        item.keys = total_keys;
        item.reserved[0] = item.reserved[1] = 0;
        a.items[j] = item;
    }
    const nz_shared_item none = {-1, 0, -1, 0, 0, 0, {0, 0}};
    for (uint32_t j = first + threadIdx.x; j < a.n_items; j += kPlanThreads) a.items[j] = none;
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) {
        const int32_t g = lds.group[i];
        nz_shared_row row = {};
        if (g >= 0) {
            const uint32_t count = cuts(lds.members[g], tile_rows);
            row.group_first = static_cast<int32_t>(lds.group_first[g] + lds.rank[i] / tile_rows);
            row.group_step = static_cast<int32_t>(count);
            row.group_count = static_cast<int32_t>(cuts(lds.shared[g], each_of(lds.shared[g])));
            row.group_place = static_cast<int32_t>(lds.rank[i] % tile_rows);
            a.order[lds.base[g] + lds.rank[i]] = static_cast<int32_t>(i);
        }
        const uint32_t place = (i - lds.start[i]) % tile_rows, tile = i - place;
        row.own_first = static_cast<int32_t>(lds.own_first[tile]);
        // (rows inside a tile begin none: their first item is the next tile's)
        row.own_count = static_cast<int32_t>(lds.own_first[tile + 1] - lds.own_first[tile]);
        row.own_place = static_cast<int32_t>(place);
        row.context = lds.context[i];
        a.rows[i] = row;
        a.order[n + i] = static_cast<int32_t>(i);
    }
    for (uint64_t i = threadIdx.x; i < static_cast<uint64_t>(n) * parts; i += kPlanThreads) a.counters[i] = 0;
}

// -------------------------------------------------------------- attention

constexpr uint32_t kWaves = 4, kThreads = 64 * kWaves;
// Columns that a wavefront takes at once, in matrix instructions of 16.
constexpr uint32_t kBlocks = kColumns / 16;

// One item: the softmax of up to kColumns columns -- rows that see the same
// keys, times the query heads of one key-value head -- over the keys begin ..
// end - 1, tile by tile with a running maximum and sum per column, each over
// the keys below its row's context (see nz_attention_kernel, whose product
// layout this has, for a tile of one row).
template <typename T, uint32_t DP, bool FULL>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(DP <= 128 && sizeof(T) == 2 ? 2 : 1)))
void nz_shared_attention_kernel(nz_shared_attention_args a) {
    using S = Shape<T, DP>;
    using P = Piece<T>;
    using piece = typename P::type;
    using value_run = vec<T, S::kValueRun>;
    __shared__ float lds_m[kWaves][kColumns], lds_l[kWaves][kColumns];
    __shared__ __align__(16) float lds_o[kWaves][kColumns][DP + 4];
    __shared__ uint32_t ended[kColumns], n_ended;

    const uint32_t group = a.heads / a.kv_heads, blocks = (group + kColumns - 1) / kColumns;
    const uint32_t turn = blockIdx.x / kXcds, unit = turn / blocks * kXcds + blockIdx.x % kXcds, block = turn % blocks;
    const uint32_t which = unit / a.kv_heads, kv_head = unit % a.kv_heads;
    if (which >= a.n_items) return;
    const nz_shared_item item = a.items[which];
    if (item.rows <= 0) return;
    const uint32_t parts = a.kv_heads * blocks, part = kv_head * blocks + block;
    const uint32_t head0 = kv_head * group + block * kColumns;
    const uint32_t heads = min(kColumns, (kv_head + 1) * group - head0);   // of a row
    const uint32_t columns = static_cast<uint32_t>(item.rows) * heads;
    const int32_t* const members = a.order + item.member;
    const uint32_t lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t shift = 31 - __clz(a.page_size), place_mask = a.page_size - 1;
    const uint32_t end = static_cast<uint32_t>(item.end);
    const bool known = static_cast<uint32_t>(item.request) < a.n_requests;
    const int32_t* table = a.tables + static_cast<uint64_t>(known ? item.request : 0) * a.max_pages;
    const float scale = a.scale * kLog2e;
    const T* const key_base = static_cast<const T*>(a.key_cache) + kv_head * a.key_head;
    const T* const value_base = static_cast<const T*>(a.value_cache) + kv_head * a.value_head;

    auto run_tiles = [&](auto width) {
        constexpr uint32_t NT = decltype(width)::value;
        piece q[NT][S::kKeySteps];
        uint32_t limit[NT], lowest = end;   // keys that a column sees
#pragma unroll
        for (uint32_t b = 0; b < NT; ++b) {
            const uint32_t c = b * 16 + col;
            const bool used = c < columns;
            const uint32_t row = used ? static_cast<uint32_t>(members[c / heads]) : 0;
            limit[b] = used ? min(static_cast<uint32_t>(max(a.rows[row].context, 0)), end) : 0;
            if (used) lowest = min(lowest, limit[b]);
            const T* src = static_cast<const T*>(a.q) + row * a.q_row + (head0 + c % heads) * a.q_head;
#pragma unroll
            for (uint32_t s = 0; s < S::kKeySteps; ++s) {
                const uint32_t d = s * 4 * S::kRun + quad * S::kRun;
                q[b][s] = piece{};
                if (used && (FULL || d < a.head_dim)) q[b][s] = *reinterpret_cast<const piece*>(src + d);
            }
        }
#pragma unroll
        for (uint32_t d = 1; d < 16; d <<= 1) lowest = min(lowest, static_cast<uint32_t>(__shfl_xor(lowest, d)));
        f32x4 o[NT][S::kValueSteps][S::kValueRun] = {};
        float m[NT], l[NT];
#pragma unroll
        for (uint32_t b = 0; b < NT; ++b) m[b] = -__builtin_inff(), l[b] = 0.0f;

        // The pages of a tile's runs of 16 keys (a run lies in one page), a
        // tile ahead of the keys, and keys a tile ahead of their products.
        // Past the end, and where there is no page, page 0 is read and
        // everything masked.
        auto entries = [&](uint32_t t0, int32_t (&page)[S::kHalves]) {
#pragma unroll
            for (uint32_t h = 0; h < S::kHalves; ++h) {
                const uint32_t t = t0 + 16 * h, entry = t >> shift;
                page[h] = table[min(entry, a.max_pages - 1)];
                if (!known || t >= end || entry >= a.max_pages) page[h] = -1;
            }
        };
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
                    if (FULL || d < a.head_dim) keys[h][s] = *reinterpret_cast<const piece*>(src + col * a.key_slot + d);
                }
            }
        };
        constexpr uint32_t kStep = kWaves * S::kKeys;
        uint32_t t0 = static_cast<uint32_t>(item.begin) / 16 * 16 + wave * S::kKeys;
        const uint32_t begin = static_cast<uint32_t>(item.begin);
        int32_t page[S::kHalves], next[S::kHalves];
        if (t0 < end) {
            entries(t0, page);
            load_keys(t0, page);
            entries(t0 + kStep, next);
        }
        for (; t0 < end; t0 += kStep) {
            const T* values[S::kHalves];
            bool valid[S::kHalves];
#pragma unroll
            for (uint32_t h = 0; h < S::kHalves; ++h) {
                valid[h] = static_cast<uint32_t>(page[h]) < a.n_pages;
                const int64_t p = valid[h] ? page[h] : 0;
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
                            v[w][s][k] = *reinterpret_cast<const value_run*>(values[h] + place * a.value_slot + d);
                    }
            float score[NT][S::kHalves][4];
#pragma unroll
            for (uint32_t h = 0; h < S::kHalves; ++h)
#pragma unroll
                for (uint32_t b = 0; b < NT; ++b) {
                    f32x4 acc = {};
#pragma unroll
                    for (uint32_t s = 0; s < S::kKeySteps; ++s) acc = P::mma(keys[h][s], q[b][s], acc);
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        const uint32_t t = t0 + 16 * h + 4 * quad + i;
                        score[b][h][i] = valid[h] && t >= begin && t < limit[b] ? acc[i] * scale : -__builtin_inff();
                    }
                }
            // every column of the item sees every key of the tile
            const bool even = t0 >= begin && t0 + S::kKeys <= lowest && valid[0] && valid[S::kHalves - 1];
            if (t0 + kStep < end) {
                load_keys(t0 + kStep, next);
#pragma unroll
                for (uint32_t h = 0; h < S::kHalves; ++h) page[h] = next[h];
                entries(t0 + 2 * kStep, next);
            }
#pragma unroll
            for (uint32_t b = 0; b < NT; ++b) {
                float top = m[b];
#pragma unroll
                for (uint32_t h = 0; h < S::kHalves; ++h)
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) top = fmaxf(top, score[b][h][i]);
                top = column_max(top);
                const float base = finite_base(top);
                const float fade = __builtin_amdgcn_exp2f(m[b] - base);
                m[b] = top;
                l[b] *= fade;
#pragma unroll
                for (uint32_t s = 0; s < S::kValueSteps; ++s)
#pragma unroll
                    for (uint32_t e = 0; e < S::kValueRun; ++e) o[b][s][e] *= fade;
#pragma unroll
                for (uint32_t h = 0; h < S::kHalves; ++h)
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        score[b][h][i] = __builtin_amdgcn_exp2f(score[b][h][i] - (base - P::kLift));
                        l[b] += score[b][h][i];
                    }
            }
            // the products with the values, 4 * kRun keys at a time
            auto weights = [&](uint32_t b, uint32_t w, piece& p_hi, piece& p_lo) {
#pragma unroll
                for (uint32_t k = 0; k < S::kRun; ++k) {
                    const float p = S::kRun == 8 ? score[b][k / 4][k % 4] : score[b][w][k];
                    p_hi[k] = P::head(p);
                    const float head = static_cast<float>(p_hi[k]);
                    p_lo[k] = static_cast<T>(__builtin_amdgcn_fmed3f(p - head, head, P::kLeast));
                }
            };
            if (even) {
#pragma unroll
                for (uint32_t w = 0; w < S::kGroups; ++w) {
                    piece p_hi[NT], p_lo[NT];
#pragma unroll
                    for (uint32_t b = 0; b < NT; ++b) weights(b, w, p_hi[b], p_lo[b]);
#pragma unroll
                    for (uint32_t s = 0; s < S::kValueSteps; ++s)
#pragma unroll
                        for (uint32_t e = 0; e < S::kValueRun; ++e) {
                            piece x;
#pragma unroll
                            for (uint32_t k = 0; k < S::kRun; ++k) x[k] = v[w][s][k][e];
#pragma unroll
                            for (uint32_t b = 0; b < NT; ++b) {
                                o[b][s][e] = P::mma(x, p_hi[b], o[b][s][e]);
                                if (S::kRun == 8) o[b][s][e] = P::mma(x, p_lo[b], o[b][s][e]);
                            }
                        }
                }
            } else {
                // Some columns see fewer of these keys than others, and the
                // values of keys that they don't see may be anything, NaN
                // among it: the columns of each limit in turn, with the
                // values past it as zeros.
#pragma unroll
                for (uint32_t b = 0; b < NT; ++b) {
                    uint64_t left = __ballot(b * 16 + col < columns);
                    while (left) {
                        const uint32_t seen = static_cast<uint32_t>(
                            __builtin_amdgcn_readlane(static_cast<int>(limit[b]), __builtin_ctzll(left)));
                        const bool mine = limit[b] == seen;
                        left &= ~__ballot(mine);
#pragma unroll
                        for (uint32_t w = 0; w < S::kGroups; ++w) {
                            piece p_hi, p_lo;
                            weights(b, w, p_hi, p_lo);
#pragma unroll
                            for (uint32_t s = 0; s < S::kValueSteps; ++s)
#pragma unroll
                                for (uint32_t e = 0; e < S::kValueRun; ++e) {
                                    piece x;
#pragma unroll
                                    for (uint32_t k = 0; k < S::kRun; ++k) {
                                        const uint32_t h = S::kRun == 8 ? k / 4 : w;
                                        const uint32_t t = t0 + 16 * h + 4 * quad + k % 4;
                                        x[k] = valid[h] && t >= begin && t < seen ? v[w][s][k][e] : T{};
                                    }
                                    f32x4 sum = P::mma(x, p_hi, o[b][s][e]);
                                    if (S::kRun == 8) sum = P::mma(x, p_lo, sum);
#pragma unroll
                                    for (uint32_t i = 0; i < 4; ++i) o[b][s][e][i] = mine ? sum[i] : o[b][s][e][i];
                                }
                        }
                    }
                }
            }
        }
#pragma unroll
        for (uint32_t b = 0; b < NT; ++b) {
            l[b] = column_sum(l[b]);
            const uint32_t c = b * 16 + col;
            if (quad == 0) {
                lds_m[wave][c] = m[b];
                lds_l[wave][c] = l[b];
            }
            if (c < columns) {
#pragma unroll
                for (uint32_t s = 0; s < S::kValueSteps; ++s)
#pragma unroll
                    for (uint32_t e = 0; e < S::kValueRun; ++e)
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i)
                            lds_o[wave][c][(s * 16 + 4 * quad + i) * S::kValueRun + e] = o[b][s][e][i];
            }
        }
    };
    if (columns <= 16) run_tiles(std::integral_constant<uint32_t, 1>());
    else run_tiles(std::integral_constant<uint32_t, kBlocks>());
    __syncthreads();

    // The item's sums over its wavefronts: rows of one item are done, of the
    // others they are parts, unnormalised and with their maximum and weight.
    const uint32_t quads = a.head_dim / 4;   // runs of 4 elements of a head
    const uint32_t width = parts * kColumns;   // an item's slots
    const auto slot_of = [&](uint32_t which_item, uint32_t column) {
        return which_item * width + part * kColumns + column;
    };
    float* const part_o = a.partials;
    float* const part_ml = a.partials + static_cast<uint64_t>(a.n_items) * width * a.head_dim;
    const rsrc_t all_o = device_buffer(part_o), all_ml = device_buffer(part_ml);
    T* const out = static_cast<T*>(a.out);
    for (uint32_t i = threadIdx.x; i < columns * quads; i += kThreads) {
        const uint32_t c = i / quads, d = i % quads * 4;
        float top = -__builtin_inff();
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) top = fmaxf(top, lds_m[w][c]);
        const float base = finite_base(top);
        float weight = 0.0f;
        f32x4 sum = {};
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) {
            const float share = __builtin_amdgcn_exp2f(lds_m[w][c] - base);
            weight += share * lds_l[w][c];
            sum += share * *reinterpret_cast<const f32x4*>(&lds_o[w][c][d]);
        }
        const uint32_t row = static_cast<uint32_t>(members[c / heads]);
        if (a.rows[row].group_count + a.rows[row].own_count == 1) {
            store_row(out + row * a.out_row + (head0 + c % heads) * a.out_head + d, sum, weight);
        } else {
            const uint32_t slot = slot_of(which, c);
            if (d == 0) put_pair(all_ml, 8 * slot, top, weight);
            put_four(all_o, 4 * (slot * a.head_dim + d), sum);
        }
    }
    // The last of a row's items to arrive joins them all, in their order.
    if (threadIdx.x == 0) n_ended = 0;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wavefront's stores have arrived
    __syncthreads();
    if (threadIdx.x < static_cast<uint32_t>(item.rows)) {
        const uint32_t row = static_cast<uint32_t>(members[threadIdx.x]);
        const uint32_t count = static_cast<uint32_t>(a.rows[row].group_count + a.rows[row].own_count);
        if (count > 1) {
            uint32_t* const counter = a.counters + static_cast<uint64_t>(row) * parts + part;
            if (__hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == count) {
                ended[atomicAdd(&n_ended, 1u)] = row;
                *counter = 0;   // for the next call
            }
        }
    }
    __syncthreads();
    // A run of 4 elements of a head: its items kBatch at a time, which are in
    // flight together and summed from their own maximum, then the batches in
    // their order. So the result is the same whether one thread takes them all
    // or, where a single row ended, one thread each batch.
    constexpr uint32_t kBatch = 8;
    const uint32_t row_runs = heads * quads, runs = n_ended * row_runs;
    if (runs == 0) return;
    struct Sums {
        f32x4 sum;
        float top, weight;
    };
    const auto batch_of = [&](const nz_shared_row& r, uint32_t k, uint32_t h, uint32_t d) {
        const uint32_t groups = static_cast<uint32_t>(r.group_count), n = groups + static_cast<uint32_t>(r.own_count);
        vec<float, 2> ml[kBatch];
        f32x4 x[kBatch];
#pragma unroll
        for (uint32_t j = 0; j < kBatch; ++j) {
            const uint32_t at = min(k + j, n - 1);
            const uint32_t from = at < groups ? r.group_first + at * r.group_step : r.own_first + (at - groups);
            const uint32_t place = static_cast<uint32_t>(at < groups ? r.group_place : r.own_place);
            const uint32_t slot = slot_of(from, place * heads + h);
            ml[j] = get_pair(all_ml, 8 * slot);
            x[j] = get_four(all_o, 4 * (slot * a.head_dim + d));
        }
        Sums s = {{}, -__builtin_inff(), 0.0f};
#pragma unroll
        for (uint32_t j = 0; j < kBatch; ++j) s.top = fmaxf(s.top, ml[j].x);
        const float base = finite_base(s.top);
#pragma unroll
        for (uint32_t j = 0; j < kBatch; ++j) {
            const float share = __builtin_amdgcn_exp2f(ml[j].x - base);
            if (k + j < n) {
                s.weight += share * ml[j].y;
                s.sum += share * x[j];
            }
        }
        return s;
    };
    const auto join = [](Sums& s, const Sums& more) {
        const float top = fmaxf(s.top, more.top), base = finite_base(top);
        const float fade = __builtin_amdgcn_exp2f(s.top - base), share = __builtin_amdgcn_exp2f(more.top - base);
        s.sum = fade * s.sum + share * more.sum;
        s.weight = fade * s.weight + share * more.weight;
        s.top = top;
    };
    const nz_shared_row first = a.rows[ended[0]];
    const uint32_t batches = (static_cast<uint32_t>(first.group_count + first.own_count) + kBatch - 1) / kBatch;
    // (the wavefronts' sums have been read)
    if (n_ended == 1 && batches > 1 && 2 * runs <= kThreads && runs * batches * sizeof(Sums) <= sizeof(lds_o)) {
        Sums* const all = reinterpret_cast<Sums*>(&lds_o[0][0][0]);
        for (uint32_t i = threadIdx.x; i < runs * batches; i += kThreads)
            all[i] = batch_of(first, i / runs * kBatch, i % runs / quads, i % quads * 4);
        __syncthreads();
        if (threadIdx.x < runs) {
            Sums s = all[threadIdx.x];
            for (uint32_t k = 1; k < batches; ++k) join(s, all[k * runs + threadIdx.x]);
            store_row(out + ended[0] * a.out_row + (head0 + threadIdx.x / quads) * a.out_head + threadIdx.x % quads * 4, s.sum,
                      s.weight);
        }
        return;
    }
    for (uint32_t i = threadIdx.x; i < runs; i += kThreads) {
        const uint32_t row = ended[i / row_runs], h = i % row_runs / quads, d = i % quads * 4;
        const nz_shared_row r = a.rows[row];
        const uint32_t n = static_cast<uint32_t>(r.group_count + r.own_count);
        Sums s = batch_of(r, 0, h, d);
        for (uint32_t k = kBatch; k < n; k += kBatch) join(s, batch_of(r, k, h, d));
        store_row(out + row * a.out_row + (head0 + h) * a.out_head + d, s.sum, s.weight);
    }
}

template <typename T, uint32_t DP>
void launch_dim(const nz_shared_attention_args& a, dim3 grid, hipStream_t stream) {
    if (a.head_dim == DP) hipLaunchKernelGGL((nz_shared_attention_kernel<T, DP, true>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((nz_shared_attention_kernel<T, DP, false>), grid, dim3(kThreads), 0, stream, a);
}

template <typename T>
void launch_shared(const nz_shared_attention_args& a, hipStream_t stream) {
    const uint32_t group = a.heads / a.kv_heads;
    const uint32_t units = a.n_items * a.kv_heads;
    const dim3 grid((units + kXcds - 1) / kXcds * kXcds * ((group + kColumns - 1) / kColumns));
    if (a.head_dim <= 32) launch_dim<T, 32>(a, grid, stream);
    else if (a.head_dim <= 64) launch_dim<T, 64>(a, grid, stream);
    else if (a.head_dim <= 128) launch_dim<T, 128>(a, grid, stream);
    else launch_dim<T, 256>(a, grid, stream);
}

}  // namespace

// The callers (capi_serving.cpp) have checked the arguments.

extern "C" int nz_hip_shared_plan(const nz_shared_plan_args* args, void* stream, char* message, size_t message_size) {
    hipLaunchKernelGGL(nz_shared_plan_kernel, dim3(1), dim3(kPlanThreads), 0, static_cast<hipStream_t>(stream), *args);
    return launched("shared attention plan", message, message_size);
}

extern "C" int nz_hip_shared_attention(const nz_shared_attention_args* args, void* stream, char* message,
                                       size_t message_size) {
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (args->type == NZ_BF16) launch_shared<bf16_t>(*args, st);
    else if (args->type == NZ_FP16) launch_shared<_Float16>(*args, st);
    else launch_shared<float>(*args, st);
    return launched("shared attention", message, message_size);
}
