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
// Items are cut to lengths of whole tiles of kTile keys, from wherever their
// keys begin; the last one of a row or group has what is left. The least length
// that they are cut to is a tile for each wavefront of a workgroup.
constexpr uint32_t kTile = 32, kLeastItem = 128;
// Keys of a group, which its other items read too, take about half as long as
// a row's own, which come from memory. (32 requests behind 8176 keys: 48 us
// against 51 with items of one length and no more of them; 64 over three
// prefixes of 16384 keys: 275 against 315.)
constexpr uint32_t kGroupLength = 2;

struct PlanLds {
    uint32_t waves[kPlanWaves], counts[kPlanWaves];
    uint64_t keys[kPlanWaves];
    int32_t request[kMaxRows], group[kMaxRows];
    uint32_t context[kMaxRows];
    uint32_t start[kMaxRows];                 // of the run of rows that are read together
    uint32_t rank[kMaxRows];                  // among the rows of its group
    uint32_t own[kMaxRows + 1];               // keys, then first item, of the tile that begins at a row (0: none does)
    uint32_t tail[kMaxRows + 1];              // the same of what a row alone sees
    uint32_t members[kMaxGroups], base[kMaxGroups], shared[kMaxGroups];
    int32_t least[kMaxGroups], most[kMaxGroups];   // requests of its rows
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

// One workgroup. Three kinds of items: the shared keys of groups of which
// several requests have rows, for tiles of as many rows as fit kColumns
// columns; the other keys that all of a tile of neighbouring rows of one
// request see; and what a row sees past those of its tile. So every row of an
// item sees all of its keys. Items of a key or of none count against the limit
// as others do: eight requests of eight rows have 64 pieces, as many as the
// items of 32 heads over 8, and their 8000 keys stay uncut (103 us; 53 at the
// rate of a copy). Once a step for all layers, and bound by the
// latencies of its scans and of the search for the items' length: 10.0 us for
// 5 rows, 12.0 for 32, 13.7 for 128 in three groups.
__global__ __launch_bounds__(kPlanThreads) void nz_shared_plan_kernel(nz_shared_plan_args a) {
    __shared__ PlanLds lds;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = a.n_rows;
    const uint32_t heads = a.heads / a.kv_heads, tile_rows = heads <= kColumns ? kColumns / heads : 1;

    for (uint32_t g = threadIdx.x; g < a.n_groups; g += kPlanThreads) {
        lds.shared[g] = static_cast<uint32_t>(max(a.shared[g], 0));
        lds.members[g] = 0;
        lds.least[g] = 0x7FFFFFFF;
        lds.most[g] = -1;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) {
        const int32_t request = a.requests ? a.requests[i] : static_cast<int32_t>(i);
        const bool known = static_cast<uint32_t>(request) < a.n_requests;
        const uint32_t context = known ? static_cast<uint32_t>(max(a.contexts[i], 0)) : 0;
        int32_t group = known && a.n_groups ? a.groups[request] : -1;
        // a row that sees less than its group shares is read by itself
        if (static_cast<uint32_t>(group) >= a.n_groups || lds.shared[group] == 0 || lds.shared[group] > context) group = -1;
        lds.context[i] = context;
        lds.request[i] = known ? request : -1;
        lds.group[i] = group;
        if (group >= 0) {
            atomicMin(&lds.least[group], request);
            atomicMax(&lds.most[group], request);
        }
    }
    __syncthreads();
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
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) {
        const int32_t group = lds.group[i];
        if (group >= 0) lds.order[lds.base[group] + lds.rank[i]] = i;
    }
    // runs of rows of one request, all of them in its group or none
    uint32_t runs_before = 0;
    for (uint32_t i0 = 0; i0 < n; i0 += kPlanThreads) {
        const uint32_t i = i0 + threadIdx.x;
        const bool begins_run = i < n && (i == 0 || lds.request[i] < 0 || lds.request[i - 1] != lds.request[i] ||
                                          lds.group[i - 1] != lds.group[i]);
        uint32_t total;
        const uint32_t upto = plan_scan(begins_run, total, lds);
        if (i < n) lds.start[i] = runs_before + upto - 1;   // the run's number, for now
        if (begins_run) lds.own[runs_before + upto - 1] = i;
        runs_before += total;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) lds.start[i] = lds.own[lds.start[i]];
    __syncthreads();
    // The tile of its request's rows that a row is in: its first row, rows, and where the keys begin and end that
    // all of them see.
    struct Tile {
        uint32_t first, rows, begin, end;
    };
    const auto tile_of = [&](uint32_t i) {
        const uint32_t start = lds.start[i];
        Tile t = {i - (i - start) % tile_rows, 0, 0, 0xFFFFFFFFu};
        while (t.rows < tile_rows && t.first + t.rows < n && lds.start[t.first + t.rows] == start)
            t.end = min(t.end, lds.context[t.first + t.rows++]);
        t.begin = lds.group[i] >= 0 ? lds.shared[lds.group[i]] : 0;
        return t;
    };
    uint64_t keys = 0;
    uint32_t longest = 0, pieces = 0;
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) {
        const Tile t = tile_of(i);
        const uint32_t own = t.first == i ? t.end - t.begin : 0, tail = lds.context[i] - t.end;
        lds.own[i] = own;
        lds.tail[i] = tail;
        keys += own + tail;
        longest = max(longest, max(own, tail));
        // (a row without any keys is an item too)
        pieces += (own > 0) + (tail > 0 || lds.context[i] == 0);
    }
    for (uint32_t g = threadIdx.x; g < a.n_groups; g += kPlanThreads) {
        const uint32_t count = cuts(lds.members[g], tile_rows);
        if (count) longest = max(longest, lds.shared[g]);
        keys += static_cast<uint64_t>(count) * lds.shared[g];
        pieces += count;
    }
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        keys += __shfl_xor(keys, d);
        longest = max(longest, static_cast<uint32_t>(__shfl_xor(longest, d)));
        pieces += __shfl_xor(pieces, d);
    }
    if (lane == 0) lds.keys[wave] = keys, lds.waves[wave] = longest, lds.counts[wave] = pieces;
    __syncthreads();
    keys = 0, pieces = 0;
#pragma unroll
    for (uint32_t w = 0; w < kPlanWaves; ++w) {
        keys += lds.keys[w];
        longest = max(longest, lds.waves[w]);
        pieces += lds.counts[w];
    }
    __syncthreads();
    // The shortest length of items, in tiles of keys, that gives few enough: half more of them where there are
    // groups, whose items are up to kGroupLength times as long as the others.
    const uint32_t whole_rounds = cuts(max(a.target, pieces), a.target) * a.target;
    const uint32_t limit = min(a.n_groups ? whole_rounds + whole_rounds / 2 : whole_rounds, a.n_items);
    uint32_t lo = kLeastItem / kTile, hi = max((longest + kTile - 1) / kTile, lo);
    const auto group_share = [](uint32_t share) { return share < 1u << 30 ? kGroupLength * share : share; };
    const auto count_items = [&](uint32_t share) {   // a wavefront's sum, or as much as is too many
        uint64_t sum = 0;
        for (uint32_t i = lane; i < n; i += 64)
            sum += cuts(lds.own[i], share) + max(cuts(lds.tail[i], share), lds.context[i] == 0 ? 1u : 0u);
        for (uint32_t g = lane; g < a.n_groups; g += 64)
            sum += static_cast<uint64_t>(cuts(lds.members[g], tile_rows)) * cuts(lds.shared[g], group_share(share));
        return last_lane(wave_scan(static_cast<uint32_t>(min<uint64_t>(sum, 1u << 25))));
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
    // items are of equal length, in whole kTile keys
    const auto each_of = [&](uint32_t length, uint32_t most) {
        const uint32_t count = max(cuts(length, most), 1u);
        return max((cuts(length, count) + kTile - 1) / kTile * kTile, kTile);
    };
    const auto items_of = [&](uint32_t length) { return cuts(length, each_of(length, share)); };
    const auto group_each = [&](uint32_t g) { return each_of(lds.shared[g], group_share(share)); };
    const auto group_items = [&](uint32_t g) { return cuts(lds.shared[g], group_each(g)); };
    __syncthreads();
    // first items, kind by kind
    uint32_t first = 0;
    for (uint32_t g0 = 0; g0 < a.n_groups; g0 += kPlanThreads) {
        const uint32_t g = g0 + threadIdx.x;
        const uint32_t count = g < a.n_groups ? cuts(lds.members[g], tile_rows) * group_items(g) : 0;
        uint32_t total;
        const uint32_t upto = plan_scan(count, total, lds);
        if (g < a.n_groups) lds.group_first[g] = first + upto - count;
        first += total;
    }
    const uint32_t grouped = first;
    for (uint32_t i0 = 0; i0 < n; i0 += kPlanThreads) {
        const uint32_t i = i0 + threadIdx.x, count = i < n ? items_of(lds.own[i]) : 0;
        uint32_t total;
        const uint32_t upto = plan_scan(count, total, lds);
        if (i < n) lds.own[i] = first + upto - count;
        first += total;
    }
    const uint32_t owned = first;
    for (uint32_t i0 = 0; i0 < n; i0 += kPlanThreads) {
        const uint32_t i = i0 + threadIdx.x;
        const uint32_t count = i < n ? max(items_of(lds.tail[i]), lds.context[i] == 0 ? 1u : 0u) : 0;
        uint32_t total;
        const uint32_t upto = plan_scan(count, total, lds);
        if (i < n) lds.tail[i] = first + upto - count;
        first += total;
    }
    if (threadIdx.x == 0) lds.group_first[a.n_groups] = grouped, lds.own[n] = owned, lds.tail[n] = first;
    __syncthreads();
    const int32_t total_keys = static_cast<int32_t>(min<uint64_t>((keys + 1023) / 1024, 0x7FFFFFFFu));
    for (uint32_t j = threadIdx.x; j < first; j += kPlanThreads) {
        nz_shared_item item;
        if (j < grouped) {
            // parts of the keys, and within them tiles of rows, so that those that read the same keys are neighbours
            // (groups without items begin where the next one does)
            const uint32_t g = owner(lds.group_first, a.n_groups, j);
            const uint32_t count = cuts(lds.members[g], tile_rows), k = j - lds.group_first[g];
            const uint32_t tile = k % count, part = k / count, each = group_each(g);
            item.member = static_cast<int32_t>(lds.base[g] + tile * tile_rows);
            item.rows = static_cast<int32_t>(min(tile_rows, lds.members[g] - tile * tile_rows));
            item.request = lds.request[lds.order[lds.base[g]]];
            item.begin = static_cast<int32_t>(part * each);
            item.end = static_cast<int32_t>(min(lds.shared[g], (part + 1) * each));
        } else if (j < owned) {
            const uint32_t i = owner(lds.own, n, j);
            const Tile t = tile_of(i);
            const uint32_t each = each_of(t.end - t.begin, share), part = j - lds.own[i];
            item.member = static_cast<int32_t>(n + i);
            item.rows = static_cast<int32_t>(t.rows);
            item.request = lds.request[i];
            item.begin = static_cast<int32_t>(t.begin + part * each);
            item.end = static_cast<int32_t>(min(t.end, t.begin + (part + 1) * each));
        } else {
            const uint32_t i = owner(lds.tail, n, j);
            const Tile t = tile_of(i);
            const uint32_t each = each_of(lds.context[i] - t.end, share), part = j - lds.tail[i];
            item.member = static_cast<int32_t>(n + i);
            item.rows = 1;
            item.request = lds.request[i];
            item.begin = static_cast<int32_t>(t.end + part * each);
            item.end = static_cast<int32_t>(min(lds.context[i], t.end + (part + 1) * each));
        }
        item.keys = total_keys;
        item.reserved[0] = item.reserved[1] = 0;
        a.items[j] = item;
    }
    const nz_shared_item none = {-1, 0, -1, 0, 0, 0, {0, 0}};
    for (uint32_t j = first + threadIdx.x; j < a.n_items; j += kPlanThreads) a.items[j] = none;
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) {
        const int32_t g = lds.group[i];
        const Tile t = tile_of(i);
        nz_shared_row row = {};
        uint32_t place = 0;
        if (g >= 0) {
            row.group_first = static_cast<int32_t>(lds.group_first[g] + lds.rank[i] / tile_rows);
            row.group_step = static_cast<int32_t>(cuts(lds.members[g], tile_rows));
            row.group_count = static_cast<int32_t>(group_items(g));
            place = lds.rank[i] % tile_rows;
            a.order[lds.base[g] + lds.rank[i]] = static_cast<int32_t>(i);
        }
        // (a row that begins no tile has no items there: its first is the next one's)
        row.own_first = static_cast<int32_t>(lds.own[t.first]);
        row.own_count = static_cast<int32_t>(lds.own[t.first + 1] - lds.own[t.first]);
        row.tail_first = static_cast<int32_t>(lds.tail[i]);
        row.tail_count = static_cast<int32_t>(lds.tail[i + 1] - lds.tail[i]);
        row.places = static_cast<int32_t>(place | (i - t.first) << 8);
        a.rows[i] = row;
        a.order[n + i] = static_cast<int32_t>(i);
    }
}

// -------------------------------------------------------------- attention

constexpr uint32_t kWaves = 4, kThreads = 64 * kWaves;
// Columns that a wavefront takes at once, in matrix instructions of 16.
constexpr uint32_t kBlocks = kColumns / 16;

// One item: the softmax of up to kColumns columns -- rows that see the same
// keys, times the query heads of one key-value head -- over the keys begin ..
// end - 1, tile by tile with a running maximum and sum per column (see
// nz_attention_kernel, whose product layout this has). Each wavefront takes
// every fourth tile for all columns; no LDS and no barrier in the loop.
//
// Where most keys are rows' own, memory bounds it: 32 rows of 32 heads over 8
// behind 8176 keys, 161 MB in 47 us. Where most are a group's, they come out of
// the L2 and two things do at two workgroups a compute unit, the softmax on the
// vector units (busy 50 % of the time; the matrix units 26 %) and the waits for
// keys and values (24 to 33 %): 128 rows of 64 heads over 8 behind three
// prefixes of 16384 keys, 74 GFLOP in 258 us. That one took 311 against then
// 252 us (without its rows' own keys) with the wavefronts sharing tiles and
// taking a block of columns each, 271 to 282 with keys passed through LDS and
// 327 with values; leaving out the rescaling where no maximum rose, the masks
// inside items, and items of groups and rows in turn changed nothing. Three
// workgroups a compute unit (queries in LDS, half of the sums there at a time,
// keys asked for after the softmax) took 297, two of such ones 275.
template <typename T, uint32_t DP, bool FULL>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(DP <= 128 && sizeof(T) == 2 ? 2 : 1)))
void nz_shared_attention_kernel(nz_shared_attention_args a) {
    using S = Shape<T, DP>;
    using P = Piece<T>;
    using piece = typename P::type;
    using value_run = vec<T, S::kValueRun>;
    __shared__ float lds_m[kWaves][kColumns], lds_l[kWaves][kColumns];
    __shared__ __align__(16) float lds_o[kWaves][kColumns][DP + 4];
    __shared__ nz_shared_row rows[kColumns];   // of the item
    __shared__ uint32_t numbers[kColumns];

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
    // A request's rows are neighbours; a group's are listed.
    const uint32_t member = static_cast<uint32_t>(item.member);
    const auto row_at = [&](uint32_t i) {
        return member >= a.n_rows ? member - a.n_rows + i : static_cast<uint32_t>(a.order[member + i]);
    };
    if (threadIdx.x < static_cast<uint32_t>(item.rows)) {
        const uint32_t row = row_at(threadIdx.x);
        numbers[threadIdx.x] = row;
        rows[threadIdx.x] = a.rows[row];
    }
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
        piece q[NT][S::kKeySteps];
#pragma unroll
        for (uint32_t b = 0; b < NT; ++b) {
            const uint32_t c = b * 16 + col;
            const bool used = c < columns;
            const uint32_t row = used ? row_at(c / heads) : 0;
            const T* src = static_cast<const T*>(a.q) + row * a.q_row + (head0 + c % heads) * a.q_head;
#pragma unroll
            for (uint32_t s = 0; s < S::kKeySteps; ++s) {
                const uint32_t d = s * 4 * S::kRun + quad * S::kRun;
                q[b][s] = piece{};
                if (used && (FULL || d < a.head_dim)) q[b][s] = *reinterpret_cast<const piece*>(src + d);
            }
        }
        entries(t0, page);
        load_keys(t0, page);
        entries(t0 + kStep, next);
        f32x4 o[NT][S::kValueSteps][S::kValueRun] = {};
        float m[NT], l[NT];
#pragma unroll
        for (uint32_t b = 0; b < NT; ++b) m[b] = -__builtin_inff(), l[b] = 0.0f;

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
                        score[b][h][i] = valid[h] && t >= begin && t < end ? acc[i] * scale : -__builtin_inff();
                    }
                }
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
            // Values of keys outside the item may be anything, NaN among it.
            if (t0 < begin || t0 + S::kKeys > end || !valid[0] || !valid[S::kHalves - 1]) {
#pragma unroll
                for (uint32_t w = 0; w < S::kGroups; ++w)
#pragma unroll
                    for (uint32_t s = 0; s < S::kValueSteps; ++s)
#pragma unroll
                        for (uint32_t k = 0; k < S::kRun; ++k) {
                            const uint32_t h = S::kRun == 8 ? k / 4 : w, t = t0 + 16 * h + 4 * quad + k % 4;
                            if (!valid[h] || t < begin || t >= end) v[w][s][k] = value_run{};
                        }
            }
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
    const uint64_t slot0 = (static_cast<uint64_t>(which) * parts + part) * kColumns;
    float* const part_o = a.partials + slot0 * a.head_dim;
    float* const part_ml = a.partials + static_cast<uint64_t>(a.n_items) * parts * kColumns * a.head_dim + 2 * slot0;
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
        const nz_shared_row& r = rows[c / heads];
        if (r.group_count + r.own_count + r.tail_count == 1) {
            store_row(out + numbers[c / heads] * a.out_row + (head0 + c % heads) * a.out_head + d, sum, weight);
        } else {
            if (d == 0) *reinterpret_cast<vec<float, 2>*>(part_ml + 2 * c) = vec<float, 2>{top, weight};
            *reinterpret_cast<f32x4*>(part_o + c * a.head_dim + d) = sum;
        }
    }
}

// The rows of several items: their parts, joined in order. A workgroup takes
// one row's query heads of a key-value head; each run of 4 elements of a head
// is joined by `subs` threads, each over a share of the items, kBatch of them
// in flight at a time. A launch of its own, since the items of a row are of up
// to three kinds and an item ends parts of up to 32 rows, whose last one to
// arrive would join them all alone. Latency bound: 4.5 us for 5 rows, 10.8 for
// 128 of 64 heads; 5.8 and 19 with batches of 16, whose last ones were mostly
// repeated loads.
constexpr uint32_t kJoinThreads = 512;

template <typename T>
__global__ __launch_bounds__(kJoinThreads) void nz_shared_join_kernel(nz_shared_attention_args a) {
    struct Sums {
        f32x4 sum;
        float top, weight;
        uint32_t pad[2];
    };
    __shared__ Sums all[kJoinThreads];
    const uint32_t row = blockIdx.y, part = blockIdx.x;
    const nz_shared_row r = a.rows[row];
    const uint32_t groups = static_cast<uint32_t>(r.group_count), own = groups + static_cast<uint32_t>(r.own_count);
    const uint32_t n = own + static_cast<uint32_t>(r.tail_count);
    if (n <= 1) return;
    const uint32_t group = a.heads / a.kv_heads, blocks = (group + kColumns - 1) / kColumns, parts = a.kv_heads * blocks;
    const uint32_t kv_head = part / blocks, head0 = kv_head * group + part % blocks * kColumns;
    const uint32_t heads = min(kColumns, (kv_head + 1) * group - head0), quads = a.head_dim / 4;
    const float* const part_ml = a.partials + static_cast<uint64_t>(a.n_items) * parts * kColumns * a.head_dim;
    const uint32_t runs = heads * quads, subs = max(kJoinThreads / runs, 1u);
    T* const out = static_cast<T*>(a.out) + row * a.out_row + head0 * a.out_head;
    for (uint32_t i = threadIdx.x; i < runs * subs; i += kJoinThreads) {
        const uint32_t run = i % runs, sub = i / runs, h = run / quads, d = run % quads * 4;
        const uint32_t k0 = sub * n / subs, k1 = (sub + 1) * n / subs;
        Sums s = {{}, -__builtin_inff(), 0.0f, {}};
        constexpr uint32_t kBatch = 8;
        for (uint32_t k = k0; k < k1; k += kBatch) {
            vec<float, 2> ml[kBatch];
            f32x4 x[kBatch];
#pragma unroll
            for (uint32_t j = 0; j < kBatch; ++j) {
                const uint32_t at = min(k + j, k1 - 1);
                const uint32_t from = at < groups ? r.group_first + at * r.group_step
                                      : at < own  ? r.own_first + (at - groups)
                                                  : r.tail_first + (at - own);
                const uint32_t place = at < groups ? r.places & 0xFF : at < own ? r.places >> 8 : 0;
                const uint64_t slot = (static_cast<uint64_t>(from) * parts + part) * kColumns + place * heads + h;
                ml[j] = *reinterpret_cast<const vec<float, 2>*>(part_ml + 2 * slot);
                x[j] = *reinterpret_cast<const f32x4*>(a.partials + slot * a.head_dim + d);
            }
            float higher = s.top;
#pragma unroll
            for (uint32_t j = 0; j < kBatch; ++j) higher = fmaxf(higher, ml[j].x);
            const float base = finite_base(higher), fade = __builtin_amdgcn_exp2f(s.top - base);
            s.top = higher;
            s.weight *= fade;
            s.sum *= fade;
#pragma unroll
            for (uint32_t j = 0; j < kBatch; ++j) {
                const float share = __builtin_amdgcn_exp2f(ml[j].x - base);
                if (k + j < k1) {
                    s.weight += share * ml[j].y;
                    s.sum += share * x[j];
                }
            }
        }
        if (subs == 1) store_row(out + h * a.out_head + d, s.sum, s.weight);
        else all[i] = s;
    }
    if (subs == 1) return;
    __syncthreads();
    if (threadIdx.x < runs) {
        const uint32_t h = threadIdx.x / quads, d = threadIdx.x % quads * 4;
        float top = -__builtin_inff(), weight = 0.0f;
        for (uint32_t sub = 0; sub < subs; ++sub) top = fmaxf(top, all[sub * runs + threadIdx.x].top);
        const float base = finite_base(top);
        f32x4 sum = {};
        for (uint32_t sub = 0; sub < subs; ++sub) {
            const Sums& s = all[sub * runs + threadIdx.x];
            const float share = __builtin_amdgcn_exp2f(s.top - base);
            weight += share * s.weight;
            sum += share * s.sum;
        }
        store_row(out + h * a.out_head + d, sum, weight);
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
    const uint32_t parts = a.kv_heads * ((group + kColumns - 1) / kColumns);
    hipLaunchKernelGGL(nz_shared_join_kernel<T>, dim3(parts, a.n_rows), dim3(kJoinThreads), 0, stream, a);
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
