// capi_serving.cpp -- argument checks of the serving-step operators
// (nz_pages_*, nz_rotary_store, nz_attention_*, nz_shared_*, nz_adjust_logits,
// nz_verify_drafts, nz_route_experts, nz_expert_mlp); the kernels' launchers
// are in hip/{serving,attention,shared_attention,verify,experts}_gfx950.hip.
#include <algorithm>
#include <cstdint>

#include "capi_internal.hpp"
#include "neuralzip_hip.h"

using nz_capi::guarded;
using nz_capi::set_error;

extern "C" int nz_hip_pages_extend(const nz_pages_extend_args* args, void* stream, char* message, size_t message_size);
extern "C" int nz_hip_pages_release(const nz_pages_release_args* args, void* stream, char* message,
                                    size_t message_size);
extern "C" int nz_hip_pages_trim(const nz_pages_trim_args* args, void* stream, char* message, size_t message_size);
extern "C" int nz_hip_rotary_store(const nz_rotary_args* args, void* stream, char* message, size_t message_size);
extern "C" int nz_hip_attention_plan(const int32_t* contexts, const int32_t* requests, uint32_t n_rows, uint32_t target,
                                     uint32_t parts, nz_attention_item* items, uint32_t* counters, void* stream,
                                     char* message, size_t message_size);
extern "C" int nz_hip_attention(const nz_attention_args* args, void* stream, char* message, size_t message_size);
extern "C" int nz_hip_adjust_logits(const nz_logits_args* args, void* stream, char* message, size_t message_size);
extern "C" int nz_hip_shared_plan(const nz_shared_plan_args* args, void* stream, char* message, size_t message_size);
extern "C" int nz_hip_shared_attention(const nz_shared_attention_args* args, void* stream, char* message,
                                       size_t message_size);
extern "C" int nz_hip_verify_drafts(const nz_verify_args* args, void* stream, char* message, size_t message_size);
extern "C" uint64_t nz_hip_verify_scratch(uint32_t n_rows, uint32_t n_requests, uint32_t vocab);
extern "C" int nz_hip_route_experts(const nz_route_args* args, void* stream, char* message, size_t message_size);
extern "C" int nz_hip_expert_mlp(const nz_expert_args* args, void* stream, char* message, size_t message_size);
extern "C" uint64_t nz_hip_expert_scratch(uint32_t tokens, uint32_t hidden, uint32_t inter, uint32_t top_k);

namespace {

constexpr uint64_t kMaxGrid = 0x7FFFFFFFull;   // workgroups of one launch dimension

[[noreturn]] void refuse(const char* message) { nz::fail(nz::kInvalidArgument, message); }

void check_pages(uint32_t n_requests, uint32_t max_pages, uint32_t page_size, uint32_t n_pages) {
    if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)))
        refuse("page_size must be a power of two from 16 to 1024.");
    if (n_requests > kMaxGrid || n_pages > kMaxGrid || max_pages == 0 ||
        static_cast<uint64_t>(max_pages) * page_size > kMaxGrid)
        refuse("Requests, pages and a request's tokens must be below 2^31 (and max_pages at least 1).");
}

uint32_t type_size(uint32_t type) {
    if (type != NZ_BF16 && type != NZ_FP16 && type != NZ_FP32) refuse("Unknown value type.");
    return type == NZ_FP32 ? 4 : 2;
}

void check_head_dim(uint32_t head_dim) {
    if (head_dim == 0 || head_dim > 256 || head_dim % 16) refuse("head_dim must be a multiple of 16 up to 256.");
}

// Columns of an item, over all key-value heads.
uint64_t shared_width(uint32_t heads, uint32_t kv_heads) {
    const uint32_t group = heads / kv_heads;
    return static_cast<uint64_t>(kv_heads) * ((group + NZ_SHARED_COLUMNS - 1ull) / NZ_SHARED_COLUMNS) * NZ_SHARED_COLUMNS;
}

void check_hidden(uint32_t hidden, const char* message) {
    if (hidden == 0 || hidden % 8) refuse(message);
}

// 16-byte accesses: the address and every element stride.
template <typename... Strides>
void check_alignment(uint32_t size, const void* p, Strides... strides) {
    bool ok = reinterpret_cast<uintptr_t>(p) % 16 == 0;
    for (int64_t s : {static_cast<int64_t>(strides)...}) ok = ok && (s * static_cast<int64_t>(size)) % 16 == 0;
    if (!ok) refuse("Addresses and strides must be multiples of 16 bytes.");
}

template <typename Args, typename Check>
int run(const Args* args, void* stream, int (*launch)(const Args*, void*, char*, size_t), Check&& check) {
    bool empty = false;
    const int bad = guarded([&] {
        if (!args) refuse("Null operator arguments.");
        empty = check(*args);
    });
    if (bad || empty) return bad;
    char message[256] = {0};
    const int rc = launch(args, stream, message, sizeof message);
    return rc ? set_error(rc, message) : 0;
}

}  // namespace

extern "C" {

int nz_pages_extend(const nz_pages_extend_args* args, void* stream) {
    return run(args, stream, nz_hip_pages_extend, [](const nz_pages_extend_args& a) {
        if (!a.lengths || !a.new_tokens || !a.tables || !a.free_pages || !a.n_free || !a.starts || !a.status ||
            !a.lengths_after || !a.n_free_after ||
            (a.max_tokens && (!a.slots || !a.positions || !a.requests || !a.contexts)))
            refuse("Null pages argument.");
        check_pages(a.n_requests, a.max_pages, a.page_size, a.n_pages);
        if (a.max_tokens > kMaxGrid) refuse("A step's tokens must be below 2^31.");
        if (a.advance > 1) refuse("advance is 0 or 1.");
        return false;
    });
}

int nz_pages_release(const nz_pages_release_args* args, void* stream) {
    return run(args, stream, nz_hip_pages_release, [](const nz_pages_release_args& a) {
        if (!a.lengths || !a.done || !a.tables || !a.free_pages || !a.n_free || !a.lengths_after || !a.n_free_after)
            refuse("Null pages argument.");
        check_pages(a.n_requests, a.max_pages, a.page_size, a.n_pages);
        if (a.advance > 1 || a.reserved) refuse("advance is 0 or 1 and reserved is 0.");
        return false;
    });
}

int nz_pages_trim(const nz_pages_trim_args* args, void* stream) {
    return run(args, stream, nz_hip_pages_trim, [](const nz_pages_trim_args& a) {
        if (!a.lengths || !a.keep || !a.tables || !a.free_pages || !a.n_free || !a.lengths_after || !a.n_free_after)
            refuse("Null pages argument.");
        check_pages(a.n_requests, a.max_pages, a.page_size, a.n_pages);
        if (a.advance > 1 || a.reserved) refuse("advance is 0 or 1 and reserved is 0.");
        return false;
    });
}

int nz_rotary_store(const nz_rotary_args* args, void* stream) {
    return run(args, stream, nz_hip_rotary_store, [](const nz_rotary_args& a) {
        const uint32_t size = type_size(a.type);
        check_head_dim(a.head_dim);
        if (a.rotary_dim % 16 || a.rotary_dim > a.head_dim)
            refuse("rotary_dim must be a multiple of 16 up to head_dim.");
        if (a.heads == 0 || a.kv_heads == 0) refuse("There must be query and key heads.");
        if (a.tokens == 0) return true;
        if (!a.q || !a.k || !a.v || !a.out || (!a.key_cache != !a.value_cache) || (a.key_cache && !a.slots) ||
            (a.rotary_dim && (!a.cos || !a.sin || !a.positions)))
            refuse("Null rotary argument.");
        if (a.weight_type != a.type && a.weight_type != NZ_FP32)
            refuse("Norm weights must be of the values' type or 32-bit.");
        check_alignment(size, a.q, a.q_token, a.q_head);
        check_alignment(size, a.k, a.k_token, a.k_head);
        check_alignment(size, a.v, a.v_token, a.v_head);
        check_alignment(size, a.out, a.out_token, a.out_head);
        check_alignment(4, a.cos, 0);
        check_alignment(4, a.sin, 0);
        check_alignment(4, a.q_weight, 0);
        check_alignment(4, a.k_weight, 0);
        if (a.key_cache) {
            check_pages(0, 1, a.page_size, a.n_pages);
            check_alignment(size, a.key_cache, a.key_page, a.key_head, a.key_slot);
            check_alignment(size, a.value_cache, a.value_page, a.value_head, a.value_slot);
        }
        if (static_cast<uint64_t>(a.tokens) * (static_cast<uint64_t>(a.heads) + 2ull * a.kv_heads) > kMaxGrid)
            refuse("Too many heads in one call.");
        return false;
    });
}

int nz_attention_plan(const int32_t* contexts, const int32_t* requests, uint32_t n_rows, uint32_t target,
                      uint32_t parts, nz_attention_item* items, uint32_t* counters, void* stream) {
    const int bad = guarded([&] {
        if (!items || !counters || (!contexts && n_rows)) refuse("Null attention plan argument.");
        if (target == 0 || target > kMaxGrid / 4 || n_rows > kMaxGrid / 4 || parts == 0)
            refuse("The plan's target and parts must be positive, and rows and target below 2^29.");
    });
    if (bad) return bad;
    char message[256] = {0};
    const int rc = nz_hip_attention_plan(contexts, requests, n_rows, target, parts, items, counters, stream, message,
                                         sizeof message);
    return rc ? set_error(rc, message) : 0;
}

uint64_t nz_attention_partials(uint32_t n_items, uint32_t heads, uint32_t head_dim) {
    return static_cast<uint64_t>(n_items) * heads * (head_dim + 2ull);
}

int nz_attention(const nz_attention_args* args, void* stream) {
    return run(args, stream, nz_hip_attention, [](const nz_attention_args& a) {
        const uint32_t size = type_size(a.type);
        check_head_dim(a.head_dim);
        if (a.kv_heads == 0 || a.heads == 0 || a.heads % a.kv_heads)
            refuse("heads must be a positive multiple of kv_heads.");
        if (a.reserved) refuse("reserved is 0.");
        if (a.n_rows == 0) return true;
        if (!a.q || !a.key_cache || !a.value_cache || !a.out || !a.tables || !a.items || !a.counters || !a.partials)
            refuse("Null attention argument.");
        check_pages(a.n_requests, a.max_pages, a.page_size, a.n_pages);
        if (a.n_pages == 0 || a.n_requests == 0) refuse("There must be pages and requests.");
        check_alignment(size, a.q, a.q_row, a.q_head);
        check_alignment(size, a.out, a.out_row, a.out_head);
        check_alignment(size, a.key_cache, a.key_page, a.key_head, a.key_slot);
        check_alignment(size, a.value_cache, a.value_page, a.value_head, a.value_slot);
        check_alignment(4, a.partials, 0);
        if (a.n_items < a.n_rows) refuse("The plan has fewer items than rows.");
        if (a.n_items > kMaxGrid || a.heads > kMaxGrid ||
            static_cast<uint64_t>(a.n_items) * a.heads > (1ull << 30) / a.head_dim)
            refuse("Too many items and heads in one call.");
        return false;
    });
}

uint32_t nz_shared_items(uint32_t n_rows, uint32_t n_groups, uint32_t heads, uint32_t kv_heads, uint32_t target) {
    if (n_rows > NZ_SHARED_MAX_ROWS || n_groups > NZ_SHARED_MAX_GROUPS || kv_heads == 0 || heads == 0 ||
        heads % kv_heads || target == 0 || target > 65536)
        return 0;
    const uint32_t tile_rows = std::max(1u, NZ_SHARED_COLUMNS / (heads / kv_heads));
    // a tile per row, and those of the groups
    const uint32_t tiles = n_rows + (n_groups ? std::min(n_rows, n_groups + n_rows / tile_rows) : 0);
    const uint32_t items = (std::max(tiles, target) + target - 1) / target * target;
    return n_groups ? items + items / 2 : items;
}

int nz_shared_plan(const nz_shared_plan_args* args, void* stream) {
    return run(args, stream, nz_hip_shared_plan, [](const nz_shared_plan_args& a) {
        if (a.reserved) refuse("reserved is 0.");
        const uint32_t items = nz_shared_items(a.n_rows, a.n_groups, a.heads, a.kv_heads, a.target);
        if (items == 0)
            refuse("heads must be a positive multiple of kv_heads, the target from 1 to 65536, and rows and groups at most "
                   "NZ_SHARED_MAX_ROWS and NZ_SHARED_MAX_GROUPS.");
        if (a.n_items < items) refuse("The plan has room for fewer items than nz_shared_items.");
        if (a.n_items > kMaxGrid || a.n_requests > kMaxGrid) refuse("Items and requests must be below 2^31.");
        if (!a.items || (a.n_rows && (!a.contexts || !a.rows || !a.order)) ||
            (a.n_groups && (!a.groups || !a.shared)))
            refuse("Null shared plan argument.");
        return false;
    });
}

uint64_t nz_shared_partials(uint32_t n_items, uint32_t heads, uint32_t kv_heads, uint32_t head_dim) {
    return kv_heads == 0 ? 0 : n_items * shared_width(heads, kv_heads) * (head_dim + 2ull);
}

int nz_shared_attention(const nz_shared_attention_args* args, void* stream) {
    return run(args, stream, nz_hip_shared_attention, [](const nz_shared_attention_args& a) {
        const uint32_t size = type_size(a.type);
        check_head_dim(a.head_dim);
        if (a.kv_heads == 0 || a.heads == 0 || a.heads % a.kv_heads)
            refuse("heads must be a positive multiple of kv_heads.");
        if (a.reserved) refuse("reserved is 0.");
        if (a.n_rows == 0) return true;
        if (!a.q || !a.key_cache || !a.value_cache || !a.out || !a.tables || !a.items || !a.rows || !a.order ||
            !a.partials)
            refuse("Null attention argument.");
        check_pages(a.n_requests, a.max_pages, a.page_size, a.n_pages);
        if (a.n_pages == 0 || a.n_requests == 0) refuse("There must be pages and requests.");
        check_alignment(size, a.q, a.q_row, a.q_head);
        check_alignment(size, a.out, a.out_row, a.out_head);
        check_alignment(size, a.key_cache, a.key_page, a.key_head, a.key_slot);
        check_alignment(size, a.value_cache, a.value_page, a.value_head, a.value_slot);
        check_alignment(4, a.partials, 0);
        if (a.n_rows > NZ_SHARED_MAX_ROWS) refuse("Too many rows in one call.");
        if (a.n_items < a.n_rows) refuse("The plan has fewer items than rows.");
        if (a.heads > kMaxGrid || a.n_items > kMaxGrid ||
            a.n_items * shared_width(a.heads, a.kv_heads) > kMaxGrid)
            refuse("Too many items and heads in one call.");
        return false;
    });
}

int nz_adjust_logits(const nz_logits_args* args, void* stream) {
    return run(args, stream, nz_hip_adjust_logits, [](const nz_logits_args& a) {
        type_size(a.type);
        if (a.reserved) refuse("reserved is 0.");
        if (a.rows == 0 || a.vocab == 0) return true;
        if (!a.logits || !a.out || (a.history && !a.lengths) ||
            (a.bias_starts && a.n_bias && (!a.bias_tokens || !a.bias_values)))
            refuse("Null logits argument.");
        if (a.history && a.history_bytes != 4 && a.history_bytes != 8) refuse("Token ids are of 4 or 8 bytes.");
        if (a.vocab > kMaxGrid || a.rows > 65535) refuse("Too many rows or tokens in one call.");
        return false;
    });
}

uint64_t nz_verify_scratch(uint32_t n_rows, uint32_t n_requests, uint32_t vocab) {
    return nz_hip_verify_scratch(n_rows, n_requests, vocab);
}

int nz_verify_drafts(const nz_verify_args* args, void* stream) {
    return run(args, stream, nz_hip_verify_drafts, [](const nz_verify_args& a) {
        type_size(a.type);
        if (a.n_rows > 65535 || a.n_requests > 65535 || a.vocab == 0 || a.vocab > NZ_VERIFY_MAX_VOCAB)
            refuse("There must be at most 65535 rows and requests, and 1 to 2^22 tokens.");
        if (a.n_requests == 0) return true;
        if (!a.starts || !a.sample || !a.accepted || !a.next ||
            (a.n_rows && (!a.logits || !a.tokens || !a.accept || !a.scratch)))
            refuse("Null verification argument.");
        if (reinterpret_cast<uintptr_t>(a.scratch) % 16) refuse("The scratch must be on a 16-byte boundary.");
        return false;
    });
}

int nz_route_experts(const nz_route_args* args, void* stream) {
    return run(args, stream, nz_hip_route_experts, [](const nz_route_args& a) {
        type_size(a.type);
        if (a.weight_type != a.type && a.weight_type != NZ_FP32)
            refuse("The router's weight must be of x's type or 32-bit.");
        if (a.scoring > NZ_ROUTE_SIGMOID || a.normalize > 1 || a.reserved)
            refuse("scoring is an nz_route_scoring, normalize 0 or 1 and reserved 0.");
        check_hidden(a.hidden, "hidden must be a positive multiple of 8.");
        if (a.hidden > 1u << 24 || a.experts > NZ_EXPERT_MAX || a.tokens > 65535)
            refuse("Too many experts or tokens, or too long rows.");
        if (a.top_k == 0 || a.top_k > NZ_ROUTE_MAX_TOP || a.top_k > a.experts)
            refuse("top_k must be from 1 to NZ_ROUTE_MAX_TOP and the experts.");
        if (a.tokens == 0) return true;
        if (!a.x || !a.weight || !a.ids || !a.weights || !a.scratch) refuse("Null router argument.");
        check_alignment(4, a.weight, 0);
        if (reinterpret_cast<uintptr_t>(a.scratch) % 8) refuse("The scratch must be on an 8-byte boundary.");
        return false;
    });
}

uint64_t nz_expert_scratch(uint32_t tokens, uint32_t hidden, uint32_t inter, uint32_t top_k) {
    return nz_hip_expert_scratch(tokens, hidden, inter, top_k);
}

int nz_expert_mlp(const nz_expert_args* args, void* stream) {
    return run(args, stream, nz_hip_expert_mlp, [](const nz_expert_args& a) {
        const uint32_t size = type_size(a.type);
        check_hidden(a.hidden, "hidden must be a positive multiple of 8.");
        check_hidden(a.inter, "inter must be a positive multiple of 8.");
        if (a.experts == 0 || a.experts > NZ_EXPERT_MAX || a.top_k == 0 || a.top_k > NZ_ROUTE_MAX_TOP)
            refuse("There must be 1 to NZ_EXPERT_MAX experts and 1 to NZ_ROUTE_MAX_TOP choices.");
        if (a.id_bytes != 4 && a.id_bytes != 8) refuse("Experts' numbers are of 4 or 8 bytes.");
        if (a.activation > NZ_EXPERT_GELU) refuse("Unknown activation.");
        if (a.tokens == 0) return true;
        if (!a.x || !a.ids || !a.weights || !a.gate_up || !a.down || !a.out || !a.scratch)
            refuse("Null experts argument.");
        if (a.tokens > 65535u * NZ_EXPERT_TOKENS || a.hidden > 1u << 24 || a.inter > 1u << 24 ||
            static_cast<uint64_t>(a.tokens) * a.hidden > 1ull << 27)
            refuse("Too many tokens in one call.");
        check_alignment(size, a.x, a.x_row);
        check_alignment(size, a.out, a.out_row);
        check_alignment(size, a.gate_up, a.gate_expert, a.gate_row);
        check_alignment(size, a.down, a.down_expert, a.down_row);
        check_alignment(4, a.scratch, 0);
        return false;
    });
}

}  // extern "C"
