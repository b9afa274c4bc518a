// capi_serving.cpp -- argument checks of the serving-step operators
// (nz_pages_*, nz_rotary_store, nz_attention_*, nz_adjust_logits); the
// kernels' launchers are in hip/serving_gfx950.hip and
// hip/attention_gfx950.hip.
#include <cstdint>

#include "capi_internal.hpp"
#include "neuralzip_hip.h"

using nz_capi::guarded;
using nz_capi::set_error;

extern "C" int nz_hip_pages_extend(const nz_pages_extend_args* args, void* stream, char* message, size_t message_size);
extern "C" int nz_hip_pages_release(const nz_pages_release_args* args, void* stream, char* message,
                                    size_t message_size);
extern "C" int nz_hip_rotary_store(const nz_rotary_args* args, void* stream, char* message, size_t message_size);
extern "C" int nz_hip_attention_plan(const int32_t* contexts, const int32_t* requests, uint32_t n_rows, uint32_t target,
                                     uint32_t parts, nz_attention_item* items, uint32_t* counters, void* stream,
                                     char* message, size_t message_size);
extern "C" int nz_hip_attention(const nz_attention_args* args, void* stream, char* message, size_t message_size);
extern "C" int nz_hip_adjust_logits(const nz_logits_args* args, void* stream, char* message, size_t message_size);

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

}  // extern "C"
