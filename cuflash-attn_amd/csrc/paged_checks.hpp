#pragma once

// The checks that the paged-cache entry points (paged_api.cpp, paged_q8_api.cpp) have in common.

#include <cmath>
#include <cstdint>

#include "paged_launch.hpp"

namespace cuflash {
namespace detail {

using Err = FlashAttentionError;

constexpr long long kIntMax = 0x7fffffffLL;
constexpr long long kMaxKeys = kIntMax - 1023;  // key positions some tiles past the end stay in 32 bits
constexpr int kMaxHeads = 65535;                // the merge's grid has the query heads in y

inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Sizes of one cache: positive, then (after head_dim and scale, which stand between) related.
inline Err check_sizes(int num_tokens, int batch_size, int num_heads, int num_kv_heads,
                       int page_size, int max_pages, int head_dim) {
    if (num_tokens <= 0 || batch_size <= 0 || num_heads <= 0 || num_kv_heads <= 0 ||
        page_size <= 0 || max_pages <= 0 || head_dim <= 0)
        return Err::INVALID_DIMENSION;
    if (head_dim != 32 && head_dim != 64 && head_dim != 128) return Err::UNSUPPORTED_HEAD_DIM;
    return Err::SUCCESS;
}
inline Err check_relations(int num_heads, int num_kv_heads, int page_size, int max_pages) {
    if (num_heads % num_kv_heads != 0) return Err::DIMENSION_MISMATCH;
    if (static_cast<long long>(page_size) * max_pages > kMaxKeys) return Err::INVALID_DIMENSION;
    return Err::SUCCESS;
}

inline Err check_append(const AppendCall& c, int elem_bytes) {
    if (!c.K || !c.V || !c.K_cache || !c.V_cache || !c.block_table || !c.seq_lens)
        return Err::NULL_POINTER;
    if (!c.Q != !c.Q_out || !c.rope_cos != !c.rope_sin) return Err::NULL_POINTER;
    const int heads = c.Q ? c.num_heads : c.num_kv_heads;  // without Q, num_heads is not used
    Err err = check_sizes(c.num_tokens, c.batch_size, heads, c.num_kv_heads, c.page_size,
                          c.max_pages, c.head_dim);
    if (err != Err::SUCCESS) return err;
    if (c.num_pages <= 0) return Err::INVALID_DIMENSION;
    if (c.rope_cos) {
        if (c.rotary_dim <= 0 || c.rotary_dim % 16 != 0 || c.max_positions <= 0)
            return Err::INVALID_DIMENSION;
        if (c.rotary_dim > c.head_dim) return Err::DIMENSION_MISMATCH;
    } else if (c.rotary_dim != 0) {
        return Err::INVALID_DIMENSION;
    }
    err = check_relations(heads, c.num_kv_heads, c.page_size, c.max_pages);
    if (err != Err::SUCCESS) return err;
    if (!c.query_starts && c.num_tokens != c.batch_size) return Err::DIMENSION_MISMATCH;
    const long long kv_row = static_cast<long long>(c.num_kv_heads) * c.head_dim;
    const long long q_row = static_cast<long long>(heads) * c.head_dim;
    if (c.k_stride < kv_row || c.v_stride < kv_row || (c.Q && c.q_stride < q_row))
        return Err::DIMENSION_MISMATCH;
    if (q_row + 2 * kv_row > kIntMax) return Err::INVALID_DIMENSION;
    const long long bytes = elem_bytes;
    if (c.k_stride * bytes % 16 || c.v_stride * bytes % 16 || (c.Q && c.q_stride * bytes % 16))
        return Err::INVALID_DIMENSION;
    for (const void* p : {c.Q, c.K, c.V, static_cast<const void*>(c.Q_out),
                          static_cast<const void*>(c.K_cache),
                          static_cast<const void*>(c.V_cache),
                          static_cast<const void*>(c.rope_cos),
                          static_cast<const void*>(c.rope_sin)})
        if (!aligned16(p)) return Err::INVALID_DIMENSION;
    // In place, a token's rotated queries must not reach another token's.
    if (c.Q && c.Q_out == c.Q && c.num_tokens > 1 && c.q_stride != q_row)
        return Err::DIMENSION_MISMATCH;
    return Err::SUCCESS;
}

// Both attentions: `shared` with prefix_table and prefix_len, the forward with query_starts.
inline Err check_attention(const PagedCall& c, bool shared) {
    if (!c.Q || !c.K_cache || !c.V_cache || !c.O || !c.L || !c.block_table || !c.seq_lens)
        return Err::NULL_POINTER;
    if (shared ? c.prefix_len > 0 && !c.prefix_table : !c.query_starts) return Err::NULL_POINTER;
    if (c.prefix_len < 0) return Err::INVALID_DIMENSION;
    Err err = check_sizes(c.num_tokens, c.batch_size, c.num_heads, c.num_kv_heads, c.page_size,
                          c.max_pages, c.head_dim);
    if (err != Err::SUCCESS) return err;
    if (!std::isfinite(c.scale) || c.scale < 0.0f) return Err::INVALID_DIMENSION;
    err = check_relations(c.num_heads, c.num_kv_heads, c.page_size, c.max_pages);
    if (err != Err::SUCCESS) return err;
    if (c.prefix_len > c.page_size * c.max_pages) return Err::DIMENSION_MISMATCH;
    if (static_cast<long long>(c.num_tokens) * c.num_heads > kIntMax || c.num_heads > kMaxHeads)
        return Err::INVALID_DIMENSION;
    for (const void* p : {c.Q, c.K_cache, c.V_cache, static_cast<const void*>(c.O)})
        if (!aligned16(p)) return Err::INVALID_DIMENSION;
    if (reinterpret_cast<uintptr_t>(c.workspace) % 256) return Err::INVALID_DIMENSION;
    return Err::SUCCESS;
}

}  // namespace detail
}  // namespace cuflash
