// Validating layer and C ABI of the paged-cache operators (include/cuflash/paged_cache.h). As in
// api.cpp, every check is made before the first HIP call.

#include <cmath>
#include <cstdint>

#include "cuflash/paged_cache.h"
#include "launch.hpp"
#include "paged_launch.hpp"

namespace cuflash {
namespace {

using E = FlashAttentionError;

constexpr long long kIntMax = 0x7fffffffLL;
constexpr long long kMaxKeys = kIntMax - 1023;  // key positions some tiles past the end stay in 32 bits
constexpr int kMaxHeads = 65535;                // the merge's grid has the query heads in y

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Sizes of one cache: positive, then (after head_dim and scale, which stand between) related.
E check_sizes(int num_tokens, int batch_size, int num_heads, int num_kv_heads, int page_size,
              int max_pages, int head_dim) {
    if (num_tokens <= 0 || batch_size <= 0 || num_heads <= 0 || num_kv_heads <= 0 ||
        page_size <= 0 || max_pages <= 0 || head_dim <= 0)
        return E::INVALID_DIMENSION;
    if (head_dim != 32 && head_dim != 64 && head_dim != 128) return E::UNSUPPORTED_HEAD_DIM;
    return E::SUCCESS;
}
E check_relations(int num_heads, int num_kv_heads, int page_size, int max_pages) {
    if (num_heads % num_kv_heads != 0) return E::DIMENSION_MISMATCH;
    if (static_cast<long long>(page_size) * max_pages > kMaxKeys) return E::INVALID_DIMENSION;
    return E::SUCCESS;
}

E check_append(const detail::AppendCall& c, int elem_bytes) {
    if (!c.K || !c.V || !c.K_cache || !c.V_cache || !c.block_table || !c.seq_lens)
        return E::NULL_POINTER;
    if (!c.Q != !c.Q_out || !c.rope_cos != !c.rope_sin) return E::NULL_POINTER;
    const int heads = c.Q ? c.num_heads : c.num_kv_heads;  // without Q, num_heads is not used
    E err = check_sizes(c.num_tokens, c.batch_size, heads, c.num_kv_heads, c.page_size,
                        c.max_pages, c.head_dim);
    if (err != E::SUCCESS) return err;
    if (c.num_pages <= 0) return E::INVALID_DIMENSION;
    if (c.rope_cos) {
        if (c.rotary_dim <= 0 || c.rotary_dim % 16 != 0 || c.max_positions <= 0)
            return E::INVALID_DIMENSION;
        if (c.rotary_dim > c.head_dim) return E::DIMENSION_MISMATCH;
    } else if (c.rotary_dim != 0) {
        return E::INVALID_DIMENSION;
    }
    err = check_relations(heads, c.num_kv_heads, c.page_size, c.max_pages);
    if (err != E::SUCCESS) return err;
    if (!c.query_starts && c.num_tokens != c.batch_size) return E::DIMENSION_MISMATCH;
    const long long kv_row = static_cast<long long>(c.num_kv_heads) * c.head_dim;
    const long long q_row = static_cast<long long>(heads) * c.head_dim;
    if (c.k_stride < kv_row || c.v_stride < kv_row || (c.Q && c.q_stride < q_row))
        return E::DIMENSION_MISMATCH;
    if (q_row + 2 * kv_row > kIntMax) return E::INVALID_DIMENSION;
    const long long bytes = elem_bytes;
    if (c.k_stride * bytes % 16 || c.v_stride * bytes % 16 || (c.Q && c.q_stride * bytes % 16))
        return E::INVALID_DIMENSION;
    for (const void* p : {c.Q, c.K, c.V, static_cast<const void*>(c.Q_out),
                          static_cast<const void*>(c.K_cache),
                          static_cast<const void*>(c.V_cache),
                          static_cast<const void*>(c.rope_cos),
                          static_cast<const void*>(c.rope_sin)})
        if (!aligned16(p)) return E::INVALID_DIMENSION;
    // In place, a token's rotated queries must not reach another token's.
    if (c.Q && c.Q_out == c.Q && c.num_tokens > 1 && c.q_stride != q_row)
        return E::DIMENSION_MISMATCH;
    return E::SUCCESS;
}

// Both attentions: `shared` with prefix_table and prefix_len, the forward with query_starts.
E check_attention(const detail::PagedCall& c, bool shared) {
    if (!c.Q || !c.K_cache || !c.V_cache || !c.O || !c.L || !c.block_table || !c.seq_lens)
        return E::NULL_POINTER;
    if (shared ? c.prefix_len > 0 && !c.prefix_table : !c.query_starts) return E::NULL_POINTER;
    if (c.prefix_len < 0) return E::INVALID_DIMENSION;
    E err = check_sizes(c.num_tokens, c.batch_size, c.num_heads, c.num_kv_heads, c.page_size,
                        c.max_pages, c.head_dim);
    if (err != E::SUCCESS) return err;
    if (!std::isfinite(c.scale) || c.scale < 0.0f) return E::INVALID_DIMENSION;
    err = check_relations(c.num_heads, c.num_kv_heads, c.page_size, c.max_pages);
    if (err != E::SUCCESS) return err;
    if (c.prefix_len > c.page_size * c.max_pages) return E::DIMENSION_MISMATCH;
    if (static_cast<long long>(c.num_tokens) * c.num_heads > kIntMax || c.num_heads > kMaxHeads)
        return E::INVALID_DIMENSION;
    for (const void* p : {c.Q, c.K_cache, c.V_cache, static_cast<const void*>(c.O)})
        if (!aligned16(p)) return E::INVALID_DIMENSION;
    if (reinterpret_cast<uintptr_t>(c.workspace) % 256) return E::INVALID_DIMENSION;
    return E::SUCCESS;
}

// For the sizes alone; page_size and max_pages do not matter to it.
template <typename T>
long long workspace_impl(int num_tokens, int batch_size, int num_heads, int num_kv_heads,
                         int head_dim, bool shared) {
    if (check_sizes(num_tokens, batch_size, num_heads, num_kv_heads, 1, 1, head_dim) !=
            E::SUCCESS ||
        num_heads % num_kv_heads != 0 || static_cast<long long>(num_tokens) * num_heads > kIntMax ||
        num_heads > kMaxHeads)
        return -1;
    detail::PagedCall c{};
    c.num_tokens = num_tokens;
    c.batch_size = batch_size;
    c.num_heads = num_heads;
    c.num_kv_heads = num_kv_heads;
    c.head_dim = head_dim;
    c.prefix_len = shared ? 1 << 30 : 0;  // no prefix is cut into more chunks than a long one
    return detail::paged_workspace<T>(c);
}

template <typename T>
E forward_impl(const detail::PagedCall& c, hipStream_t stream) {
    E err = check_attention(c, false);
    if (err != E::SUCCESS) return err;
    return detail::launch_paged<T>(c, stream);
}

template <typename T>
E shared_impl(const detail::PagedCall& c, hipStream_t stream) {
    E err = check_attention(c, true);
    if (err != E::SUCCESS) return err;
    // A captured call needs memory that is the caller's, which that entry point has no argument for.
    if (c.prefix_len == 0 && !detail::stream_capturing(stream))
        return detail::launch_decode_paged<T>(
            static_cast<const T*>(c.Q), static_cast<const T*>(c.K_cache),
            static_cast<const T*>(c.V_cache), static_cast<T*>(c.O), c.L, c.block_table, c.seq_lens,
            c.batch_size, c.num_heads, c.num_kv_heads, c.page_size, c.max_pages, c.head_dim,
            c.scale, 0, stream);
    return detail::launch_paged<T>(c, stream);
}

template <typename T>
E append_impl(const detail::AppendCall& c, hipStream_t stream) {
    E err = check_append(c, sizeof(T));
    if (err != E::SUCCESS) return err;
    return detail::launch_append_paged<T>(c, stream);
}

}  // namespace

#define CUFLASH_PAGED_CACHE(SFX, T)                                                              \
    E flash_attention_append_paged(                                                              \
        const T* Q, const T* K, const T* V, T* Q_out, T* K_cache, T* V_cache,                    \
        const int* block_table, const int* seq_lens, const int* query_starts,                    \
        const float* rope_cos, const float* rope_sin, int num_tokens, int batch_size,            \
        int num_heads, int num_kv_heads, int q_stride, int k_stride, int v_stride,               \
        int num_pages, int page_size, int max_pages_per_seq, int head_dim, int rotary_dim,       \
        int max_positions, bool interleaved, hipStream_t stream) {                               \
        return append_impl<T>(                                                                   \
            detail::AppendCall{Q, K, V, Q_out, K_cache, V_cache, block_table, seq_lens,          \
                               query_starts, rope_cos, rope_sin, num_tokens, batch_size,         \
                               num_heads, num_kv_heads, q_stride, k_stride, v_stride, num_pages, \
                               page_size, max_pages_per_seq, head_dim, rotary_dim,               \
                               max_positions, interleaved},                                      \
            stream);                                                                             \
    }                                                                                            \
    extern "C" int cuflash_attention_append_paged_##SFX(                                         \
        const T* Q, const T* K, const T* V, T* Q_out, T* K_cache, T* V_cache,                    \
        const int* block_table, const int* seq_lens, const int* query_starts,                    \
        const float* rope_cos, const float* rope_sin, int num_tokens, int batch_size,            \
        int num_heads, int num_kv_heads, int q_stride, int k_stride, int v_stride,               \
        int num_pages, int page_size, int max_pages_per_seq, int head_dim, int rotary_dim,       \
        int max_positions, bool interleaved, hipStream_t stream) {                               \
        return static_cast<int>(flash_attention_append_paged(                                    \
            Q, K, V, Q_out, K_cache, V_cache, block_table, seq_lens, query_starts, rope_cos,     \
            rope_sin, num_tokens, batch_size, num_heads, num_kv_heads, q_stride, k_stride,       \
            v_stride, num_pages, page_size, max_pages_per_seq, head_dim, rotary_dim,             \
            max_positions, interleaved, stream));                                                \
    }                                                                                            \
    E flash_attention_forward_paged(                                                             \
        const T* Q, const T* K_cache, const T* V_cache, T* O, float* L, const int* block_table,  \
        const int* seq_lens, const int* query_starts, int num_tokens, int batch_size,            \
        int num_heads, int num_kv_heads, int page_size, int max_pages_per_seq, int head_dim,     \
        float scale, bool causal, void* workspace, size_t workspace_bytes, hipStream_t stream) { \
        return forward_impl<T>(                                                                  \
            detail::PagedCall{Q, K_cache, V_cache, O, L, block_table, nullptr, seq_lens,         \
                              query_starts, num_tokens, batch_size, num_heads, num_kv_heads, 0,  \
                              page_size, max_pages_per_seq, head_dim, scale, causal, workspace,  \
                              workspace_bytes},                                                  \
            stream);                                                                             \
    }                                                                                            \
    extern "C" int cuflash_attention_forward_paged_##SFX(                                        \
        const T* Q, const T* K_cache, const T* V_cache, T* O, float* L, const int* block_table,  \
        const int* seq_lens, const int* query_starts, int num_tokens, int batch_size,            \
        int num_heads, int num_kv_heads, int page_size, int max_pages_per_seq, int head_dim,     \
        float scale, bool causal, void* workspace, size_t workspace_bytes, hipStream_t stream) { \
        return static_cast<int>(flash_attention_forward_paged(                                   \
            Q, K_cache, V_cache, O, L, block_table, seq_lens, query_starts, num_tokens,          \
            batch_size, num_heads, num_kv_heads, page_size, max_pages_per_seq, head_dim, scale,  \
            causal, workspace, workspace_bytes, stream));                                        \
    }                                                                                            \
    extern "C" long long cuflash_attention_forward_paged_workspace_##SFX(                        \
        int num_tokens, int batch_size, int num_heads, int num_kv_heads, int head_dim) {         \
        return workspace_impl<T>(num_tokens, batch_size, num_heads, num_kv_heads, head_dim,      \
                                 false);                                                         \
    }                                                                                            \
    E flash_attention_decode_shared(                                                             \
        const T* Q, const T* K_cache, const T* V_cache, T* O, float* L, const int* prefix_table, \
        const int* block_table, const int* seq_lens, int batch_size, int num_heads,              \
        int num_kv_heads, int prefix_len, int page_size, int max_pages_per_seq, int head_dim,    \
        float scale, void* workspace, size_t workspace_bytes, hipStream_t stream) {              \
        return shared_impl<T>(                                                                   \
            detail::PagedCall{Q, K_cache, V_cache, O, L, block_table, prefix_table, seq_lens,    \
                              nullptr, batch_size, batch_size, num_heads, num_kv_heads,          \
                              prefix_len, page_size, max_pages_per_seq, head_dim, scale, false,  \
                              workspace, workspace_bytes},                                       \
            stream);                                                                             \
    }                                                                                            \
    extern "C" int cuflash_attention_decode_shared_##SFX(                                        \
        const T* Q, const T* K_cache, const T* V_cache, T* O, float* L, const int* prefix_table, \
        const int* block_table, const int* seq_lens, int batch_size, int num_heads,              \
        int num_kv_heads, int prefix_len, int page_size, int max_pages_per_seq, int head_dim,    \
        float scale, void* workspace, size_t workspace_bytes, hipStream_t stream) {              \
        return static_cast<int>(flash_attention_decode_shared(                                   \
            Q, K_cache, V_cache, O, L, prefix_table, block_table, seq_lens, batch_size,          \
            num_heads, num_kv_heads, prefix_len, page_size, max_pages_per_seq, head_dim, scale,  \
            workspace, workspace_bytes, stream));                                                \
    }                                                                                            \
    extern "C" long long cuflash_attention_decode_shared_workspace_##SFX(                        \
        int batch_size, int num_heads, int num_kv_heads, int head_dim) {                         \
        return workspace_impl<T>(batch_size, batch_size, num_heads, num_kv_heads, head_dim,      \
                                 true);                                                          \
    }
CUFLASH_PAGED_CACHE(f32, float)
CUFLASH_PAGED_CACHE(f16, __half)
CUFLASH_PAGED_CACHE(bf16, __hip_bfloat16)
#undef CUFLASH_PAGED_CACHE

}  // namespace cuflash
