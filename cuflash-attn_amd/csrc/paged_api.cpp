// Validating layer and C ABI of the paged-cache operators (include/cuflash/paged_cache.h). As in
// api.cpp, every check is made before the first HIP call.

#include "cuflash/paged_cache.h"
#include "launch.hpp"
#include "paged_checks.hpp"
#include "paged_launch.hpp"

namespace cuflash {
namespace {

using E = FlashAttentionError;
using detail::check_append;
using detail::check_attention;
using detail::check_sizes;
using detail::kIntMax;
using detail::kMaxHeads;

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
