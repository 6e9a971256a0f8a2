#pragma once

// Internal launcher interface between the validating paged-cache API (paged_api.cpp) and its
// kernels (append.hip, paged.hip). Arguments have been validated when a launcher runs.

#include "cuflash/paged_cache.h"

namespace cuflash {
namespace detail {

// The arguments of flash_attention_append_paged, tensors untyped.
struct AppendCall {
    const void *Q, *K, *V;
    void *Q_out, *K_cache, *V_cache;
    const int *block_table, *seq_lens, *query_starts;
    const float *rope_cos, *rope_sin;
    int num_tokens, batch_size, num_heads, num_kv_heads;
    int q_stride, k_stride, v_stride;
    int num_pages, page_size, max_pages;
    int head_dim, rotary_dim, max_positions;
    bool interleaved;
};
template <typename T>
FlashAttentionError launch_append_paged(const AppendCall& call, hipStream_t stream);

// Attention over a paged cache: flash_attention_forward_paged, and with query_starts null
// flash_attention_decode_shared (num_tokens == batch_size).
struct PagedCall {
    const void *Q, *K_cache, *V_cache;
    void* O;
    float* L;
    const int *block_table, *prefix_table, *seq_lens, *query_starts;
    int num_tokens, batch_size, num_heads, num_kv_heads;
    int prefix_len, page_size, max_pages, head_dim;
    float scale;
    bool causal;
    void* workspace;  // the caller's, or null
    size_t workspace_bytes;
};
// Bytes of the partial results of a call of these sizes (the others are not read), 0 without
// chunks, -1 where its grid would be too large.
template <typename T>
long long paged_workspace(const PagedCall& call);
template <typename T>
FlashAttentionError launch_paged(const PagedCall& call, hipStream_t stream);

}  // namespace detail
}  // namespace cuflash
