#pragma once

// Internal launcher interface between the validating paged-cache API (paged_api.cpp) and its
// kernels (append.hip). Arguments have been validated when a launcher runs.

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

}  // namespace detail
}  // namespace cuflash
