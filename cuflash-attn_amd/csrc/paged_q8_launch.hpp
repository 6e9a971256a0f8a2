#pragma once

// Internal launcher interface between paged_q8_api.cpp and its kernels (append_q8.hip,
// attention_q8.hip). Arguments have been validated when a launcher runs.

#include "cuflash/paged_cache_q8.h"
#include "paged_launch.hpp"

namespace cuflash {
namespace detail {

struct AppendQ8Call {
    AppendCall rows;  // K_cache, V_cache: codes
    uint8_t *K_exp, *V_exp;
    QuantCode code;
};
template <typename T>
FlashAttentionError launch_append_paged_q8(const AppendQ8Call& call, hipStream_t stream);

struct ReadQ8Call {
    const void *K_cache, *V_cache;
    const uint8_t *K_exp, *V_exp;
    void *K_out, *V_out;
    const int *block_table, *seq_lens, *key_starts;
    int num_tokens, batch_size, num_kv_heads;
    int num_pages, page_size, max_pages, head_dim;
    QuantCode code;
};
template <typename T>
FlashAttentionError launch_read_paged_q8(const ReadQ8Call& call, hipStream_t stream);

// flash_attention_forward_paged_q8, and with query_starts null flash_attention_decode_paged_q8
// (num_tokens == batch_size).
struct PagedQ8Call {
    PagedCall call;  // K_cache, V_cache: codes
    const uint8_t *K_exp, *V_exp;
    QuantCode code;
};
// Bytes of the partial results of a call of these sizes (query_starts: null for a decode; the others are
// not read).
template <typename T>
long long paged_q8_workspace(const PagedCall& call);
template <typename T>
FlashAttentionError launch_paged_q8(const PagedQ8Call& call, hipStream_t stream);

}  // namespace detail
}  // namespace cuflash
