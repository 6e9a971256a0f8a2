#pragma once

// Serving from a paged key/value cache (additive; no counterpart in the reference, which has no
// cache). Beside flash_attention_decode_paged (flash_attention.h), on the same cache:
//   flash_attention_append_paged   writes new tokens' keys and values to their pages, rotating
//                                  queries and keys by their positions on the way;
//   flash_attention_forward_paged  several new tokens of every sequence attend to the cache;
//   flash_attention_decode_shared  one query per sequence, for a batch whose first keys are the
//                                  same pages: these are read once for the whole batch.
//
// Common to the three:
//  * K_cache, V_cache [num_pages, page_size, num_kv_heads, head_dim]; block_table [batch_size,
//    max_pages_per_seq] (int32): key j of sequence b is row j % page_size of page
//    block_table[b][j / page_size].
//  * Tokens are packed, [num_tokens, heads, head_dim]: those of sequence b are query_starts[b] ..
//    query_starts[b + 1] - 1 (int32, batch_size + 1 values that do not decrease), the newest of
//    the sequence. Sequences without tokens are allowed. Tokens from query_starts[batch_size] on
//    are padding: their outputs are left as they were.
//  * seq_lens [batch_size] (int32) counts a sequence's keys WITH its new tokens, so token t of
//    sequence b stands at position seq_lens[b] - (query_starts[b + 1] - t), and the same array
//    goes to the append and to the attention after it. The attentions take a length past the block
//    table's max_pages_per_seq * page_size keys for that many.
//  * head_dim 32, 64 or 128; num_heads a multiple of num_kv_heads (query head h reads key/value
//    head h / (num_heads / num_kv_heads)).
//  * Pointers and token strides are multiples of 16 bytes. Every pointer is a device pointer.
//    Calls are asynchronous on `stream` and can be captured into a HIP graph (see Workspaces).
// Validation, in this order: null pointers (NULL_POINTER), dimensions that are not positive
// (INVALID_DIMENSION), head_dim (UNSUPPORTED_HEAD_DIM), scale (INVALID_DIMENSION), then the
// relations between sizes (DIMENSION_MISMATCH), sizes that are too large and alignment
// (INVALID_DIMENSION). Too large: page_size * max_pages_per_seq beyond 2^31 - 1024, num_tokens *
// num_heads beyond 2^31 - 1, num_heads beyond 65535 (the attentions), more than 2^32 - 1 threads in one
// launch.

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "cuflash/export.h"
#include "cuflash/flash_attention.h"

namespace cuflash {

// ---- Append ----
// Writes K [num_tokens, num_kv_heads, head_dim] and V to the cache rows of their positions. Rows
// of Q, K and V are q_stride, k_stride and v_stride elements apart from token to token (the heads of
// a token are contiguous), so the three may be parts of one projection's output.
// rope_cos, rope_sin: float [max_positions, rotary_dim / 2], or both null (no rotation; rotary_dim
// 0). The first rotary_dim elements of every query and key head (a multiple of 16, at most head_dim)
// are rotated by row p = position: the pair (x1, x2) = elements (i, i + rotary_dim / 2), or (2 i,
// 2 i + 1) if `interleaved`, becomes (x1 cos - x2 sin, x2 cos + x1 sin), computed in float and
// rounded once. Rotated queries go to Q_out [num_tokens, num_heads, head_dim], which may be Q itself
// where Q is packed (q_stride = num_heads * head_dim; otherwise DIMENSION_MISMATCH). Q and Q_out may both be null.
// query_starts may be null: then token t is the one new token of sequence t (num_tokens ==
// batch_size).
// What the host cannot see is not an error but left out: a token whose position is negative or past
// the block table, and one whose page is not in [0, num_pages) (so -1 marks rows that have none), is
// not written; the rotated elements of a query whose position is outside the rotation's tables become NaN,
// and its token is not written. Where tables name one cache row for two tokens, it holds parts of either afterwards.
CUFLASH_EXPORT FlashAttentionError flash_attention_append_paged(
    const float* Q, const float* K, const float* V, float* Q_out, float* K_cache, float* V_cache,
    const int* block_table, const int* seq_lens, const int* query_starts, const float* rope_cos,
    const float* rope_sin, int num_tokens, int batch_size, int num_heads, int num_kv_heads,
    int q_stride, int k_stride, int v_stride, int num_pages, int page_size, int max_pages_per_seq,
    int head_dim, int rotary_dim, int max_positions, bool interleaved, hipStream_t stream = 0);
CUFLASH_EXPORT FlashAttentionError flash_attention_append_paged(
    const __half* Q, const __half* K, const __half* V, __half* Q_out, __half* K_cache,
    __half* V_cache, const int* block_table, const int* seq_lens, const int* query_starts,
    const float* rope_cos, const float* rope_sin, int num_tokens, int batch_size, int num_heads,
    int num_kv_heads, int q_stride, int k_stride, int v_stride, int num_pages, int page_size,
    int max_pages_per_seq, int head_dim, int rotary_dim, int max_positions, bool interleaved,
    hipStream_t stream = 0);
CUFLASH_EXPORT FlashAttentionError flash_attention_append_paged(
    const __hip_bfloat16* Q, const __hip_bfloat16* K, const __hip_bfloat16* V,
    __hip_bfloat16* Q_out, __hip_bfloat16* K_cache, __hip_bfloat16* V_cache,
    const int* block_table, const int* seq_lens, const int* query_starts, const float* rope_cos,
    const float* rope_sin, int num_tokens, int batch_size, int num_heads, int num_kv_heads,
    int q_stride, int k_stride, int v_stride, int num_pages, int page_size, int max_pages_per_seq,
    int head_dim, int rotary_dim, int max_positions, bool interleaved, hipStream_t stream = 0);

// ---- Workspaces of the two attentions ----
// Keys that are cut into chunks leave partial results in a workspace. With workspace null the library
// uses its own per-stream buffer, as every call with a workspace does (see
// cuflash_release_workspaces). A call that is captured into a graph gets its workspace from the
// caller: a device buffer of the size that cuflash_attention_forward_paged_workspace_* and
// cuflash_attention_decode_shared_workspace_* return for its sizes, 256-byte aligned, that stays
// allocated as long as the graph and is not used by other work while a replay runs (graphs that are
// replayed one after the other may share it). Captured without one, the forward runs in one chunk,
// slower where few tokens meet long caches and with sums in another order, and the shared decode is
// refused: OUT_OF_MEMORY. A workspace that is given is used by eager calls too; one that is too small
// is OUT_OF_MEMORY, one that is not aligned INVALID_DIMENSION.
// ---- Several new tokens of every sequence ----
// O = softmax(scale Q K^T) V over the cache, L the logsumexp: Q, O [num_tokens, num_heads,
// head_dim], L [num_tokens, num_heads] float. In 16 bits the softmax's weights are rounded to that type
// before they meet V (the shared decode's too), as in the library's matrix-core kernels; scores and sums are
// float. Token t of sequence b sees all seq_lens[b] keys (fewer
// where the block table ends before), with `causal` those up to its own position. A query that sees
// no key, or whose scores are all -inf, has O = 0 and L = -inf. How keys are cut goes by num_tokens: beside
// prompts that fill the chip, or padding as long, a token with a cache much longer than these is faster in a
// call of its own. Cache rows from seq_lens[b] on and
// table entries past a sequence's pages are not read. The entries of a sequence's keys must name pages
// of the cache (they are not range-checked). Keys that a query does not see do not reach it, whatever
// they hold. Of the values that `causal` hides from it it may take 0 times those of up to 94 positions past
// its own (the 32 rows that share a wave end up to 31 positions later, in blocks of 64 keys): a NaN or an
// infinity there makes its output NaN. A query that sees no key has O = 0 whatever the cache holds.
CUFLASH_EXPORT FlashAttentionError flash_attention_forward_paged(
    const float* Q, const float* K_cache, const float* V_cache, float* O, float* L,
    const int* block_table, const int* seq_lens, const int* query_starts, int num_tokens,
    int batch_size, int num_heads, int num_kv_heads, int page_size, int max_pages_per_seq,
    int head_dim, float scale, bool causal, void* workspace,
    size_t workspace_bytes, hipStream_t stream = 0);
CUFLASH_EXPORT FlashAttentionError flash_attention_forward_paged(
    const __half* Q, const __half* K_cache, const __half* V_cache, __half* O, float* L,
    const int* block_table, const int* seq_lens, const int* query_starts, int num_tokens,
    int batch_size, int num_heads, int num_kv_heads, int page_size, int max_pages_per_seq,
    int head_dim, float scale, bool causal, void* workspace,
    size_t workspace_bytes, hipStream_t stream = 0);
CUFLASH_EXPORT FlashAttentionError flash_attention_forward_paged(
    const __hip_bfloat16* Q, const __hip_bfloat16* K_cache, const __hip_bfloat16* V_cache,
    __hip_bfloat16* O, float* L, const int* block_table, const int* seq_lens,
    const int* query_starts, int num_tokens, int batch_size, int num_heads, int num_kv_heads,
    int page_size, int max_pages_per_seq, int head_dim, float scale, bool causal, void* workspace,
    size_t workspace_bytes, hipStream_t stream = 0);

// ---- Decode of a batch that shares its first keys ----
// flash_attention_decode_paged for sequences whose first prefix_len keys are the same: these are read
// from the pages that prefix_table (int32, ceil(prefix_len / page_size) of them) names, once for the
// batch, the others from block_table. Q, O [batch_size, num_heads, 1, head_dim], L [batch_size,
// num_heads] float. seq_lens counts all keys of a sequence, the shared ones among them; positions stay
// what they are, so block_table[b][j / page_size] is read for the keys j >= prefix_len only (where the
// prefix ends inside a page, that entry is the sequence's own page, whose first rows are not read). A
// sequence shorter than the prefix sees its first seq_lens[b] keys; of the shared values behind these it may
// take 0 times any, which a NaN or an infinity there makes NaN (a length of 0: O = 0 all the same).
// prefix_len 0 is flash_attention_decode_paged, which does not use the workspace (captured: the same result
// up to rounding, in the caller's workspace); prefix_len past the block table's capacity is DIMENSION_MISMATCH.
CUFLASH_EXPORT FlashAttentionError flash_attention_decode_shared(
    const float* Q, const float* K_cache, const float* V_cache, float* O, float* L,
    const int* prefix_table, const int* block_table, const int* seq_lens, int batch_size,
    int num_heads, int num_kv_heads, int prefix_len, int page_size, int max_pages_per_seq,
    int head_dim, float scale, void* workspace, size_t workspace_bytes, hipStream_t stream = 0);
CUFLASH_EXPORT FlashAttentionError flash_attention_decode_shared(
    const __half* Q, const __half* K_cache, const __half* V_cache, __half* O, float* L,
    const int* prefix_table, const int* block_table, const int* seq_lens, int batch_size,
    int num_heads, int num_kv_heads, int prefix_len, int page_size, int max_pages_per_seq,
    int head_dim, float scale, void* workspace, size_t workspace_bytes, hipStream_t stream = 0);
CUFLASH_EXPORT FlashAttentionError flash_attention_decode_shared(
    const __hip_bfloat16* Q, const __hip_bfloat16* K_cache, const __hip_bfloat16* V_cache,
    __hip_bfloat16* O, float* L, const int* prefix_table, const int* block_table,
    const int* seq_lens, int batch_size, int num_heads, int num_kv_heads, int prefix_len,
    int page_size, int max_pages_per_seq, int head_dim, float scale, void* workspace,
    size_t workspace_bytes, hipStream_t stream = 0);

}  // namespace cuflash

#ifdef __cplusplus
extern "C" {
#endif

// C ABI of the functions above; the integer value of cuflash::FlashAttentionError. The workspace
// sizes: bytes for a call of these sizes, 0 where none is needed, -1 where it would be refused.
#define CUFLASH_DECLARE_PAGED_CACHE(SFX, T)                                                       \
    CUFLASH_EXPORT int cuflash_attention_append_paged_##SFX(                                      \
        const T* Q, const T* K, const T* V, T* Q_out, T* K_cache, T* V_cache,                     \
        const int* block_table, const int* seq_lens, const int* query_starts,                     \
        const float* rope_cos, const float* rope_sin, int num_tokens, int batch_size,             \
        int num_heads, int num_kv_heads, int q_stride, int k_stride, int v_stride, int num_pages, \
        int page_size, int max_pages_per_seq, int head_dim, int rotary_dim, int max_positions,    \
        bool interleaved, hipStream_t stream);                                                    \
    CUFLASH_EXPORT int cuflash_attention_forward_paged_##SFX(                                     \
        const T* Q, const T* K_cache, const T* V_cache, T* O, float* L, const int* block_table,   \
        const int* seq_lens, const int* query_starts, int num_tokens, int batch_size,             \
        int num_heads, int num_kv_heads, int page_size, int max_pages_per_seq, int head_dim,      \
        float scale, bool causal, void* workspace, size_t workspace_bytes, hipStream_t stream);   \
    CUFLASH_EXPORT long long cuflash_attention_forward_paged_workspace_##SFX(                     \
        int num_tokens, int batch_size, int num_heads, int num_kv_heads, int head_dim);           \
    CUFLASH_EXPORT int cuflash_attention_decode_shared_##SFX(                                     \
        const T* Q, const T* K_cache, const T* V_cache, T* O, float* L, const int* prefix_table,  \
        const int* block_table, const int* seq_lens, int batch_size, int num_heads,               \
        int num_kv_heads, int prefix_len, int page_size, int max_pages_per_seq, int head_dim,     \
        float scale, void* workspace, size_t workspace_bytes, hipStream_t stream);                \
    CUFLASH_EXPORT long long cuflash_attention_decode_shared_workspace_##SFX(                     \
        int batch_size, int num_heads, int num_kv_heads, int head_dim);
CUFLASH_DECLARE_PAGED_CACHE(f32, float)
CUFLASH_DECLARE_PAGED_CACHE(f16, __half)
CUFLASH_DECLARE_PAGED_CACHE(bf16, __hip_bfloat16)
#undef CUFLASH_DECLARE_PAGED_CACHE

#ifdef __cplusplus
}
#endif
