#pragma once

// Serving from a paged key/value cache of one byte an element (additive; no counterpart in the
// reference). Beside the operators of cuflash/paged_cache.h, on a cache of half the bytes:
//   flash_attention_append_paged_q8   writes new tokens' keys and values to their pages, rotating
//                                     queries and keys by their positions and quantising on the way;
//   flash_attention_read_paged_q8     the numbers that tokens' keys and values have in the cache;
//   flash_attention_decode_paged_q8   one query per sequence over the cache;
//   flash_attention_forward_paged_q8  several new tokens of every sequence over the cache.
//
// The cache:
//  * K_cache, V_cache [num_pages, page_size, num_kv_heads, head_dim]: codes of one byte, all of them
//    int8 (-127 .. 127) or all of them e4m3 (OCP, the largest number is 448; 0x7f and 0xff are NaN).
//  * K_exp, V_exp [num_pages, num_kv_heads, page_size]: one byte x for the head_dim codes of a key (of
//    a value) of one key/value head. An element is code * 2^(x - 127); x = 255 makes every element NaN.
//    A power of two because such a product is exact in float and bf16, and in fp16 where that has the
//    number: the attentions take it as it is, without a rounding, and gfx950 scales as it converts.
//  * In calls with fp16 queries an element beyond fp16's range is its nearest fp16 number, or infinite.
//    The fp16 append writes none that is infinite. x above 248 (e4m3: 246), which no append writes, leads beyond
//    float's range: the attentions take such an element as infinite or as the number that it is.
// Pages, tables, packed tokens, positions, padding, lengths, head_dim, head groups, alignment (of
// the exponents' pointers too) and errors are as in cuflash/paged_cache.h; a QuantCode that is none is
// UNSUPPORTED_DTYPE, found after null pointers, and a page of 2^31 bytes or more in an attention INVALID_DIMENSION.

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cuflash/export.h"
#include "cuflash/flash_attention.h"

namespace cuflash {

enum class QuantCode : int { INT8 = 0, E4M3 = 1 };

// The functions below exist for T = float, __half and __hip_bfloat16.
//
// ---- Append ----
// flash_attention_append_paged with a quantised cache. A rotated pair is (x1 cos - x2 sin, x2 cos + x1
// sin) in float, products and sum each rounded; queries are then rounded to T, keys quantised as they
// are. A row, the head_dim elements of one key/value head, gets the least exponent e with
// max |element| <= top 2^e (top = 127 or 448), but at least -100 and at most 121 (e4m3: 119), for fp16 9
// (7), beyond which the largest code would not be finite in T; its codes are element / 2^e rounded to
// the nearest, ties to even, those past the top the top; x = e + 127. A row with an infinity or a NaN
// gets x = 255 and codes 0 (e4m3: NaN): it reads as NaN.
#define CUFLASH_Q8_APPEND(T)                                                                      \
    CUFLASH_EXPORT FlashAttentionError flash_attention_append_paged_q8(                           \
        const T* Q, const T* K, const T* V, T* Q_out, void* K_cache, void* V_cache,               \
        uint8_t* K_exp, uint8_t* V_exp, const int* block_table, const int* seq_lens,              \
        const int* query_starts, const float* rope_cos, const float* rope_sin, int num_tokens,    \
        int batch_size, int num_heads, int num_kv_heads, int q_stride, int k_stride,              \
        int v_stride, int num_pages, int page_size, int max_pages_per_seq, int head_dim,          \
        int rotary_dim, int max_positions, bool interleaved, QuantCode code,                      \
        hipStream_t stream = 0)

// ---- Read ----
// K_out, V_out [num_tokens, num_kv_heads, head_dim]: the keys and values of tokens key_starts[b] ..
// key_starts[b + 1] - 1 of every sequence b, its newest, as T: what the append of those tokens left in
// the cache. A token without a row (a negative position, one past the table, a page that is none of
// [0, num_pages)) reads as NaN. Rows from key_starts[batch_size] on are left as they were.
#define CUFLASH_Q8_READ(T)                                                                        \
    CUFLASH_EXPORT FlashAttentionError flash_attention_read_paged_q8(                             \
        const void* K_cache, const void* V_cache, const uint8_t* K_exp, const uint8_t* V_exp,     \
        T* K_out, T* V_out, const int* block_table, const int* seq_lens, const int* key_starts,   \
        int num_tokens, int batch_size, int num_kv_heads, int num_pages, int page_size,           \
        int max_pages_per_seq, int head_dim, QuantCode code, hipStream_t stream = 0)

// ---- Attention ----
// flash_attention_decode_paged and flash_attention_forward_paged over a quantised cache, with the
// same meaning of every argument, masks, empty rows and outputs. Where keys are cut into parts these
// leave partial results in a workspace, as described in cuflash/paged_cache.h: null takes the library's, a
// captured call needs the caller's, of the size that the *_workspace_* functions return, and is refused
// without one (OUT_OF_MEMORY). Only a decode from tables of at most 1024 keys (page_size * max_pages_per_seq) never
// takes one. Short tables (page_size * max_pages_per_seq) are faster than long ones that hold the same lengths: such a
// call may be one launch. A call of several launches that may have more than 2^30 tiles of rows, which takes some 900
// million sequences with tokens, or 2^31 - 63 sequences and more is refused (INVALID_DIMENSION; the *_workspace_*
// functions do not look at this).
// All keys are cut into equal shares, whatever the lengths, so no long cache leaves the rest of the chip without work.
// But in 16 bits a call takes the tokens of all its sequences in tiles of one height, of 256 rows where their average
// is more than 48 rows (head_dim 64 and 32: 96; a single sequence: 16): single tokens beside prompts then cost as much
// for each of their keys as 256 rows do, and are faster in a call of their own (4 prompts of 2000 tokens and 32 tokens
// behind 4000 keys 367 us, in two calls 255; 5000 tokens and one behind 100000 keys 430 and 348, behind 8000 keys 334
// and 337; bf16, 32 heads over 8, head_dim 128).
// In 16 bits the softmax's weights are rounded to that type before they meet V (also where a query head has a key/value
// head for itself, where flash_attention_decode_paged keeps them in float). float queries take part as three bf16
// numbers each, and so do their weights: what is lost is below float's own rounding, at more than the rate of the
// float matrix products (193 TFLOP/s in a prompt of 4096 tokens over int8, head_dim 128, 219 over e4m3, head_dim 64,
// where a large product of float matrices runs at 151).
// Most calls scale the scores of int8 keys instead of their codes: queries of 2^113 and more, which bf16 and float
// have, may there reach infinite scores whose scaled numbers would be finite.
// Cache rows from seq_lens[b] on may hold anything; table entries past a sequence's pages are not read. Keys that
// a query does not see do not reach it. Of the values that `causal` hides from it it may take 0 times those of up to
// 94 positions past its own (the 32 rows that share a wave end up to 31 positions later, in steps of 64 keys): a NaN
// there makes its output NaN. A query that sees no key has O = 0 whatever the cache holds.
#define CUFLASH_Q8_DECODE(T)                                                                      \
    CUFLASH_EXPORT FlashAttentionError flash_attention_decode_paged_q8(                           \
        const T* Q, const void* K_cache, const void* V_cache, const uint8_t* K_exp,               \
        const uint8_t* V_exp, T* O, float* L, const int* block_table, const int* seq_lens,        \
        int batch_size, int num_heads, int num_kv_heads, int page_size, int max_pages_per_seq,    \
        int head_dim, float scale, QuantCode code, void* workspace, size_t workspace_bytes,       \
        hipStream_t stream = 0)
#define CUFLASH_Q8_FORWARD(T)                                                                     \
    CUFLASH_EXPORT FlashAttentionError flash_attention_forward_paged_q8(                          \
        const T* Q, const void* K_cache, const void* V_cache, const uint8_t* K_exp,               \
        const uint8_t* V_exp, T* O, float* L, const int* block_table, const int* seq_lens,        \
        const int* query_starts, int num_tokens, int batch_size, int num_heads,                   \
        int num_kv_heads, int page_size, int max_pages_per_seq, int head_dim, float scale,        \
        bool causal, QuantCode code, void* workspace, size_t workspace_bytes,                     \
        hipStream_t stream = 0)

CUFLASH_Q8_APPEND(float);
CUFLASH_Q8_APPEND(__half);
CUFLASH_Q8_APPEND(__hip_bfloat16);
CUFLASH_Q8_READ(float);
CUFLASH_Q8_READ(__half);
CUFLASH_Q8_READ(__hip_bfloat16);
CUFLASH_Q8_DECODE(float);
CUFLASH_Q8_DECODE(__half);
CUFLASH_Q8_DECODE(__hip_bfloat16);
CUFLASH_Q8_FORWARD(float);
CUFLASH_Q8_FORWARD(__half);
CUFLASH_Q8_FORWARD(__hip_bfloat16);
#undef CUFLASH_Q8_APPEND
#undef CUFLASH_Q8_READ
#undef CUFLASH_Q8_DECODE
#undef CUFLASH_Q8_FORWARD

}  // namespace cuflash

#ifdef __cplusplus
extern "C" {
#endif

// C ABI of the functions above; the integer value of cuflash::FlashAttentionError. `code`: 0 int8, 1
// e4m3. The workspace sizes: bytes for a call of these sizes, 0 where none is needed, -1 where it would be
// refused.
#define CUFLASH_DECLARE_PAGED_CACHE_Q8(SFX, T)                                                    \
    CUFLASH_EXPORT int cuflash_attention_append_paged_q8_##SFX(                                   \
        const T* Q, const T* K, const T* V, T* Q_out, void* K_cache, void* V_cache,               \
        uint8_t* K_exp, uint8_t* V_exp, const int* block_table, const int* seq_lens,              \
        const int* query_starts, const float* rope_cos, const float* rope_sin, int num_tokens,    \
        int batch_size, int num_heads, int num_kv_heads, int q_stride, int k_stride,              \
        int v_stride, int num_pages, int page_size, int max_pages_per_seq, int head_dim,          \
        int rotary_dim, int max_positions, bool interleaved, int code, hipStream_t stream);       \
    CUFLASH_EXPORT int cuflash_attention_read_paged_q8_##SFX(                                     \
        const void* K_cache, const void* V_cache, const uint8_t* K_exp, const uint8_t* V_exp,     \
        T* K_out, T* V_out, const int* block_table, const int* seq_lens, const int* key_starts,   \
        int num_tokens, int batch_size, int num_kv_heads, int num_pages, int page_size,           \
        int max_pages_per_seq, int head_dim, int code, hipStream_t stream);                       \
    CUFLASH_EXPORT int cuflash_attention_decode_paged_q8_##SFX(                                   \
        const T* Q, const void* K_cache, const void* V_cache, const uint8_t* K_exp,               \
        const uint8_t* V_exp, T* O, float* L, const int* block_table, const int* seq_lens,        \
        int batch_size, int num_heads, int num_kv_heads, int page_size, int max_pages_per_seq,    \
        int head_dim, float scale, int code, void* workspace, size_t workspace_bytes,             \
        hipStream_t stream);                                                                      \
    CUFLASH_EXPORT long long cuflash_attention_decode_paged_q8_workspace_##SFX(                   \
        int batch_size, int num_heads, int num_kv_heads, int head_dim);                           \
    CUFLASH_EXPORT int cuflash_attention_forward_paged_q8_##SFX(                                  \
        const T* Q, const void* K_cache, const void* V_cache, const uint8_t* K_exp,               \
        const uint8_t* V_exp, T* O, float* L, const int* block_table, const int* seq_lens,        \
        const int* query_starts, int num_tokens, int batch_size, int num_heads,                   \
        int num_kv_heads, int page_size, int max_pages_per_seq, int head_dim, float scale,        \
        bool causal, int code, void* workspace, size_t workspace_bytes, hipStream_t stream);      \
    CUFLASH_EXPORT long long cuflash_attention_forward_paged_q8_workspace_##SFX(                  \
        int num_tokens, int batch_size, int num_heads, int num_kv_heads, int head_dim);
CUFLASH_DECLARE_PAGED_CACHE_Q8(f32, float)
CUFLASH_DECLARE_PAGED_CACHE_Q8(f16, __half)
CUFLASH_DECLARE_PAGED_CACHE_Q8(bf16, __hip_bfloat16)
#undef CUFLASH_DECLARE_PAGED_CACHE_Q8

#ifdef __cplusplus
}
#endif
