// Validating layer and C ABI of the operators on an 8-bit paged cache (include/cuflash/paged_cache_q8.h).
// As in api.cpp, every check is made before the first HIP call.

#include "launch.hpp"
#include "paged_checks.hpp"
#include "paged_q8_launch.hpp"

namespace cuflash {
namespace {

using E = FlashAttentionError;
using detail::aligned16;

// Null exponents and the code come right behind the other null pointers, which `err` tells of.
E check_cache(E err, const void* k_exp, const void* v_exp, QuantCode code) {
    if (err == E::NULL_POINTER || !k_exp || !v_exp) return E::NULL_POINTER;
    if (code != QuantCode::INT8 && code != QuantCode::E4M3) return E::UNSUPPORTED_DTYPE;
    if (err != E::SUCCESS) return err;
    return aligned16(k_exp) && aligned16(v_exp) ? E::SUCCESS : E::INVALID_DIMENSION;
}

E check_read(const detail::ReadQ8Call& c) {
    if (!c.K_cache || !c.V_cache || !c.K_out || !c.V_out || !c.block_table || !c.seq_lens ||
        !c.key_starts)
        return E::NULL_POINTER;
    E err = detail::check_sizes(c.num_tokens, c.batch_size, c.num_kv_heads, c.num_kv_heads,
                                c.page_size, c.max_pages, c.head_dim);
    if (err != E::SUCCESS) return err;
    if (c.num_pages <= 0) return E::INVALID_DIMENSION;
    err = detail::check_relations(c.num_kv_heads, c.num_kv_heads, c.page_size, c.max_pages);
    if (err != E::SUCCESS) return err;
    if (2LL * c.num_kv_heads * c.head_dim > detail::kIntMax) return E::INVALID_DIMENSION;
    for (const void* p : {c.K_cache, c.V_cache, static_cast<const void*>(c.K_out),
                          static_cast<const void*>(c.V_out)})
        if (!aligned16(p)) return E::INVALID_DIMENSION;
    return E::SUCCESS;
}

template <typename T>
E append_impl(const detail::AppendQ8Call& c, hipStream_t stream) {
    const E err = check_cache(detail::check_append(c.rows, sizeof(T)), c.K_exp, c.V_exp, c.code);
    if (err != E::SUCCESS) return err;
    return detail::launch_append_paged_q8<T>(c, stream);
}

template <typename T>
E read_impl(const detail::ReadQ8Call& c, hipStream_t stream) {
    const E err = check_cache(check_read(c), c.K_exp, c.V_exp, c.code);
    if (err != E::SUCCESS) return err;
    return detail::launch_read_paged_q8<T>(c, stream);
}

template <typename T>
E attention_impl(const detail::PagedQ8Call& c, bool decode, hipStream_t stream) {
    const E err = check_cache(detail::check_attention(c.call, decode), c.K_exp, c.V_exp, c.code);
    if (err != E::SUCCESS) return err;
    // The kernels' offsets in a page have 32 bits.
    if (static_cast<long long>(c.call.page_size) * c.call.num_kv_heads > detail::kIntMax / c.call.head_dim)
        return E::INVALID_DIMENSION;
    return detail::launch_paged_q8<T>(c, stream);
}

template <typename T>
long long workspace_impl(int num_tokens, int batch_size, int num_heads, int num_kv_heads,
                         int head_dim, bool decode) {
    if (detail::check_sizes(num_tokens, batch_size, num_heads, num_kv_heads, 1, 1, head_dim) !=
            E::SUCCESS ||
        num_heads % num_kv_heads != 0 ||
        static_cast<long long>(num_tokens) * num_heads > detail::kIntMax ||
        num_heads > detail::kMaxHeads)
        return -1;
    static const int kStarts = 0;  // not read
    detail::PagedCall c{};
    c.query_starts = decode ? nullptr : &kStarts;
    c.num_tokens = num_tokens;
    c.batch_size = batch_size;
    c.num_heads = num_heads;
    c.num_kv_heads = num_kv_heads;
    c.head_dim = head_dim;
    return detail::paged_q8_workspace<T>(c);
}

}  // namespace

#define CUFLASH_PAGED_CACHE_Q8(SFX, T)                                                            \
    E flash_attention_append_paged_q8(                                                            \
        const T* Q, const T* K, const T* V, T* Q_out, void* K_cache, void* V_cache,               \
        uint8_t* K_exp, uint8_t* V_exp, const int* block_table, const int* seq_lens,              \
        const int* query_starts, const float* rope_cos, const float* rope_sin, int num_tokens,    \
        int batch_size, int num_heads, int num_kv_heads, int q_stride, int k_stride,              \
        int v_stride, int num_pages, int page_size, int max_pages_per_seq, int head_dim,          \
        int rotary_dim, int max_positions, bool interleaved, QuantCode code,                      \
        hipStream_t stream) {                                                                     \
        return append_impl<T>(                                                                    \
            {detail::AppendCall{Q, K, V, Q_out, K_cache, V_cache, block_table, seq_lens,          \
                                query_starts, rope_cos, rope_sin, num_tokens, batch_size,         \
                                num_heads, num_kv_heads, q_stride, k_stride, v_stride, num_pages, \
                                page_size, max_pages_per_seq, head_dim, rotary_dim,               \
                                max_positions, interleaved},                                      \
             K_exp, V_exp, code},                                                                 \
            stream);                                                                              \
    }                                                                                             \
    extern "C" int cuflash_attention_append_paged_q8_##SFX(                                       \
        const T* Q, const T* K, const T* V, T* Q_out, void* K_cache, void* V_cache,               \
        uint8_t* K_exp, uint8_t* V_exp, const int* block_table, const int* seq_lens,              \
        const int* query_starts, const float* rope_cos, const float* rope_sin, int num_tokens,    \
        int batch_size, int num_heads, int num_kv_heads, int q_stride, int k_stride,              \
        int v_stride, int num_pages, int page_size, int max_pages_per_seq, int head_dim,          \
        int rotary_dim, int max_positions, bool interleaved, int code, hipStream_t stream) {      \
        return static_cast<int>(flash_attention_append_paged_q8(                                  \
            Q, K, V, Q_out, K_cache, V_cache, K_exp, V_exp, block_table, seq_lens, query_starts,  \
            rope_cos, rope_sin, num_tokens, batch_size, num_heads, num_kv_heads, q_stride,        \
            k_stride, v_stride, num_pages, page_size, max_pages_per_seq, head_dim, rotary_dim,    \
            max_positions, interleaved, static_cast<QuantCode>(code), stream));                   \
    }                                                                                             \
    E flash_attention_read_paged_q8(                                                              \
        const void* K_cache, const void* V_cache, const uint8_t* K_exp, const uint8_t* V_exp,     \
        T* K_out, T* V_out, const int* block_table, const int* seq_lens, const int* key_starts,   \
        int num_tokens, int batch_size, int num_kv_heads, int num_pages, int page_size,           \
        int max_pages_per_seq, int head_dim, QuantCode code, hipStream_t stream) {                \
        return read_impl<T>(                                                                      \
            {K_cache, V_cache, K_exp, V_exp, K_out, V_out, block_table, seq_lens, key_starts,     \
             num_tokens, batch_size, num_kv_heads, num_pages, page_size, max_pages_per_seq,       \
             head_dim, code},                                                                     \
            stream);                                                                              \
    }                                                                                             \
    extern "C" int cuflash_attention_read_paged_q8_##SFX(                                         \
        const void* K_cache, const void* V_cache, const uint8_t* K_exp, const uint8_t* V_exp,     \
        T* K_out, T* V_out, const int* block_table, const int* seq_lens, const int* key_starts,   \
        int num_tokens, int batch_size, int num_kv_heads, int num_pages, int page_size,           \
        int max_pages_per_seq, int head_dim, int code, hipStream_t stream) {                      \
        return static_cast<int>(flash_attention_read_paged_q8(                                    \
            K_cache, V_cache, K_exp, V_exp, K_out, V_out, block_table, seq_lens, key_starts,      \
            num_tokens, batch_size, num_kv_heads, num_pages, page_size, max_pages_per_seq,        \
            head_dim, static_cast<QuantCode>(code), stream));                                     \
    }                                                                                             \
    E flash_attention_decode_paged_q8(                                                            \
        const T* Q, const void* K_cache, const void* V_cache, const uint8_t* K_exp,               \
        const uint8_t* V_exp, T* O, float* L, const int* block_table, const int* seq_lens,        \
        int batch_size, int num_heads, int num_kv_heads, int page_size, int max_pages_per_seq,    \
        int head_dim, float scale, QuantCode code, void* workspace, size_t workspace_bytes,       \
        hipStream_t stream) {                                                                     \
        return attention_impl<T>(                                                                 \
            {detail::PagedCall{Q, K_cache, V_cache, O, L, block_table, nullptr, seq_lens,         \
                               nullptr, batch_size, batch_size, num_heads, num_kv_heads, 0,       \
                               page_size, max_pages_per_seq, head_dim, scale, false, workspace,   \
                               workspace_bytes},                                                  \
             K_exp, V_exp, code},                                                                 \
            true, stream);                                                                        \
    }                                                                                             \
    extern "C" int cuflash_attention_decode_paged_q8_##SFX(                                       \
        const T* Q, const void* K_cache, const void* V_cache, const uint8_t* K_exp,               \
        const uint8_t* V_exp, T* O, float* L, const int* block_table, const int* seq_lens,        \
        int batch_size, int num_heads, int num_kv_heads, int page_size, int max_pages_per_seq,    \
        int head_dim, float scale, int code, void* workspace, size_t workspace_bytes,             \
        hipStream_t stream) {                                                                     \
        return static_cast<int>(flash_attention_decode_paged_q8(                                  \
            Q, K_cache, V_cache, K_exp, V_exp, O, L, block_table, seq_lens, batch_size,           \
            num_heads, num_kv_heads, page_size, max_pages_per_seq, head_dim, scale,               \
            static_cast<QuantCode>(code), workspace, workspace_bytes, stream));                   \
    }                                                                                             \
    extern "C" long long cuflash_attention_decode_paged_q8_workspace_##SFX(                       \
        int batch_size, int num_heads, int num_kv_heads, int head_dim) {                          \
        return workspace_impl<T>(batch_size, batch_size, num_heads, num_kv_heads, head_dim,       \
                                 true);                                                           \
    }                                                                                             \
    E flash_attention_forward_paged_q8(                                                           \
        const T* Q, const void* K_cache, const void* V_cache, const uint8_t* K_exp,               \
        const uint8_t* V_exp, T* O, float* L, const int* block_table, const int* seq_lens,        \
        const int* query_starts, int num_tokens, int batch_size, int num_heads,                   \
        int num_kv_heads, int page_size, int max_pages_per_seq, int head_dim, float scale,        \
        bool causal, QuantCode code, void* workspace, size_t workspace_bytes,                     \
        hipStream_t stream) {                                                                     \
        return attention_impl<T>(                                                                 \
            {detail::PagedCall{Q, K_cache, V_cache, O, L, block_table, nullptr, seq_lens,         \
                               query_starts, num_tokens, batch_size, num_heads, num_kv_heads, 0,  \
                               page_size, max_pages_per_seq, head_dim, scale, causal, workspace,  \
                               workspace_bytes},                                                  \
             K_exp, V_exp, code},                                                                 \
            false, stream);                                                                       \
    }                                                                                             \
    extern "C" int cuflash_attention_forward_paged_q8_##SFX(                                      \
        const T* Q, const void* K_cache, const void* V_cache, const uint8_t* K_exp,               \
        const uint8_t* V_exp, T* O, float* L, const int* block_table, const int* seq_lens,        \
        const int* query_starts, int num_tokens, int batch_size, int num_heads,                   \
        int num_kv_heads, int page_size, int max_pages_per_seq, int head_dim, float scale,        \
        bool causal, int code, void* workspace, size_t workspace_bytes, hipStream_t stream) {     \
        return static_cast<int>(flash_attention_forward_paged_q8(                                 \
            Q, K_cache, V_cache, K_exp, V_exp, O, L, block_table, seq_lens, query_starts,         \
            num_tokens, batch_size, num_heads, num_kv_heads, page_size, max_pages_per_seq,        \
            head_dim, scale, causal, static_cast<QuantCode>(code), workspace, workspace_bytes,    \
            stream));                                                                             \
    }                                                                                             \
    extern "C" long long cuflash_attention_forward_paged_q8_workspace_##SFX(                      \
        int num_tokens, int batch_size, int num_heads, int num_kv_heads, int head_dim) {          \
        return workspace_impl<T>(num_tokens, batch_size, num_heads, num_kv_heads, head_dim,       \
                                 false);                                                          \
    }
CUFLASH_PAGED_CACHE_Q8(f32, float)
CUFLASH_PAGED_CACHE_Q8(f16, __half)
CUFLASH_PAGED_CACHE_Q8(bf16, __hip_bfloat16)
#undef CUFLASH_PAGED_CACHE_Q8

}  // namespace cuflash
