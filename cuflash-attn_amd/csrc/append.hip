// Append to a paged cache for gfx950 (MI355X): new tokens' keys and values go to the rows of their
// positions, queries and keys rotated on the way (cuflash/paged_cache.h has the definitions).
//
// One workgroup per token; a lane owns two 16-byte chunks of one head's row, in a rotated row the
// two that hold the elements of the same pairs, so every element is read and written once, and a
// rotation in place (Q_out == Q) reads both chunks before it writes either. The rows do not depend
// on the token's place in the cache, so their loads run beside the walk to it: query_starts ->
// seq_lens -> block_table, three loads that need each other.
// Bound by memory: the rows are read and written once, 3 operations per rotated element. 36856 tokens of 48
// heads, head_dim 128, bf16: 151 to 156 us, 5.9 to 6.1 TB/s (a copy of 1 GiB runs at 5.1); one token 2.4 us.
// Where a token's rows are small its walk shows: 65536 tokens of 10 heads, head_dim 32, bf16 (640 bytes, 20 of
// a wave's lanes) 26 us, 3.5 TB/s, a copy of as many bytes 14; in fp32 28 us, the copy 25.

#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "launch.hpp"
#include "paged_launch.hpp"
#include "profile.hpp"
#include "wave.hpp"

namespace cuflash {
namespace dev {

struct AppendArgs {
    const int* block_table;
    const int* seq_lens;
    const int* query_starts;
    const float* rope_cos;
    const float* rope_sin;
    int B, H, Hkv;  // H 0: no queries
    int q_stride, k_stride, v_stride;
    int num_pages, page_size, max_pages;
    int rotary, max_positions;
};

template <typename T, int D, bool kInterleaved>
__global__ void __launch_bounds__(1024)
    append_kernel(const typename Mma<T>::elem* Q, const typename Mma<T>::elem* K,
                  const typename Mma<T>::elem* V, typename Mma<T>::elem* Q_out,
                  typename Mma<T>::elem* K_cache, typename Mma<T>::elem* V_cache, AppendArgs a) {
    using E = typename Mma<T>::elem;
    constexpr int VEC = 16 / static_cast<int>(sizeof(E));
    constexpr int UPR = D / (2 * VEC);  // units (pairs of chunks) per row
    const int t = blockIdx.x;
    const int units = (a.H + 2 * a.Hkv) * UPR;
    const int turned = a.rotary / (2 * VEC);  // rotated units of a row

    // Unit u: a head's row of the token and its two chunks there, (w, w + rotary / 2) where the pairs
    // span the rotated part, else neighbours.
    int head, w, c0, c1;
    bool is_q, is_v, turn;
    u32x4 x0, x1;
    auto fetch = [&](int u) {
        const int row = u / UPR;
        w = u % UPR;
        is_q = row >= 2 * a.Hkv;
        is_v = !is_q && row >= a.Hkv;
        head = is_q ? row - 2 * a.Hkv : is_v ? row - a.Hkv : row;
        turn = !is_v && w < turned;
        c0 = turn && !kInterleaved ? w * VEC : 2 * w * VEC;
        c1 = turn && !kInterleaved ? c0 + a.rotary / 2 : c0 + VEC;
        const E* src = (is_q   ? Q + static_cast<size_t>(t) * a.q_stride
                        : is_v ? V + static_cast<size_t>(t) * a.v_stride
                               : K + static_cast<size_t>(t) * a.k_stride) +
                       head * D;
        x0 = ld16(src + c0);
        x1 = ld16(src + c1);
    };
    int u = threadIdx.x;
    fetch(min(u, units - 1));  // every lane stays for the walk to the cache row

    int b = t;
    int last = t + 1;  // end of the sequence's tokens
    if (a.query_starts) {
        b = sequence_of(a.query_starts, a.B, t);
        if (b == a.B) return;  // padding
        last = a.query_starts[b + 1];
    }
    // -1: no position, or one outside the rotation's tables.
    int pos = static_cast<int>(
        max(-1LL, static_cast<long long>(a.seq_lens[b]) - (static_cast<long long>(last) - t)));
    if (a.rotary > 0 && pos >= a.max_positions) pos = -1;
    long long cache_row = -1;  // -1: the token is not written
    if (pos >= 0 && pos / a.page_size < a.max_pages) {
        const int page = a.block_table[static_cast<size_t>(b) * a.max_pages + pos / a.page_size];
        if (page >= 0 && page < a.num_pages)
            cache_row = static_cast<long long>(page) * a.page_size + pos % a.page_size;
    }

    for (; u < units; u += blockDim.x) {
        if (u != static_cast<int>(threadIdx.x)) fetch(u);
        E* dst;
        if (is_q) {
            dst = Q_out + (static_cast<size_t>(t) * a.H + head) * D;
        } else {
            if (cache_row < 0) continue;
            dst = (is_v ? V_cache : K_cache) +
                  (static_cast<size_t>(cache_row) * a.Hkv + head) * D;
        }
        if (turn && pos < 0) {
            // Outside the tables (a key of such a token is not written): NaN in every type.
            x0 = x1 = u32x4{0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu};
        } else if (turn) {
            const size_t at = static_cast<size_t>(pos) * (a.rotary / 2) + w * VEC;
            float c[VEC], s[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i += 4) {
                const f32x4 c4 = __builtin_bit_cast(f32x4, ld16(a.rope_cos + at + i));
                const f32x4 s4 = __builtin_bit_cast(f32x4, ld16(a.rope_sin + at + i));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    c[i + j] = c4[j];
                    s[i + j] = s4[j];
                }
            }
            float x[2 * VEC];
            if constexpr (std::is_same<T, float>::value) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = __uint_as_float(x0[i]);
                    x[4 + i] = __uint_as_float(x1[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[2 * i] = Elem<T>::to_f(static_cast<uint16_t>(x0[i]));
                    x[2 * i + 1] = Elem<T>::to_f(static_cast<uint16_t>(x0[i] >> 16));
                    x[VEC + 2 * i] = Elem<T>::to_f(static_cast<uint16_t>(x1[i]));
                    x[VEC + 2 * i + 1] = Elem<T>::to_f(static_cast<uint16_t>(x1[i] >> 16));
                }
            }
            // Pair i of the unit: elements (i, VEC + i) of x, or (2 i, 2 i + 1).
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                float& p = x[kInterleaved ? 2 * i : i];
                float& q = x[kInterleaved ? 2 * i + 1 : VEC + i];
                const float np = fmaf(p, c[i], -(q * s[i]));
                q = fmaf(q, c[i], p * s[i]);
                p = np;
            }
            if constexpr (std::is_same<T, float>::value) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x0[i] = __float_as_uint(x[i]);
                    x1[i] = __float_as_uint(x[4 + i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x0[i] = Elem<T>::pack2(x[2 * i], x[2 * i + 1]);
                    x1[i] = Elem<T>::pack2(x[VEC + 2 * i], x[VEC + 2 * i + 1]);
                }
            }
        }
        st16(dst + c0, x0);
        st16(dst + c1, x1);
    }
}

}  // namespace dev

namespace detail {
namespace {

template <typename T, int D>
FlashAttentionError run_append(const AppendCall& c, hipStream_t stream) {
    using E = typename dev::Mma<T>::elem;
    dev::AppendArgs a{};
    a.block_table = c.block_table;
    a.seq_lens = c.seq_lens;
    a.query_starts = c.query_starts;
    a.rope_cos = c.rope_cos;
    a.rope_sin = c.rope_sin;
    a.B = c.batch_size;
    a.H = c.Q ? c.num_heads : 0;
    a.Hkv = c.num_kv_heads;
    a.q_stride = c.q_stride;
    a.k_stride = c.k_stride;
    a.v_stride = c.v_stride;
    a.num_pages = c.num_pages;
    a.page_size = c.page_size;
    a.max_pages = c.max_pages;
    a.rotary = c.rotary_dim;
    a.max_positions = c.max_positions;
    constexpr int kUnits = D * static_cast<int>(sizeof(E)) / 32;  // per row
    const long long units = (static_cast<long long>(a.H) + 2LL * a.Hkv) * kUnits;
    const int threads = static_cast<int>(std::min(1024LL, (units + 63) / 64 * 64));
    // A launch has at most 2^32 - 1 threads in x.
    if (static_cast<long long>(c.num_tokens) * threads > 0xffffffffLL)
        return FlashAttentionError::INVALID_DIMENSION;
    ProfileEvents tok = profile_kernel<T, D>("append");
    auto go = [&](auto kernel) {
        launch_kernel(tok, kernel, dim3(static_cast<unsigned>(c.num_tokens)),
                      dim3(static_cast<unsigned>(threads)), 0, stream,
                      static_cast<const E*>(c.Q), static_cast<const E*>(c.K),
                      static_cast<const E*>(c.V), static_cast<E*>(c.Q_out),
                      static_cast<E*>(c.K_cache), static_cast<E*>(c.V_cache), a);
    };
    if (c.interleaved)
        go(dev::append_kernel<T, D, true>);
    else
        go(dev::append_kernel<T, D, false>);
    return from_hip(hipGetLastError());
}

}  // namespace

template <typename T>
FlashAttentionError launch_append_paged(const AppendCall& c, hipStream_t stream) {
    switch (c.head_dim) {
        case 32:
            return run_append<T, 32>(c, stream);
        case 64:
            return run_append<T, 64>(c, stream);
        case 128:
            return run_append<T, 128>(c, stream);
    }
    return FlashAttentionError::UNSUPPORTED_HEAD_DIM;
}
template FlashAttentionError launch_append_paged<float>(const AppendCall&, hipStream_t);
template FlashAttentionError launch_append_paged<__half>(const AppendCall&, hipStream_t);
template FlashAttentionError launch_append_paged<__hip_bfloat16>(const AppendCall&, hipStream_t);

}  // namespace detail
}  // namespace cuflash
