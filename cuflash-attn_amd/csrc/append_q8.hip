// Into an 8-bit paged cache and out of it, for gfx950 (MI355X): append_q8_kernel rotates new tokens'
// queries and keys and writes keys and values as codes with one exponent a row, read_q8_kernel gives the
// numbers that tokens' rows have (cuflash/paged_cache_q8.h has the definitions).
//
// As in append.hip a workgroup has a token and a lane two 16-byte chunks of one head's row, in a rotated
// row the two that hold the elements of the same pairs. A row's largest element is then found among the
// D / (2 VEC) neighbouring lanes that hold it, by DPP, and each lane turns its elements into codes in its
// registers: every element is read once and written once.
// The exponent is exact integer arithmetic on the bits of the largest element and of the top code, and
// everything before the codes' rounding is single float operations (no fused products), so that the same
// operations give the same codes anywhere.

#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "launch.hpp"
#include "paged_q8_launch.hpp"
#include "profile.hpp"
#include "q8.hpp"
#include "wave.hpp"

namespace cuflash {
namespace dev {

struct RowsQ8Args {
    const int* block_table;
    const int* seq_lens;
    const int* starts;  // null: token t is the newest of sequence t
    int B, Hkv;
    int num_pages, page_size, max_pages;
};

// Token t's position in its sequence, -1 where that is negative, and its row's place in the cache.
struct TokenRow {
    bool padding;
    int pos;
    int page, row;  // page -1: none

    __device__ __forceinline__ TokenRow(const RowsQ8Args& a, int t) {
        int b = t, last = t + 1;
        if (a.starts) {
            b = sequence_of(a.starts, a.B, t);
            padding = b == a.B;
            if (padding) return;
            last = a.starts[b + 1];
        }
        padding = false;
        pos = static_cast<int>(
            max(-1LL, static_cast<long long>(a.seq_lens[b]) - (static_cast<long long>(last) - t)));
        page = -1;
        row = 0;
        if (pos < 0) return;
        const int entry = pos / a.page_size;
        if (entry >= a.max_pages) return;
        row = pos - entry * a.page_size;
        page = a.block_table[static_cast<size_t>(b) * a.max_pages + entry];
        if (page >= a.num_pages) page = -1;
    }
    // Of head h: the first code, and the exponent.
    __device__ __forceinline__ size_t code(const RowsQ8Args& a, int h, int D) const {
        return ((static_cast<size_t>(page) * a.page_size + row) * a.Hkv + h) * D;
    }
    __device__ __forceinline__ size_t exponent(const RowsQ8Args& a, int h) const {
        return (static_cast<size_t>(page) * a.Hkv + h) * a.page_size + row;
    }
};

// The largest of v over groups of N (2 .. 16) neighbouring lanes.
template <int N>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
    auto with = [&](auto ctrl) {
        const uint32_t w = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
            0, static_cast<int>(v), decltype(ctrl)::value, 0xF, 0xF, false));
        v = v > w ? v : w;
    };
    with(std::integral_constant<int, kDppXor1>{});
    if constexpr (N >= 4) with(std::integral_constant<int, kDppXor2>{});
    if constexpr (N >= 8) with(std::integral_constant<int, kDppHalfMirror>{});
    if constexpr (N >= 16) with(std::integral_constant<int, kDppMirror>{});
    return v;
}

struct AppendQ8Args {
    RowsQ8Args rows;
    const float* rope_cos;
    const float* rope_sin;
    int H;  // 0: no queries
    int q_stride, k_stride, v_stride;
    int rotary, max_positions;
    int most;  // largest exponent
};

template <typename T, int D, QuantCode C, bool kInterleaved>
__global__ void __launch_bounds__(1024)
    append_q8_kernel(const typename Mma<T>::elem* Q, const typename Mma<T>::elem* K,
                     const typename Mma<T>::elem* V, typename Mma<T>::elem* Q_out,
                     uint8_t* K_cache, uint8_t* V_cache, uint8_t* K_exp, uint8_t* V_exp,
                     AppendQ8Args a) {
#pragma clang fp contract(off)
    using E = typename Mma<T>::elem;
    constexpr int VEC = 16 / static_cast<int>(sizeof(E));
    constexpr int UPR = D / (2 * VEC);  // units (pairs of chunks) per row
    const int t = blockIdx.x;
    const int Hkv = a.rows.Hkv;
    const int units = (a.H + 2 * Hkv) * UPR;
    const int turned = a.rotary / (2 * VEC);  // rotated units of a row

    // Unit u: a head's row of the token and its two chunks there, (w, w + rotary / 2) where the pairs
    // span the rotated part, else neighbours.
    int head, w, c0, c1;
    bool is_q, is_v, turn;
    u32x4 x0, x1;
    auto fetch = [&](int u) {
        const int row = u / UPR;
        w = u % UPR;
        is_q = row >= 2 * Hkv;
        is_v = !is_q && row >= Hkv;
        head = is_q ? row - 2 * Hkv : is_v ? row - Hkv : row;
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
    const TokenRow at(a.rows, t);
    if (at.padding) return;
    // Outside the rotation's tables a token has no angle.
    const bool angle = at.pos >= 0 && (a.rotary == 0 || at.pos < a.max_positions);
    const bool written = angle && at.page >= 0;

    for (; u < units; u += blockDim.x) {
        if (u != static_cast<int>(threadIdx.x)) fetch(u);
        if (!is_q && !written) continue;
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
        if (turn && angle) {
            const size_t from = static_cast<size_t>(at.pos) * (a.rotary / 2) + w * VEC;
            float c[VEC], s[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i += 4) {
                const f32x4 c4 = __builtin_bit_cast(f32x4, ld16(a.rope_cos + from + i));
                const f32x4 s4 = __builtin_bit_cast(f32x4, ld16(a.rope_sin + from + i));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    c[i + j] = c4[j];
                    s[i + j] = s4[j];
                }
            }
            // Pair i of the unit: elements (i, VEC + i) of x, or (2 i, 2 i + 1).
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                float& p = x[kInterleaved ? 2 * i : i];
                float& q = x[kInterleaved ? 2 * i + 1 : VEC + i];
                const float np = p * c[i] - q * s[i];
                q = q * c[i] + p * s[i];
                p = np;
            }
        }
        if (is_q) {
            E* dst = Q_out + (static_cast<size_t>(t) * a.H + head) * D;
            if (turn && !angle) {
                // NaN in every type.
                x0 = x1 = u32x4{0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu};
            } else if (turn) {
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
            continue;
        }
        // As bits magnitudes are in their order, infinities and NaN above all others.
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 2 * VEC; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
        m = group_max<UPR>(m);
        const bool number = m < 0x7f800000u;
        // ceil(log2(m / top)), for m and top with their fractions.
        int e = static_cast<int>(m - __builtin_bit_cast(uint32_t, Q8<C>::kTop) + 0x7fffffu) >> 23;
        e = min(max(e, -100), a.most);
        const float by = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);  // 2^-e
        uint32_t code[VEC / 2];
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                y[j] = fminf(fmaxf(x[4 * i + j] * by, -Q8<C>::kTop), Q8<C>::kTop);
            code[i] = number ? Q8<C>::pack4(y) : Q8<C>::kNone;
        }
        uint8_t* dst = (is_v ? V_cache : K_cache) + at.code(a.rows, head, D);
        if constexpr (VEC == 8) {
            st8(dst + c0, u32x2{code[0], code[1]});
            st8(dst + c1, u32x2{code[2], code[3]});
        } else {
            *reinterpret_cast<uint32_t*>(dst + c0) = code[0];
            *reinterpret_cast<uint32_t*>(dst + c1) = code[1];
        }
        if (w == 0)
            (is_v ? V_exp : K_exp)[at.exponent(a.rows, head)] =
                static_cast<uint8_t>(number ? e + 127 : 255);
    }
}

// A workgroup per token; a lane has 16 codes of one head's row, of keys or of values.
template <typename T, int D, QuantCode C>
__global__ void __launch_bounds__(1024)
    read_q8_kernel(const uint8_t* __restrict__ K_cache, const uint8_t* __restrict__ V_cache,
                   const uint8_t* __restrict__ K_exp, const uint8_t* __restrict__ V_exp,
                   typename Mma<T>::elem* __restrict__ K_out,
                   typename Mma<T>::elem* __restrict__ V_out, RowsQ8Args a) {
    using E = typename Mma<T>::elem;
    constexpr int UPR = D / 16;
    const int t = blockIdx.x;
    const TokenRow at(a, t);
    if (at.padding) return;
    for (int u = threadIdx.x; u < 2 * a.Hkv * UPR; u += blockDim.x) {
        const int row = u / UPR;
        const int c = (u % UPR) * 16;
        const bool is_v = row >= a.Hkv;
        const int head = is_v ? row - a.Hkv : row;
        E* dst = (is_v ? V_out : K_out) + (static_cast<size_t>(t) * a.Hkv + head) * D + c;
        u32x4 codes = {0u, 0u, 0u, 0u};
        uint32_t x = 255;  // every code is NaN
        if (at.page >= 0) {
            // Read once: 69620 keys of 8 heads, head_dim 128, to fp16 98.9 -> 81.3 us with the hint, 5.3 TB/s
            // (124 with one for the stores).
            codes = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(
                (is_v ? V_cache : K_cache) + at.code(a, head, D) + c));
            x = (is_v ? V_exp : K_exp)[at.exponent(a, head)];
        }
        const float f = Q8<C>::factor(x);
        if constexpr (std::is_same<T, float>::value) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x2 lo = Q8<C>::template expand_f32<0>(codes[i], f);
                const f32x2 hi = Q8<C>::template expand_f32<1>(codes[i], f);
                st16(dst + 4 * i, __builtin_bit_cast(u32x4, f32x4{lo[0], lo[1], hi[0], hi[1]}));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i += 2)
                st16(dst + 4 * i, u32x4{Q8<C>::template expand<T, 0>(codes[i], f),
                                        Q8<C>::template expand<T, 1>(codes[i], f),
                                        Q8<C>::template expand<T, 0>(codes[i + 1], f),
                                        Q8<C>::template expand<T, 1>(codes[i + 1], f)});
        }
    }
}

}  // namespace dev

namespace detail {
namespace {

// A launch has at most 2^32 - 1 threads in x.
bool too_many(int groups, int threads) {
    return static_cast<long long>(groups) * threads > 0xffffffffLL;
}

template <typename T, int D, QuantCode C>
FlashAttentionError run_append(const AppendQ8Call& call, hipStream_t stream) {
    using E = typename dev::Mma<T>::elem;
    const AppendCall& c = call.rows;
    dev::AppendQ8Args a{};
    a.rows = {c.block_table, c.seq_lens, c.query_starts, c.batch_size, c.num_kv_heads,
              c.num_pages, c.page_size, c.max_pages};
    a.rope_cos = c.rope_cos;
    a.rope_sin = c.rope_sin;
    a.H = c.Q ? c.num_heads : 0;
    a.q_stride = c.q_stride;
    a.k_stride = c.k_stride;
    a.v_stride = c.v_stride;
    a.rotary = c.rotary_dim;
    a.max_positions = c.max_positions;
    constexpr bool kE4m3 = C == QuantCode::E4M3;
    a.most = std::is_same<T, __half>::value ? (kE4m3 ? 7 : 9) : (kE4m3 ? 119 : 121);
    constexpr int kUnits = D * static_cast<int>(sizeof(E)) / 32;  // per row
    const long long units = (static_cast<long long>(a.H) + 2LL * c.num_kv_heads) * kUnits;
    const int threads = static_cast<int>(std::min(1024LL, (units + 63) / 64 * 64));
    if (too_many(c.num_tokens, threads)) return FlashAttentionError::INVALID_DIMENSION;
    ProfileEvents tok = profile_kernel<T, D>("append_q8");
    auto go = [&](auto kernel) {
        launch_kernel(tok, kernel, dim3(static_cast<unsigned>(c.num_tokens)),
                      dim3(static_cast<unsigned>(threads)), 0, stream,
                      static_cast<const E*>(c.Q), static_cast<const E*>(c.K),
                      static_cast<const E*>(c.V), static_cast<E*>(c.Q_out),
                      static_cast<uint8_t*>(c.K_cache), static_cast<uint8_t*>(c.V_cache),
                      call.K_exp, call.V_exp, a);
    };
    if (c.interleaved)
        go(dev::append_q8_kernel<T, D, C, true>);
    else
        go(dev::append_q8_kernel<T, D, C, false>);
    return from_hip(hipGetLastError());
}

template <typename T, int D, QuantCode C>
FlashAttentionError run_read(const ReadQ8Call& c, hipStream_t stream) {
    using E = typename dev::Mma<T>::elem;
    const dev::RowsQ8Args a{c.block_table,  c.seq_lens,  c.key_starts, c.batch_size,
                            c.num_kv_heads, c.num_pages, c.page_size,  c.max_pages};
    const long long units = 2LL * c.num_kv_heads * (D / 16);
    const int threads = static_cast<int>(std::min(1024LL, (units + 63) / 64 * 64));
    if (too_many(c.num_tokens, threads)) return FlashAttentionError::INVALID_DIMENSION;
    launch_kernel(profile_kernel<T, D>("read_q8"), dev::read_q8_kernel<T, D, C>,
                  dim3(static_cast<unsigned>(c.num_tokens)),
                  dim3(static_cast<unsigned>(threads)), 0, stream,
                  static_cast<const uint8_t*>(c.K_cache), static_cast<const uint8_t*>(c.V_cache),
                  c.K_exp, c.V_exp, static_cast<E*>(c.K_out), static_cast<E*>(c.V_out), a);
    return from_hip(hipGetLastError());
}

// run(D, C) for the call's head_dim and code.
template <class Run>
FlashAttentionError dispatch(int head_dim, QuantCode code, Run run) {
    auto with = [&](auto d) {
        return code == QuantCode::E4M3
                   ? run(d, std::integral_constant<QuantCode, QuantCode::E4M3>{})
                   : run(d, std::integral_constant<QuantCode, QuantCode::INT8>{});
    };
    switch (head_dim) {
        case 32:
            return with(std::integral_constant<int, 32>{});
        case 64:
            return with(std::integral_constant<int, 64>{});
        case 128:
            return with(std::integral_constant<int, 128>{});
    }
    return FlashAttentionError::UNSUPPORTED_HEAD_DIM;
}

}  // namespace

template <typename T>
FlashAttentionError launch_append_paged_q8(const AppendQ8Call& c, hipStream_t stream) {
    return dispatch(c.rows.head_dim, c.code, [&](auto d, auto code) {
        return run_append<T, decltype(d)::value, decltype(code)::value>(c, stream);
    });
}
template <typename T>
FlashAttentionError launch_read_paged_q8(const ReadQ8Call& c, hipStream_t stream) {
    return dispatch(c.head_dim, c.code, [&](auto d, auto code) {
        return run_read<T, decltype(d)::value, decltype(code)::value>(c, stream);
    });
}
#define CUFLASH_ROWS_Q8(T)                                                                  \
    template FlashAttentionError launch_append_paged_q8<T>(const AppendQ8Call&, hipStream_t); \
    template FlashAttentionError launch_read_paged_q8<T>(const ReadQ8Call&, hipStream_t);
CUFLASH_ROWS_Q8(float)
CUFLASH_ROWS_Q8(__half)
CUFLASH_ROWS_Q8(__hip_bfloat16)
#undef CUFLASH_ROWS_Q8

}  // namespace detail
}  // namespace cuflash
