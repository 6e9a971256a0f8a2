// Attention over an 8-bit paged cache for gfx950 (MI355X): flash_attention_decode_paged_q8 and
// flash_attention_forward_paged_q8 (cuflash/paged_cache_q8.h).
//
// attention_q8_kernel: a wave takes an equal share of all keys of all tiles of rows (paged_q8_plan.hpp),
// by itself: no LDS, no barrier. Tiles have 16 or 32 rows, the query heads of one key/value head over a few
// tokens, so that a key is read once for all of them. Blocks of 32 keys, in 16 x 16 x 32 products:
//   S^T = K Q^T   A: lane l has key l % 16 of a half block, of its codes the 16 bytes at 64 i + 16 (l / 16):
//                 two k-steps from one load; Q is laid out alike. C: lane l has row l % 16 and the keys
//                 4 (l / 16) + r of both halves, 8 in all.
//   O^T += V^T P^T  B: these 8 weights as they stand. A: the lane's same 8 keys, of each the D / 16
//                 neighbouring codes from D / 16 (l % 16) on, one load a key: tile j of the output has the
//                 columns D / 16 n + j, so a lane's codes of one key go to D / 16 tiles.
// Codes become 16-bit numbers in registers (q8.hpp) and stay exact; scores, maxima, sums and O are
// float, the weights are rounded to T before they meet V (half a step, 2^-8 of p |v| in bf16, as in the
// library's other matrix-core kernels), float ones taken apart into three bf16 numbers without a loss.
// Codes of the next block are asked for before this one is worked on. The waves of neighbouring key/value
// heads have the same share and so read the same cache rows at the same time.
// combine_q8_kernel (attention_q8.hpp) merges the rows that several waves have and writes those without a
// key. Where sequences have many 16-bit rows prompt_q8.hip takes over.

#include "attention_q8.hpp"

namespace cuflash {
namespace dev {

template <typename M>
__device__ __forceinline__ f32x4 mma16(typename Elem<M>::frag a, typename Elem<M>::frag b, f32x4 c) {
    if constexpr (std::is_same<M, __half>::value)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Over the lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float quad_max(float v) {
    v = pair_max(v);
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float quad_sum(float v) {
    v = pair_sum(v);
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// a and b, floats, as kParts pairs of 16-bit numbers whose sums they are: one, rounded, of type M, or three
// bf16 ones, each the upper half of what is left (8 of 24 bits, nothing is lost).
template <typename M, int kParts>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&to)[kParts]) {
    if constexpr (kParts == 1) {
        to[0] = Elem<M>::pack2(a, b);
    } else {
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            to[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
            a -= __uint_as_float(to[i] << 16);
            b -= __uint_as_float(to[i] & 0xffff0000u);
        }
    }
}

template <typename T, int D, QuantCode C, int NR, bool kWhole>
struct AttentionQ8 {
    using M = typename Q8Operand<T>::type;
    using E = typename Mma<T>::elem;
    using Frag = typename Elem<M>::frag;
    static constexpr int kParts = std::is_same<T, float>::value ? 3 : 1;
    static constexpr int R = 16 * NR;
    static constexpr int KS = D / 32;                 // k-steps of S
    static constexpr int KB = D >= 64 ? 16 : 8;       // bytes of a load of K codes
    static constexpr int KI = D / 4 / KB;             // such loads a key
    static constexpr int VB = D / 16;                 // bytes of a lane's V codes of a key
    static constexpr int VW = VB >= 4 ? VB / 4 : 1;   // in dwords
    static constexpr int VT = VB;                     // tiles of O

    const AttentionQ8Args& a;
    const E* Q;
    const uint8_t* K;  // of the key/value head
    const uint8_t* V;
    const uint8_t* Kx;
    const uint8_t* Vx;
    E* O;
    float* L;
    int hk;

    struct Codes {
        uint32_t k[2][KI][KB / 4];
        uint32_t v[8][VW];
        uint32_t kx[2];  // the exponent of the lane's key of each half block
        uint32_t vx[2];  // of its four keys
    };
    // The table entries of a block's halves (kWhole).
    typedef const __attribute__((address_space(4))) int* ConstInts;

    template <int N>
    static __device__ __forceinline__ void copy(uint32_t (&to)[N], const uint8_t* from, int bytes) {
        if constexpr (N == 4) {
            const u32x4 v = ld16(from);
            to[0] = v[0];
            to[1] = v[1];
            to[2] = v[2];
            to[3] = v[3];
        } else if constexpr (N == 2) {
            const u32x2 v = *reinterpret_cast<const u32x2*>(from);
            to[0] = v[0];
            to[1] = v[1];
        } else {
            to[0] = bytes == 2 ? *reinterpret_cast<const uint16_t*>(from)
                               : *reinterpret_cast<const uint32_t*>(from);
        }
    }

    // Entries of the table for the halves of the block at key0 of a segment that ends at kend.
    __device__ __forceinline__ void entries(const int* table, int key0, int kend, int (&page)[2]) const {
        const int last = (kend - 1) & ~15;
#pragma unroll
        for (int t = 0; t < 2; ++t)
            page[t] = ((ConstInts)table)[a.page_div(min(key0 + 16 * t, last))];
    }
    // The codes of the block at key0. Of a half that lies behind the end another's rows are read, and of
    // one that ends inside it the page's rows behind the end; neither is used.
    __device__ __forceinline__ void load(const int* table, const int (&page)[2], int key0, int kend,
                                         Codes& x) const {
        const int lane = threadIdx.x & 63;
        const int l16 = lane & 15, q = lane >> 4;
        const size_t pitch = static_cast<size_t>(a.Hkv) * D;
        if constexpr (kWhole) {
            const int last = (kend - 1) & ~15;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int at = min(key0 + 16 * t, last);
                const int in_page = at - a.page_div(at) * a.page_size;
                const size_t row = (static_cast<size_t>(page[t]) * a.page_size + in_page) * pitch;
                const size_t ex = static_cast<size_t>(page[t]) * a.Hkv * a.page_size + in_page;
                const uint32_t k_at = l16 * static_cast<uint32_t>(pitch) + q * KB;
#pragma unroll
                for (int i = 0; i < KI; ++i) copy(x.k[t][i], K + row + (k_at + 64u * i), KB);
                const uint32_t v_at = 4 * q * static_cast<uint32_t>(pitch) + l16 * VB;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    copy(x.v[4 * t + r], V + row + r * pitch + v_at, VB);
                x.kx[t] = *(Kx + ex + l16);
                x.vx[t] = *reinterpret_cast<const uint32_t*>(Vx + ex + 4 * q);
            }
        } else {
            auto place = [&](int key, size_t& row, size_t& ex) {
                key = min(key, kend - 1);
                const int entry = a.page_div(key);
                const int in_page = key - entry * a.page_size;
                const size_t pg = static_cast<size_t>(table[entry]);
                row = (pg * a.page_size + in_page) * pitch;
                ex = pg * a.Hkv * a.page_size + in_page;
            };
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                size_t row, ex;
                place(key0 + 16 * t + l16, row, ex);
#pragma unroll
                for (int i = 0; i < KI; ++i) copy(x.k[t][i], K + row + q * KB + 64 * i, KB);
                x.kx[t] = Kx[ex];
                x.vx[t] = 0;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    place(key0 + 16 * t + 4 * q + r, row, ex);
                    copy(x.v[4 * t + r], V + row + l16 * VB, VB);
                    x.vx[t] |= static_cast<uint32_t>(Vx[ex]) << (8 * r);
                }
            }
        }
    }

    // The outputs of a segment's rows, or their partial results, those of wave p.
    __device__ __forceinline__ void segment(const Q8Segment& g, const int* table, int p) const {
        const Q8Seq& s = g.seq;
        const int kbeg = g.kbeg, kend = g.kend;
        const int lane = threadIdx.x & 63;
        const int l16 = lane & 15, q = lane >> 4;
        Frag f[NR][kParts][KS];
        int lim[NR], orow[NR];
        int least = kend;
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            const int r = g.r0 + 16 * nr + l16;
            const bool on = r < g.rows;
            const int i = a.plan.group_div(on ? r : 0);
            orow[nr] = on ? (s.t0 + i) * a.H + hk * a.plan.group + (r - i * a.plan.group) : -1;
            lim[nr] = on ? min(kend, q8_limit(a.plan, s, i)) : kend;
            least = min(least, lim[nr]);
            const E* src = Q + static_cast<size_t>(on ? orow[nr] : 0) * D;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int at = D >= 64 ? 64 * (ks >> 1) + 16 * q + 8 * (ks & 1) : 8 * q;
                if constexpr (kParts == 1) {
                    u32x4 v = {0u, 0u, 0u, 0u};
                    if (on) v = ld16(src + at);
                    f[nr][0][ks] = as_frag<M>(v);
                } else {
                    u32x4 part[kParts];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
                        if (on) v = __builtin_bit_cast(f32x4, ld16(src + at + 4 * h));
#pragma unroll
                        for (int j = 0; j < 4; j += 2) {
                            uint32_t to[kParts];
                            split2<M, kParts>(v[j], v[j + 1], to);
                            // An infinity or a NaN is one number.
                            const bool odd0 = !(fabsf(v[j]) <= 3.402823466e38f),
                                       odd1 = !(fabsf(v[j + 1]) <= 3.402823466e38f);
                            if (odd0 || odd1) {
                                to[0] = Elem<M>::pack2(odd0 ? v[j] : 0.0f, odd1 ? v[j + 1] : 0.0f) |
                                        (odd0 ? 0u : to[0] & 0xffffu) |
                                        (odd1 ? 0u : to[0] & 0xffff0000u);
#pragma unroll
                                for (int k = 1; k < kParts; ++k)
                                    to[k] &= (odd0 ? 0u : 0xffffu) | (odd1 ? 0u : 0xffff0000u);
                            }
#pragma unroll
                            for (int k = 0; k < kParts; ++k) part[k][2 * h + j / 2] = to[k];
                        }
                    }
#pragma unroll
                    for (int k = 0; k < kParts; ++k) f[nr][k][ks] = as_frag<M>(part[k]);
                }
            }
        }
#pragma unroll
        for (int w = 8; w >= 1; w >>= 1) least = min(least, __shfl_xor(least, w, 64));
        const int mask_from = __builtin_amdgcn_readfirstlane(least);

        f32x4 o[NR][VT];
        float m[NR], l[NR];
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            m[nr] = -INFINITY;
            l[nr] = 0.0f;
#pragma unroll
            for (int j = 0; j < VT; ++j) o[nr][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        const float cs = fmaxf(a.c, kFltMin);  // scale 0: -inf * 0 would make the masked scores NaN

        auto block = [&](const Codes& x, int key0) {
            f32x4 sc[NR][2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) sc[nr][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                const float by = Q8<C>::factor(x.kx[t]);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const uint32_t* w = &x.k[t][ks / (KB / 8)][ks % (KB / 8) * 2];
                    const Frag k = as_frag<M>(u32x4{Q8<C>::template expand<M, 0>(w[0], by),
                                                    Q8<C>::template expand<M, 1>(w[0], by),
                                                    Q8<C>::template expand<M, 0>(w[1], by),
                                                    Q8<C>::template expand<M, 1>(w[1], by)});
#pragma unroll
                    for (int part = kParts - 1; part >= 0; --part) {
#pragma unroll
                        for (int nr = 0; nr < NR; ++nr)
                            sc[nr][t] = mma16<M>(k, f[nr][part][ks], sc[nr][t]);
                    }
                }
            }
            if (key0 + 32 > mask_from) {
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) {
                    const int n = lim[nr] - key0 - 4 * q;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            sc[nr][t][r] = 16 * t + r < n ? sc[nr][t][r] : -INFINITY;
                    }
                }
            }
            Frag pf[NR][kParts];
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                float mx = -INFINITY;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) mx = __builtin_elementwise_maximum(mx, sc[nr][t][r]);
                }
                const float m_new = fmaxf(m[nr], quad_max(mx) * cs);
                const bool grow = m_new > m[nr] + kLazyRescale;
                if (__ballot(grow) != 0) {
                    const float alpha =
                        grow ? fast_exp2(m_new == -INFINITY ? 0.0f : m[nr] - m_new) : 1.0f;
                    m[nr] = grow ? m_new : m[nr];
                    l[nr] *= alpha;
#pragma unroll
                    for (int j = 0; j < VT; ++j) o[nr][j] *= alpha;
                }
                const float m_use = m[nr] == -INFINITY ? 0.0f : m[nr];
                float sum = 0.0f;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        sc[nr][t][r] = fast_exp2(fmaf(sc[nr][t][r], cs, -m_use));
                        sum += sc[nr][t][r];
                    }
                }
                l[nr] += sum;
                u32x4 part[kParts];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t to[kParts];
                    split2<M, kParts>(sc[nr][i >> 1][2 * (i & 1)], sc[nr][i >> 1][2 * (i & 1) + 1], to);
#pragma unroll
                    for (int k = 0; k < kParts; ++k) part[k][i] = to[k];
                }
#pragma unroll
                for (int k = 0; k < kParts; ++k) pf[nr][k] = as_frag<M>(part[k]);
            }
            float by[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) by[e] = Q8<C>::factor((x.vx[e >> 2] >> (8 * (e & 3))) & 0xffu);
            // The codes of columns 2 j and 2 j + 1 of the lane's 8 keys: 8 pairs, turned.
            auto columns = [&](auto jc) {
                constexpr int j = decltype(jc)::value;
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    w[e] = Q8<C>::template expand<M, (j & 1)>(x.v[e][j >> 1], by[e]);
                u32x4 lo, hi;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    lo[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x05040100u);
                    hi[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x07060302u);
                }
#pragma unroll
                for (int part = kParts - 1; part >= 0; --part) {
#pragma unroll
                    for (int nr = 0; nr < NR; ++nr) {
                        o[nr][2 * j] = mma16<M>(as_frag<M>(lo), pf[nr][part], o[nr][2 * j]);
                        o[nr][2 * j + 1] = mma16<M>(as_frag<M>(hi), pf[nr][part], o[nr][2 * j + 1]);
                    }
                }
            };
            columns(std::integral_constant<int, 0>{});
            if constexpr (VT >= 4) columns(std::integral_constant<int, 1>{});
            if constexpr (VT >= 8) {
                columns(std::integral_constant<int, 2>{});
                columns(std::integral_constant<int, 3>{});
            }
        };
        // Values behind the end may be anything: 0, as 0 times an infinity or a NaN would be seen.
        auto cut = [&](Codes& x, int key0) {
            if (key0 + 32 <= kend) return;
            const int n = kend - key0 - 4 * q;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool in = 16 * (e >> 2) + (e & 3) < n;
#pragma unroll
                for (int i = 0; i < VW; ++i) x.v[e][i] = in ? x.v[e][i] : 0u;
                const uint32_t byte = 0xffu << (8 * (e & 3));
                x.vx[e >> 2] = in ? x.vx[e >> 2] : (x.vx[e >> 2] & ~byte) | (0x7f7f7f7fu & byte);
            }
        };

        Codes x[2];
        int page[2] = {0, 0};
        if constexpr (kWhole) entries(table, kbeg, kend, page);
        load(table, page, kbeg, kend, x[0]);
        if constexpr (kWhole) entries(table, kbeg + 32, kend, page);
        for (int key0 = kbeg; key0 < kend; key0 += 64) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = key0 + 32 * h;
                if (h == 1 && at >= kend) break;
                if (at + 32 < kend) {
                    load(table, page, at + 32, kend, x[1 - h]);
                    if constexpr (kWhole) entries(table, at + 64, kend, page);
                }
                cut(x[h], at);
                block(x[h], at);
            }
        }

#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            const float lt = quad_sum(l[nr]);
            if (orow[nr] < 0) continue;
            // Columns D / 4 q .. of the row, in order.
            if (g.slot >= 0) {
                const size_t to = q8_slot_row(a, p, g.slot, hk, 16 * nr + l16);
                float* dst = a.acc + to * D + q * (D / 4);
                store(dst, o[nr], 1.0f);
                if (q == 0) a.ml[to] = make_float2(m[nr], lt);
                continue;
            }
            const bool none = lt == 0.0f;  // no key, or every score -inf: O = 0, L = -inf
            if (none) {
#pragma unroll
                for (int j = 0; j < VT; ++j) o[nr][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
            store(O + static_cast<size_t>(orow[nr]) * D + q * (D / 4), o[nr],
                  none ? 0.0f : 1.0f / lt);
            if (q == 0) L[orow[nr]] = none ? -INFINITY : (m[nr] + fast_log2(lt)) * kLn2;
        }
    }

    // A lane's D / 4 columns: (4 q + r) VT + j.
    static __device__ __forceinline__ void store(float* dst, const f32x4 (&o)[VT], float by) {
#pragma unroll
        for (int i = 0; i < D / 4; i += 4) {
            f32x4 w;
#pragma unroll
            for (int u = 0; u < 4; ++u) w[u] = o[(i + u) % VT][(i + u) / VT] * by;
            st16(dst + i, __builtin_bit_cast(u32x4, w));
        }
    }
    static __device__ __forceinline__ void store(uint16_t* dst, const f32x4 (&o)[VT], float by) {
#pragma unroll
        for (int i = 0; i < D / 4; i += 8) {
            u32x4 w;
#pragma unroll
            for (int u = 0; u < 8; u += 2)
                w[u / 2] = Elem<M>::pack2(o[(i + u) % VT][(i + u) / VT] * by,
                                          o[(i + u + 1) % VT][(i + u + 1) / VT] * by);
            st16(dst + i, w);
        }
    }
};

constexpr int kQ8Waves = 4;  // of a workgroup: each for itself

template <typename T, int D, QuantCode C, int NR, bool kWhole>
__global__ void __launch_bounds__((64 * kQ8Waves), 2)
    attention_q8_kernel(const typename Mma<T>::elem* __restrict__ Q,
                        const uint8_t* __restrict__ K, const uint8_t* __restrict__ V,
                        const uint8_t* __restrict__ Kx, const uint8_t* __restrict__ Vx,
                        typename Mma<T>::elem* __restrict__ O, float* __restrict__ L,
                        AttentionQ8Args a) {
    constexpr int R = 16 * NR;
    const int wave = blockIdx.x * kQ8Waves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int p = wave / a.Hkv;
    const int hk = wave - p * a.Hkv;
    if (p >= a.plan.shares) return;
    Q8Walk<R, GpuWave> walk(a.plan, p);
    const AttentionQ8<T, D, C, NR, kWhole> work{
        a,
        Q,
        K + static_cast<size_t>(hk) * D,
        V + static_cast<size_t>(hk) * D,
        Kx + static_cast<size_t>(hk) * a.page_size,
        Vx + static_cast<size_t>(hk) * a.page_size,
        O,
        L,
        hk};
    Q8Segment s;
    while (walk.next(a.plan, s))
        work.segment(s, a.block_table + static_cast<size_t>(s.b) * a.max_pages, p);
}

}  // namespace dev

namespace detail {
namespace {

// Where most sequences have more rows than this, workgroups share the keys (prompt_q8.hip).
constexpr long long kManyRows = 96;
template <typename T>
bool many_rows(const PagedCall& c) {
    return !std::is_same<T, float>::value && c.query_starts &&
           static_cast<long long>(c.num_tokens) * (c.num_heads / c.num_kv_heads) >
               kManyRows * c.batch_size;
}

// Tiles of 16 rows, or of 32 where sequences have more and registers suffice (float queries of 128 elements
// in three parts are too many). Two waves a SIMD (registers); with 32 rows a little fewer, whose partial
// results then fit the library's workspace of a stream.
template <typename T>
Q8Grid waves_grid(const PagedCall& c) {
    const bool wide = (!std::is_same<T, float>::value || c.head_dim < 128) &&
                      static_cast<long long>(c.num_tokens) * (c.num_heads / c.num_kv_heads) >
                          16LL * c.batch_size;
    const int waves = compute_units() * 8;
    return Q8Grid(c, wide ? 32 : 16, (wide ? waves / 16 * 15 : waves) / c.num_kv_heads, 0);
}

template <typename T, int D, QuantCode C>
FlashAttentionError run_attention(const PagedQ8Call& q8, hipStream_t stream) {
    using E = typename dev::Mma<T>::elem;
    const PagedCall& c = q8.call;
    if (many_rows<T>(c)) {
        if constexpr (!std::is_same<T, float>::value) return launch_prompt_q8<T>(q8, stream);
    }
    const Q8Grid grid = waves_grid<T>(c);
    const bool whole = c.page_size % 16 == 0;  // half a block's rows lie on one page
    auto run = [&](auto nr) {
        constexpr int NR = decltype(nr)::value;
        return run_q8<T, D, 16 * NR>(c, grid, stream, [&](const dev::AttentionQ8Args& a) {
            const long long waves = static_cast<long long>(grid.shares) * grid.kv_heads;
            auto go = [&](auto kernel) {
                launch_kernel(profile_kernel<T, D>(c.query_starts ? "forward_q8" : "decode_q8"),
                              kernel,
                              dim3(static_cast<unsigned>((waves + dev::kQ8Waves - 1) /
                                                         dev::kQ8Waves)),
                              dim3(64 * dev::kQ8Waves), 0, stream, static_cast<const E*>(c.Q),
                              static_cast<const uint8_t*>(c.K_cache),
                              static_cast<const uint8_t*>(c.V_cache), q8.K_exp, q8.V_exp,
                              static_cast<E*>(c.O), c.L, a);
            };
            if (whole)
                go(dev::attention_q8_kernel<T, D, C, NR, true>);
            else
                go(dev::attention_q8_kernel<T, D, C, NR, false>);
        });
    };
    if constexpr (!std::is_same<T, float>::value || D < 128) {
        if (grid.rows == 32) return run(std::integral_constant<int, 2>{});
    }
    return run(std::integral_constant<int, 1>{});
}

template <typename T, QuantCode C>
FlashAttentionError run_dim(const PagedQ8Call& c, hipStream_t stream) {
    switch (c.call.head_dim) {
        case 32:
            return run_attention<T, 32, C>(c, stream);
        case 64:
            return run_attention<T, 64, C>(c, stream);
        case 128:
            return run_attention<T, 128, C>(c, stream);
    }
    return FlashAttentionError::UNSUPPORTED_HEAD_DIM;
}

}  // namespace

template <typename T>
long long paged_q8_workspace(const PagedCall& c) {
    auto grid = [&] {
        if constexpr (!std::is_same<T, float>::value) {
            if (many_rows<T>(c)) return prompt_q8_grid<T>(c);
        }
        return waves_grid<T>(c);
    }();
    return static_cast<long long>(grid.bytes());
}

template <typename T>
FlashAttentionError launch_paged_q8(const PagedQ8Call& c, hipStream_t stream) {
    return c.code == QuantCode::E4M3 ? run_dim<T, QuantCode::E4M3>(c, stream)
                                     : run_dim<T, QuantCode::INT8>(c, stream);
}
#define CUFLASH_PAGED_Q8(T)                                     \
    template long long paged_q8_workspace<T>(const PagedCall&); \
    template FlashAttentionError launch_paged_q8<T>(const PagedQ8Call&, hipStream_t);
CUFLASH_PAGED_Q8(float)
CUFLASH_PAGED_Q8(__half)
CUFLASH_PAGED_Q8(__hip_bfloat16)
#undef CUFLASH_PAGED_Q8

}  // namespace detail
}  // namespace cuflash
