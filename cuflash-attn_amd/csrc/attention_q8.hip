// Attention over an 8-bit paged cache for gfx950 (MI355X): flash_attention_decode_paged_q8 and
// flash_attention_forward_paged_q8 (cuflash/paged_cache_q8.h).
//
// attention_q8_kernel: a wave takes an equal share of all keys of all tiles of rows (paged_q8_plan.hpp),
// by itself, without a barrier: keys and values go from memory to registers, and LDS only turns results into
// whole rows. Tiles have 16 or 32 rows, the query heads of one key/value head over a few tokens, so that a key
// is read once for all of them. Blocks of 32 keys, in 16 x 16 x 32 products:
//   S^T = K Q^T   A: lane l has key l % 16 of a half block, of its codes the 16 bytes at 64 i + 16 (l / 16):
//                 two k-steps from one load; Q is laid out alike. C: lane l has row l % 16 and the keys
//                 4 (l / 16) + r of both halves, 8 in all.
//   O^T += V^T P^T  B: these 8 weights as they stand. A: the lane's same 8 keys, of each the D / 16
//                 neighbouring codes from D / 16 (l % 16) on, one load a key: tile j of the output has the
//                 columns D / 16 n + j, so a lane's codes of one key go to D / 16 tiles.
// Codes become 16-bit numbers in registers (q8.hpp) and stay exact; scores, maxima, sums and O are
// float, the weights are rounded to T before they meet V (half a step, 2^-8 of p |v| in bf16, as in the
// library's other matrix-core kernels), float ones taken apart into three bf16 numbers without a loss.
// Codes of the next block are asked for before this one is worked on, or where registers are short as
// its own have been used. The waves of neighbouring key/value heads have the same share and so read the same
// cache rows at the same time.
// combine_q8_kernel or merge_q8_kernel (attention_q8.hpp) merges the rows that several waves have and writes those
// without a key; from short tables all is one launch, attention_q8_short_kernel. Where sequences have many 16-bit
// rows prompt_q8.hip takes over.
// Bound by HBM (32 heads over 8, head_dim 128; a 1 GiB copy reaches 5.1 TB/s): 4 sequences of up to 131072 keys, bf16
// over e4m3, 167 us, 6.5 TB/s; 64 of up to 8192 keys, fp16 over int8, 94 us, 5.9, float over int8 102 us, 5.4; 16 x 5
// tokens of 8196 keys, fp16 over e4m3, 54 us, 5.0. float prompts by the conversions and three bf16 products for one:
// 4096 tokens over int8 712 us, 193 TFLOP/s.
// Every wave sums the sequences' sizes to find its share, 64 in a step: 1024 sequences of 1100 keys 384 us where 64 of
// 17600 take 374, 16384 sequences of one 8-head group, head_dim 64, 591 where 256 with as many keys take 432.

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

template <typename T, int D, QuantCode C, int NR, int kPage>
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
    static constexpr int kPitch = D + 4;              // floats from row to row in LDS

    const AttentionQ8Args& a;
    const E* Q;
    const uint8_t* K;  // of the key/value head
    const uint8_t* V;
    const uint8_t* Kx;
    const uint8_t* Vx;
    E* O;
    float* L;
    int hk;

    // e4m3 codes are scaled as they are converted; for int8 codes that would be an instruction an element, so
    // their scores are scaled instead.
    static constexpr bool kScaleK = C == QuantCode::E4M3;
    // The rows that surely lie on one page, from a multiple of their number on: of a page of 16 n rows those of
    // half a block, found by one walk; of one of 4 n rows a lane's four keys.
    static constexpr bool kWhole = kPage == 16, kFours = kPage >= 4;
    static constexpr int XW = kFours ? 2 : 8;
    struct Codes {
        uint32_t k[2][KI][KB / 4];
        uint32_t v[8][VW];
        // The exponents of the lane's four keys of each half block, in one word or (!kFours) in one each;
        // kScaleK: of its one key of each half.
        uint32_t kx[kScaleK ? 2 : XW];
        uint32_t vx[XW];
    };
    typedef const __attribute__((address_space(4))) int* ConstInts;
    // Two blocks in registers, or one, whose keys and then values give way to the next as they have been used.
    static constexpr bool kDouble = NR == 1 && kParts == 1;

    template <int N>
    static __device__ __forceinline__ void copy(uint32_t (&to)[N], const uint8_t* from, int bytes) {
        if constexpr (N == 4) {
            const u32x4 v = ld16(from);
#pragma unroll
            for (int i = 0; i < 4; ++i) to[i] = v[i];
        } else if constexpr (N == 2) {
            const u32x2 v = *reinterpret_cast<const u32x2*>(from);
            to[0] = v[0];
            to[1] = v[1];
        } else {
            to[0] = bytes == 2 ? *reinterpret_cast<const uint16_t*>(from)
                               : *reinterpret_cast<const uint32_t*>(from);
        }
    }
    // The same for lines that one load reads whole and, where a sequence has one tile of rows, nothing reads again (64
    // sequences of up to 8192 keys, int8: 111 -> 99 us; K, half a line a load, so 100 -> 123). Measured in decodes: what
    // the hint does where several tiles of rows read the same values is not known.
    template <int N>
    static __device__ __forceinline__ void copy_once(uint32_t (&to)[N], const uint8_t* from, int bytes) {
        if constexpr (N == 2) {
            const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(from));
            to[0] = v[0];
            to[1] = v[1];
        } else {
            copy(to, from, bytes);
        }
    }

    // The place of the half block that is loaded next (kWhole: its rows lie on one page): the walk over a
    // segment's halves, the table read one ahead. Behind the last it stays there.
    struct Place {
        const int* table;
        int entry, in_page;  // of the next half
        int page;
        int left;  // halves behind it
    };
    __device__ __forceinline__ Place place_of(const int* table, int kbeg, int kend) const {
        Place at;
        at.table = table;
        at.entry = a.page_div(kbeg);
        at.in_page = kbeg - at.entry * a.page_size;
        at.page = ((ConstInts)table)[at.entry];
        at.left = (kend - kbeg - 1) >> 4;
        return at;
    }
    __device__ __forceinline__ void advance(Place& at) const {
        if (at.left == 0) return;
        --at.left;
        at.in_page += 16;
        if (at.in_page >= a.page_size) {
            at.in_page = 0;
            ++at.entry;
            at.page = ((ConstInts)at.table)[at.entry];
        }
    }

    // base + offset as a load from a scalar base and a 32-bit lane offset: seen as a constant of the loop the
    // offset would be widened in front of it, to two registers and an addition a load.
    static __device__ __forceinline__ const uint8_t* lane_at(const uint8_t* base, uint32_t offset) {
        asm volatile("" : "+v"(offset));
        return base + offset;
    }

    // Where the halves of a block lie (kWhole): their first row, in bytes, and its exponent.
    struct Rows {
        uint64_t row[2], ex[2];
        int key0;
    };
    __device__ __forceinline__ Rows rows_of(Place& next, int key0) const {
        Rows at;
        at.key0 = key0;
        if constexpr (kWhole) {
            const uint32_t pitch = static_cast<uint32_t>(a.Hkv) * D;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint64_t pg = static_cast<uint32_t>(next.page);
                at.row[t] = pg * a.page_bytes + static_cast<uint64_t>(next.in_page) * pitch;
                at.ex[t] = pg * a.page_exps + next.in_page;
                advance(next);
            }
        }
        return at;
    }
    // The same of one key, that of a lane.
    __device__ __forceinline__ void row_of(const int* table, int key, uint64_t& row, uint64_t& ex) const {
        const int entry = a.page_div(key);
        const uint32_t in_page = key - entry * a.page_size;
        const uint64_t pg = static_cast<uint32_t>(table[entry]);
        row = pg * a.page_bytes + static_cast<uint64_t>(in_page) * (static_cast<uint32_t>(a.Hkv) * D);
        ex = pg * a.page_exps + in_page;
    }
    // The codes of a block. Of a half that lies behind the end another's rows are read, and of one that ends
    // inside it the page's rows behind the end; neither is used.
    __device__ __forceinline__ void load_k(const Rows& at, const int* table, int kend, Codes& x) const {
        const int lane = threadIdx.x & 63;
        const int l16 = lane & 15, q = lane >> 4;
        const uint32_t pitch = static_cast<uint32_t>(a.Hkv) * D;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if constexpr (kWhole) {
#pragma unroll
                for (int i = 0; i < KI; ++i)
                    copy(x.k[t][i], lane_at(K + at.row[t] + 64 * i, l16 * pitch + q * KB), KB);
                x.kx[t] = kScaleK
                              ? *lane_at(Kx + at.ex[t], l16)
                              : *reinterpret_cast<const uint32_t*>(lane_at(Kx + at.ex[t], 4 * q));
            } else {
                uint64_t row, ex;
                row_of(table, min(at.key0 + 16 * t + l16, kend - 1), row, ex);
#pragma unroll
                for (int i = 0; i < KI; ++i) copy(x.k[t][i], K + row + (q * KB + 64 * i), KB);
                if constexpr (kScaleK)
                    x.kx[t] = Kx[ex];
                else
                    load_x(at.key0 + 16 * t + 4 * q, table, kend, Kx, &x.kx[XW / 2 * t]);
            }
        }
    }
    // The exponents of keys key .. key + 3, where half a block is no walk.
    __device__ __forceinline__ void load_x(int key, const int* table, int kend, const uint8_t* exps,
                                           uint32_t* x) const {
        uint64_t row, ex;
        if constexpr (kFours) {
            row_of(table, min(key, (kend - 1) & ~3), row, ex);
            *x = *reinterpret_cast<const uint32_t*>(exps + ex);
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                row_of(table, min(key + r, kend - 1), row, ex);
                x[r] = exps[ex];
            }
        }
    }
    __device__ __forceinline__ void load_v(const Rows& at, const int* table, int kend, Codes& x) const {
        const int lane = threadIdx.x & 63;
        const int l16 = lane & 15, q = lane >> 4;
        const uint32_t pitch = static_cast<uint32_t>(a.Hkv) * D;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if constexpr (kWhole) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    copy_once(x.v[4 * t + r],
                              lane_at(V + at.row[t] + static_cast<uint64_t>(r) * pitch,
                                      4 * q * pitch + l16 * VB),
                              VB);
                x.vx[t] = *reinterpret_cast<const uint32_t*>(lane_at(Vx + at.ex[t], 4 * q));
            } else {
                const int key = at.key0 + 16 * t + 4 * q;
                uint64_t row, ex;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (!kFours)
                        row_of(table, min(key + r, kend - 1), row, ex);
                    else if (r == 0)
                        row_of(table, min(key, (kend - 1) & ~3), row, ex);
                    copy(x.v[4 * t + r],
                         V + row + (static_cast<uint64_t>(kFours ? r : 0) * pitch + l16 * VB), VB);
                }
                load_x(key, table, kend, Vx, &x.vx[XW / 2 * t]);
            }
        }
    }
    // Of key e of the lane's eight.
    static __device__ __forceinline__ float factor(const uint32_t (&x)[XW], int e) {
        return Q8<C>::factor(kFours ? (x[e >> 2] >> (8 * (e & 3))) & 0xffu : x[e]);
    }
    // Of int8 keys, whether one of the lane's has an exponent that leads beyond fp16's numbers: 137 or more (127 *
    // 2^10 is infinite there) or less than 103 (2^-25 is none of them). Such a block's codes become fp16 numbers
    // before the product, as in prompt_q8.hip and the read: which kernel a call takes does not show. (The look costs
    // up to 4%: 16 x 5 tokens of 8196 keys, head_dim 64, 30.4 -> 31.6 us; 64 sequences of 4000 keys, head_dim 64, 34.0
    // -> 34.8, head_dim 128 93.3 -> 94.1.)
    static __device__ __forceinline__ bool beyond_half(const uint32_t (&x)[XW]) {
        uint32_t high = 0u, low = ~0u;  // in a byte's top bit: one is 137 or more, all are 103 or more
#pragma unroll
        for (int i = 0; i < XW; ++i) {
            const uint32_t w7 = x[i] & 0x7f7f7f7fu;
            high |= (w7 + 0x77777777u) & x[i];
            low &= (w7 + 0x19191919u) | x[i];
        }
        return ((high | ~low) & (kFours ? 0x80808080u : 0x80u)) != 0u;
    }
    // Of key l % 16 of half t: lanes 16 (key / 4) .. + 15 have it as one of their four.
    static __device__ __forceinline__ float key_factor(const uint32_t (&x)[XW], int t) {
        const int key = threadIdx.x & 15;
        float f = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float of = __shfl(factor(x, 4 * t + r), key >> 2 << 4, 64);
            f = (key & 3) == r ? of : f;
        }
        return f;
    }

    // The outputs of a segment's rows, or (slot >= 0) their partial results, those of row r of the tile D floats
    // at acc_of(r) and (m, l) at ml_of(r). `stage`: 16 rows of the wave's in LDS; kKeep: R rows, and the partial
    // results stay there.
    template <bool kKeep, class Acc, class Ml>
    __device__ __forceinline__ void segment(const Q8Segment& g, const int* table, float* stage,
                                            Acc acc_of, Ml ml_of) const {
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

        f32x4 sc[NR][2];
        // Half t's scores, its codes scaled by `by` on their way or (kScaled false) as they are.
        auto half = [&](const Codes& x, int t, auto scaled, float by) {
            constexpr bool kScaled = decltype(scaled)::value;
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) sc[nr][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const uint32_t* w = &x.k[t][ks / (KB / 8)][ks % (KB / 8) * 2];
                const u32x2 lo = Q8<C>::template four<M, kScaled>(w[0], by);
                const u32x2 hi = Q8<C>::template four<M, kScaled>(w[1], by);
                const Frag k = as_frag<M>(u32x4{lo[0], lo[1], hi[0], hi[1]});
#pragma unroll
                for (int part = kParts - 1; part >= 0; --part) {
#pragma unroll
                    for (int nr = 0; nr < NR; ++nr)
                        sc[nr][t] = mma16<M>(k, f[nr][part][ks], sc[nr][t]);
                }
            }
        };
        auto scores = [&](const Codes& x) {
            if constexpr (kScaleK) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    half(x, t, std::integral_constant<bool, true>{}, Q8<C>::factor(x.kx[t]));
            } else {
                bool beyond = false;
                if constexpr (std::is_same<M, __half>::value) beyond = __ballot(beyond_half(x.kx)) != 0;
                if (__builtin_expect(beyond, false)) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        half(x, t, std::integral_constant<bool, true>{}, key_factor(x.kx, t));
                } else {
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        half(x, t, std::integral_constant<bool, false>{}, 1.0f);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float by = factor(x.kx, 4 * t + r);
#pragma unroll
                            for (int nr = 0; nr < NR; ++nr) sc[nr][t][r] *= by;
                        }
                    }
                }
            }
        };
        auto values = [&](const Codes& x, int key0) {
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
            for (int e = 0; e < 8; ++e) by[e] = factor(x.vx, e);
            // The codes of columns 2 j and 2 j + 1 of the lane's 8 keys: 8 pairs, turned.
            auto columns = [&](auto jc) {
                constexpr int j = decltype(jc)::value;
                u32x4 lo, hi;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const u32x2 two = Q8<C>::template turned<M, (j & 1)>(
                        x.v[2 * i][j >> 1], by[2 * i], x.v[2 * i + 1][j >> 1], by[2 * i + 1]);
                    lo[i] = two[0];
                    hi[i] = two[1];
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
                const uint32_t byte = kFours ? 0xffu << (8 * (e & 3)) : 0xffu;
                uint32_t& exps = x.vx[kFours ? e >> 2 : e];
                exps = in ? exps : (exps & ~byte) | (0x7f7f7f7fu & byte);
            }
        };

        Place next = place_of(table, kbeg, kend);
        int key0 = kbeg;
        Codes last;
        if constexpr (kDouble) {
            Codes x[2];
            auto load = [&](int at, Codes& to) {
                const Rows rows = rows_of(next, at);
                load_k(rows, table, kend, to);
                load_v(rows, table, kend, to);
            };
            load(kbeg, x[0]);
            while (key0 + 32 < kend) {
                load(key0 + 32, x[1]);
                scores(x[0]);
                values(x[0], key0);
                key0 += 32;
                if (key0 + 32 >= kend) {
                    x[0] = x[1];
                    break;
                }
                load(key0 + 32, x[0]);
                scores(x[1]);
                values(x[1], key0);
                key0 += 32;
            }
            last = x[0];
        } else {
            const Rows first = rows_of(next, kbeg);
            load_k(first, table, kend, last);
            load_v(first, table, kend, last);
            while (key0 + 32 < kend) {
                scores(last);
                const Rows rows = rows_of(next, key0 + 32);
                load_k(rows, table, kend, last);
                values(last, key0);
                load_v(rows, table, kend, last);
                key0 += 32;
            }
        }
        cut(last, key0);
        scores(last);
        values(last, key0);

        // Rows leave through LDS, so that a store writes whole ones: from a lane's D / 4 columns it would write 16
        // bytes of each of 64 lines (16 x 5 tokens of 8196 keys 57.4 -> 52.7 us).
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            const float lt = quad_sum(l[nr]);
            const bool none = lt == 0.0f;  // no key, or every score -inf: O = 0, L = -inf
            const bool part = kKeep || g.slot >= 0;
            const float by = part ? 1.0f : none ? 0.0f : 1.0f / lt;
            float* rows = stage + (kKeep ? 16 * nr * kPitch : 0);
            // Columns (4 q + r) VT + j of the lane's row, in order.
#pragma unroll
            for (int i = 0; i < D / 4; i += 4) {
                f32x4 w;
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    w[u] = none && !part ? 0.0f : o[nr][(i + u) % VT][(i + u) / VT] * by;
                st16(rows + l16 * kPitch + q * (D / 4) + i, __builtin_bit_cast(u32x4, w));
            }
            if (part) {
                if (q == 0 && orow[nr] >= 0) *ml_of(16 * nr + l16) = make_float2(m[nr], lt);
            } else if (q == 0 && orow[nr] >= 0) {
                L[orow[nr]] = none ? -INFINITY : (m[nr] + fast_log2(lt)) * kLn2;
            }
            if constexpr (kKeep) continue;
            asm volatile("" ::: "memory");  // a wave's LDS accesses are performed in order
            constexpr int VEC = 16 / static_cast<int>(sizeof(E));
            if (part) {
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const int r = (64 * i + lane) / (D / 4), c = (64 * i + lane) % (D / 4) * 4;
                    if (g.r0 + 16 * nr + r < g.rows)
                        st16(acc_of(16 * nr + r) + c, ld16(rows + r * kPitch + c));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16 * (D / VEC) / 64; ++i) {
                    const int r = (64 * i + lane) / (D / VEC), c = (64 * i + lane) % (D / VEC) * VEC;
                    const int to = __shfl(orow[nr], r, 64);
                    if (to < 0) continue;
                    const f32x4 x = __builtin_bit_cast(f32x4, ld16(rows + r * kPitch + c));
                    u32x4 w;
                    if constexpr (VEC == 4) {
                        w = __builtin_bit_cast(u32x4, x);
                    } else {
                        const f32x4 y = __builtin_bit_cast(f32x4, ld16(rows + r * kPitch + c + 4));
                        w = u32x4{Elem<M>::pack2(x[0], x[1]), Elem<M>::pack2(x[2], x[3]),
                                  Elem<M>::pack2(y[0], y[1]), Elem<M>::pack2(y[2], y[3])};
                    }
                    st16(O + static_cast<size_t>(to) * D + c, w);
                }
            }
            asm volatile("" ::: "memory");
        }
    }
};

// Of a workgroup, each for itself: the eight key/value heads of a common model then read their shares of the
// cache's rows from one CU.
constexpr int kQ8Waves = 8;

template <typename T, int D, QuantCode C, int NR, int kPage>
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
    using Work = AttentionQ8<T, D, C, NR, kPage>;
    __shared__ __attribute__((aligned(16))) float s_rows[kQ8Waves][16 * Work::kPitch];
    Q8Walk<R, GpuWave> walk(a.plan, p);
    const Work work{
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
    while (walk.next(a.plan, s)) {
        auto row = [&](int r) { return q8_slot_row(a, p, s.slot, hk, r); };
        work.template segment<false>(
            s, a.block_table + static_cast<size_t>(s.b) * a.max_pages,
            s_rows[__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)],
            [&](int r) { return a.acc + row(r) * D; }, [&](int r) { return a.ml + row(r); });
    }
}

// Attention from short tables in one launch: a workgroup has a tile, each wave a piece of its keys, and their parts
// are merged through LDS.
template <typename T, int D, QuantCode C, int NR, int kPage>
__global__ void __launch_bounds__((64 * kQ8Waves), 2)
    attention_q8_short_kernel(const typename Mma<T>::elem* __restrict__ Q,
                              const uint8_t* __restrict__ K, const uint8_t* __restrict__ V,
                              const uint8_t* __restrict__ Kx, const uint8_t* __restrict__ Vx,
                              typename Mma<T>::elem* __restrict__ O, float* __restrict__ L,
                              AttentionQ8Args a, uint32_t items) {
    constexpr int R = 16 * NR;
    using Work = AttentionQ8<T, D, C, NR, kPage>;
    __shared__ __attribute__((aligned(16))) float s_acc[kQ8Waves][R][Work::kPitch];
    __shared__ float2 s_ml[kQ8Waves][R];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int x = item / a.Hkv;
        const int hk = item - x * a.Hkv;
        int b, tile;
        if (!q8_tile_at<R, GpuWave>(a.plan, x, b, tile)) return;
        const Work work{
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
        s.seq = q8_seq(a.plan, b);
        s.b = b;
        const Q8Line<R> line(a.plan, s.seq);
        const int keys = line.keys(a.plan, s.seq, tile);
        s.rows = line.rows;
        s.r0 = tile * R;
        s.slot = 0;
        const int blocks = (keys + 31) / 32;
        const int each = (blocks + kQ8Waves - 1) / kQ8Waves * 32;
        s.kbeg = wave * each;
        s.kend = min(s.kbeg + each, keys);
        if (s.kbeg < s.kend) {
            work.template segment<true>(
                s, a.block_table + static_cast<size_t>(b) * a.max_pages, s_acc[wave][0],
                [&](int r) { return s_acc[wave][r]; }, [&](int r) { return &s_ml[wave][r]; });
        } else if (lane < R) {
            s_ml[wave][lane] = make_float2(-INFINITY, 0.0f);
        }
        __syncthreads();
        constexpr int LPR = D / 4;
        const int part = threadIdx.x % LPR;
        for (int r = threadIdx.x / LPR; r < min(R, s.rows - s.r0); r += 64 * kQ8Waves / LPR) {
            float2 v[kQ8Waves];
            f32x4 x[kQ8Waves];
#pragma unroll
            for (int w = 0; w < kQ8Waves; ++w) {
                v[w] = s_ml[w][r];
                x[w] = __builtin_bit_cast(f32x4, ld16(&s_acc[w][r][4 * part]));
            }
            Q8Merge sum;
            sum.add(v, x);
            const int token = a.plan.group_div(s.r0 + r);
            const size_t row = static_cast<size_t>(s.seq.t0 + token) * a.H + hk * a.plan.group +
                               (s.r0 + r - token * a.plan.group);
            sum.store<T>(O + row * D + 4 * part, L + row, part == 0);
        }
        __syncthreads();  // before the next item's parts
    }
}

}  // namespace dev

namespace detail {
namespace {

// Where sequences have more rows than this, 16-bit ones, workgroups share the keys (prompt_q8.hip): on average 48 a
// sequence, 96 at head_dim 64 and 32, 16 for a single sequence, whose waves would have few blocks each and leave as
// many partial results (bf16 over e4m3, us of kernels by waves and by workgroups; head_dim 128, 32 heads over 8: 16
// sequences of 4000 keys, 32 rows each 41 and 61, 48 rows 63 and 66, 64 rows 80 and 67; one of 8000 keys, 32 rows 29
// and 20; head_dim 64 over 4, 16 of 4000 keys: 96 rows 33 and 36, 128 rows 41 and 38).
template <typename T>
bool many_rows(const PagedCall& c) {
    const long long most = c.batch_size == 1 ? 16 : c.head_dim == 128 ? 48 : 96;
    return !std::is_same<T, float>::value && c.query_starts &&
           static_cast<long long>(c.num_tokens) * (c.num_heads / c.num_kv_heads) >
               most * c.batch_size;
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
    return Q8Grid(c, wide ? 32 : 16, (wide ? waves / 16 * 15 : waves) / c.num_kv_heads, 0,
                  1);
}

// Whether a call is one launch, a workgroup a tile of rows. Decodes are, from tables of at most 1024 keys (bf16 over
// e4m3, 32 heads over 8, head_dim 128, us of kernels in one and in two: one sequence of 500 keys 6.7 and 11.5, of 1000
// 9.8 and 12.1, of 2000 15.9 and 12.0; 64 of up to 500 13.5 and 17.4, of up to 1000 23.2 and 24.1, of up to 2000 37.7
// and 33.0). Of several tokens, where the workgroups' rounds are few for their keys and the rest of the chip would not
// be of much use: the same heads, 4 tokens of 200 keys 6.5 and 13.2, 250 of 1000 13.1 and 40.9, 500 of 1000 23 and 44,
// 250 of 2000 20 and 44, 500 of 2000 35 and 52, 128 of 4000 32 and 39; against that 2000 of 2000 101 and 66, 32 of 4000
// 32 and 23, 128 of 8000 57 and 47, 256 sequences with 2 tokens of 60 keys 40 and 22; fp32, 8 heads over 4, head_dim 64,
// 1000 of 1000 14.5 and 31.7, 2000 of 2000 35 and 43, 32 of 2000 23 and 18, 250 of 4000 38 and 31.
bool one_launch(const PagedCall& c, const Q8Grid& grid) {
    const long long keys = static_cast<long long>(c.page_size) * c.max_pages;
    if (!c.query_starts) return keys <= 1024;
    const long long items = dev::q8_most_tiles(grid.args(c).plan, grid.rows) * c.num_kv_heads;
    const long long rounds = (items + compute_units() - 1) / compute_units();
    return rounds * (keys + 700) <= 5500 && (keys <= 1024 || items * 32 >= keys);
}

template <typename T>
long long workspace_of(const PagedCall& c) {
    auto grid = [&] {
        if constexpr (!std::is_same<T, float>::value) {
            if (many_rows<T>(c)) return prompt_q8_grid<T>(c);
        }
        return waves_grid<T>(c);
    }();
    return static_cast<long long>(grid.bytes());
}

template <typename T, int D, QuantCode C>
FlashAttentionError run_attention(const PagedQ8Call& q8, hipStream_t stream) {
    using E = typename dev::Mma<T>::elem;
    const PagedCall& c = q8.call;
    const Q8Grid grid = waves_grid<T>(c);
    const bool one = one_launch(c, grid);
    // A forward's workspace is asked for by its sizes, whether keys are cut or not.
    if (one && c.query_starts) {
        const FlashAttentionError err = workspace_refusal(c, workspace_of<T>(c), stream);
        if (err != FlashAttentionError::SUCCESS) return err;
    }
    if (!one && many_rows<T>(c)) {
        if constexpr (!std::is_same<T, float>::value) return launch_prompt_q8<T>(q8, stream);
    }
    // go(n) with n rows that lie on one page.
    auto by_page = [&](auto go) {
        if (c.page_size % 16 == 0)
            go(std::integral_constant<int, 16>{});
        else if (c.page_size % 4 == 0)
            go(std::integral_constant<int, 4>{});
        else
            go(std::integral_constant<int, 1>{});
    };
    if (one) {
        auto run = [&](auto nr) {
            constexpr int NR = decltype(nr)::value;
            const dev::AttentionQ8Args a = grid.args(c);
            // At most B H of them, below 2^31. A launch has at most 2^32 - 1 threads in x; workgroups take several
            // items beyond.
            const long long items = dev::q8_most_tiles(a.plan, grid.rows) * c.num_kv_heads;
            const long long groups = std::min<long long>(1 << 22, items);
            auto go = [&](auto kernel) {
                launch_kernel(profile_kernel<T, D>("attention_q8_short"), kernel,
                              dim3(static_cast<unsigned>(groups)), dim3(64 * dev::kQ8Waves), 0,
                              stream, static_cast<const E*>(c.Q),
                              static_cast<const uint8_t*>(c.K_cache),
                              static_cast<const uint8_t*>(c.V_cache), q8.K_exp, q8.V_exp,
                              static_cast<E*>(c.O), c.L, a, static_cast<uint32_t>(items));
            };
            by_page([&](auto page) {
                go(dev::attention_q8_short_kernel<T, D, C, NR, decltype(page)::value>);
            });
            return from_hip(hipGetLastError());
        };
        if constexpr (!std::is_same<T, float>::value || D < 128) {
            if (grid.rows == 32) return run(std::integral_constant<int, 2>{});
        }
        return run(std::integral_constant<int, 1>{});
    }
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
            by_page([&](auto page) {
                go(dev::attention_q8_kernel<T, D, C, NR, decltype(page)::value>);
            });
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
    return workspace_of<T>(c);
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
