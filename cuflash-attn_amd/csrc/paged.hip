// Attention of packed tokens over a paged cache for gfx950 (MI355X): flash_attention_forward_paged
// and flash_attention_decode_shared (cuflash/paged_cache.h). One launch of paged_kernel, cut by
// paged_plan.hpp, and where keys are cut into chunks a launch of paged_combine_kernel.
//
// The query heads of one key/value head are packed into the rows of a tile (row r of a unit is token
// r / group, head r % group), so its keys are read once for all of them. A wave holds 32 rows in the
// forward kernels' transposed tiles: S^T = K Q^T, a lane pair per row, the online softmax in the
// score registers, O^T += V^T P^T (kv_block32). The two kinds of items:
//  * many rows: each wave has 32 rows of its own, and all of them share the key tiles;
//  * few rows: 32 rows in all, each wave takes other 32-key blocks through tiles of its own, and the
//    waves' (O, m, l) are merged through LDS at the end. This is what keeps enough bytes in flight
//    where a sequence's keys are read for a handful of rows.
// Tiles are filled by LDS-DMA loads, one kilobyte of whole key rows each: where the rows of a load
// cannot cross a page, from a scalar base (the page index by a scalar load) and a fixed lane offset;
// otherwise, and in a sequence's last tile, from an address per lane. Rows past the end are the last
// key again, and masked.
//
// P is rounded to the inputs' type before P V, as in the forward kernels (at most half a step of it per
// value: 2^-8 of p |v| in bf16), as the 16-bit matrix instructions take no wider operand; scores,
// maxima, sums and O are fp32. Against 64-bit results bf16 outputs are off by 0.0023 of their size so, and by
// 0.0017 with P in fp32 (fp16 0.00029 and 0.00021).
//
// Bound by MFMA where a sequence has many rows (one prompt of 16384 tokens, 32 heads
// over 8, head_dim 128, bf16: 1.85 to 1.96 ms a call, 1120 to 1191 TFLOP/s), at head_dim 64 by the softmax
// beside it (seven prompts of 285 to 2001 tokens 97 to 102 us a call, 736 to 770 TFLOP/s), by HBM where it
// has few (16 x 5 tokens of up to 8196 keys: 60 us a call, the first kernel 57 us, 5.05 TB/s).

#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "kv_block.hpp"
#include "launch.hpp"
#include "paged_launch.hpp"
#include "paged_plan.hpp"
#include "profile.hpp"
#include "softmax.hpp"
#include "tile_groups.hpp"
#include "wave.hpp"

namespace cuflash {
namespace dev {

// LDS-DMA load from a scalar base (lds_dma16_async_s) with the non-temporal hint. As there, one wait state is
// enough because base and LDS address are SALU values: pages come by scalar loads here, where the decode's
// come from a lane (lds_dma16_nt_s, five). tests/test_code_hazards.py checks the built code.
__device__ __forceinline__ void lds_dma16_once_s(const void* sbase, unsigned voff,
                                                 unsigned char* lds_base) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt"
                 :
                 : "v"(voff), "s"(sbase),
                   "{m0}"(__builtin_amdgcn_readfirstlane(lds_address(lds_base)))
                 : "memory");
}

// What differs between the types: tiles of 32 keys in LDS and the block over one of them.
template <typename T_, int D_, int NW>
struct PagedEngine {
    using T = T_;
    static constexpr int D = D_;
    using Lay = TileGroups<D>;
    using Frag = typename Elem<T>::frag;
    static constexpr int kWaves = NW;
    static constexpr int kPerCu = D <= 64 || NW <= 4 ? 2 : 1;  // workgroups (LDS)
    static constexpr int kRoundCost = 2;
    // Rows from which on waves have rows of their own. A few-rows item loads its keys for 32 rows: 4 x 61
    // tokens of 8253 keys, 32 heads over 8, 244 rows a sequence, take 52 us so, and 79 as eight of these.
    static constexpr int kManyRows = 96;
    static constexpr bool kInTurn = NW == 8;
    static constexpr int kStepBlocks = 2;              // 32-key blocks of a step (many rows)
    static constexpr int kGroupRows = Lay::kRows;      // key rows of one load
    static constexpr int kGroups = 32 / kGroupRows;    // loads of a tile
    static constexpr int kGroupBytes = Lay::kBytes;
    static constexpr int kTile = kGroups * kGroupBytes;
    struct Query {
        Frag f[D / 16];
    };
    __device__ __forceinline__ static void load(Query& q, const uint16_t* row, bool on, int g2) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            u32x4 v = {0u, 0u, 0u, 0u};
            if (on) v = ld16(row + 16 * ks + 8 * g2);
            q.f[ks] = as_frag<T>(v);
        }
    }
    __device__ __forceinline__ static int ld_row(int lane) { return Lay::ld_row(lane); }
    __device__ __forceinline__ static int ld_col(int lane, int) { return Lay::ld_col(lane); }
    struct Offsets {
        int k[2], v;
    };
    __device__ __forceinline__ static Offsets offsets(int lane) {
        return {{Lay::row_base(lane, 0), Lay::row_base(lane, 1)}, Lay::tr_off(lane)};
    }
    template <class F>
    __device__ __forceinline__ static void block(const unsigned char* kt, const unsigned char* vt,
                                                 const Offsets& at, int key0, int mask_from,
                                                 int kend, int g2, float cs, const Query& q,
                                                 f32x16 (&o)[D / 32], float& m, float& l,
                                                 F&& before_pv) {
        kv_block32<T, D, Lay>(kt, vt, at.k, at.v, key0, mask_from, kend, g2, cs, q.f, o, m, l,
                              before_pv);
    }
};

// fp32 on v_mfma_f32_32x32x2f32. Key row r of a tile starts at 4 D r, its 16-byte chunk c at slot
// c ^ (r & kSwizzle): 16 rows read at one chunk fall into 16 bank slots (8 at head_dim 32). Lane
// half h supplies chunk 2 j + h of both K and Q to the four products of step j: any assignment of
// the k index does, as long as both agree. The scores and P stay in fp32.
template <int D_, int NW>
struct PagedEngine<float, D_, NW> {
    using T = float;
    static constexpr int D = D_;
    static constexpr int kWaves = NW;
    static constexpr int kPerCu = D <= 64 ? 2 : 1;
    static constexpr int kRoundCost = 1;
    // Few-rows items only: the products take so long that a wave's own loads hide behind them, and tiles of
    // 32 rows spread better (700 tokens, 16 heads over 4, head_dim 128: 69 -> 53 us).
    static constexpr int kManyRows = 0x7fffffff;
    static constexpr bool kInTurn = false;
    static constexpr int kStepBlocks = 1;
    static constexpr int kGroupRows = 256 / D;
    static constexpr int kGroups = 32 / kGroupRows;
    static constexpr int kGroupBytes = 1024;
    static constexpr int kTile = kGroups * kGroupBytes;
    static constexpr int kSwizzle = D >= 64 ? 15 : 7;
    struct Query {
        f32x4 f[D / 8];
    };
    __device__ __forceinline__ static void load(Query& q, const float* row, bool on, int g2) {
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
            u32x4 v = {0u, 0u, 0u, 0u};
            if (on) v = ld16(row + 8 * j + 4 * g2);
            q.f[j] = __builtin_bit_cast(f32x4, v);
        }
    }
    __device__ __forceinline__ static int ld_row(int lane) { return lane / (D / 4); }
    __device__ __forceinline__ static int ld_col(int lane, int g) {
        const int r = kGroupRows * g + ld_row(lane);
        return ((lane % (D / 4)) ^ (r & kSwizzle)) * 4;
    }
    struct Offsets {
        int k;     // K row l32
        int k_x;   // its swizzle
        int v[4];  // V row 4 g2 + i, this lane's column of dims 0 .. 31
    };
    __device__ __forceinline__ static Offsets offsets(int lane) {
        const int l32 = lane & 31, g2 = lane >> 5;
        Offsets o;
        o.k = l32 * 4 * D;
        o.k_x = l32 & kSwizzle;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            o.v[i] = (4 * g2 + i) * 4 * D + (((l32 >> 2) ^ (4 * g2 + i)) * 16) + (l32 & 3) * 4;
        return o;
    }
    template <class F>
    __device__ __forceinline__ static void block(const unsigned char* kt, const unsigned char* vt,
                                                 const Offsets& at, int key0, int mask_from,
                                                 int kend, int g2, float cs, const Query& q,
                                                 f32x16 (&o)[D / 32], float& m, float& l,
                                                 F&& before_pv) {
        f32x16 s = f32x16{};
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
            const f32x4 k = __builtin_bit_cast(
                f32x4, ld16(kt + at.k + (((2 * j + g2) ^ at.k_x) * 16)));
#pragma unroll
            for (int i = 0; i < 4; ++i) s = mma_f32(k[i], q.f[j][i], s);
        }
        if (key0 + 32 > mask_from) {
            const int lim = kend - key0 - 4 * g2;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = (8 * (r >> 2) + (r & 3) < lim) ? s[r] : -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = __builtin_elementwise_maximum(mx, s[r]);
        const float m_new = fmaxf(m, pair_max(mx) * cs);
        const bool grow = m_new > m + kLazyRescale;
        const float alpha = grow ? fast_exp2(m_new == -INFINITY ? 0.0f : m - m_new) : 1.0f;
        m = grow ? m_new : m;
        l *= alpha;
        if (__ballot(grow) != 0) {
#pragma unroll
            for (int dt = 0; dt < D / 32; ++dt) o[dt] *= alpha;
        }
        const float m_use = (m == -INFINITY) ? 0.0f : m;
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = fast_exp2(fmaf(s[r], cs, -m_use));
            sum += s[r];
        }
        l += sum;
        before_pv();
        // Score register r holds key 8 (r / 4) + 4 g2 + r % 4: bit 3 of its swizzle swaps
        // neighbouring 32-column tiles (head_dim 64 and 128).
#pragma unroll
        for (int r = 0; r < 16; ++r) {
#pragma unroll
            for (int dt = 0; dt < D / 32; ++dt) {
                const int tile = D >= 64 ? dt ^ ((r >> 2) & 1) : dt;
                const float v = *reinterpret_cast<const float*>(
                    vt + at.v[r & 3] + (r >> 2) * 8 * 4 * D + tile * 128);
                o[dt] = mma_f32(v, s[r], o[dt]);
            }
        }
    }
};

template <class Eng>
using PagedShapeOf =
    PagedShape<32 * Eng::kWaves, 32 * Eng::kStepBlocks, 32 * Eng::kWaves, Eng::kRoundCost,
               Eng::kManyRows>;

// The rows of one key/value head in the cache, from their position in a sequence.
template <typename E>
struct CacheRows {
    // Uniform reads go through the scalar cache: the table does not change during the launch.
    typedef const __attribute__((address_space(4))) int* ConstInts;
    const int* table;
    FastDiv page_div;
    int page_size;
    size_t pitch;  // elements from key to key
    __device__ __forceinline__ int entry(int j) const { return ((ConstInts)table)[j]; }
    __device__ __forceinline__ int page(int t) const { return entry(page_div(t)); }
    __device__ __forceinline__ size_t from_page(int t, int page) const {
        return (static_cast<size_t>(page) * page_size + (t - page_div(t) * page_size)) * pitch;
    }
    __device__ __forceinline__ size_t uniform(int t) const { return from_page(t, page(t)); }
    __device__ __forceinline__ size_t lane(int t) const {
        return from_page(t, table[page_div(t)]);
    }
};

template <class Eng>
struct PagedWork {
    using T = typename Eng::T;
    static constexpr int D = Eng::D;
    using E = typename Mma<T>::elem;
    const E* Q;
    const E* K;  // of the item's key/value head
    const E* V;
    E* O;
    float* L;
    const PagedArgs& a;
    const PagedItem& it;
    int hk;
    CacheRows<E> rows;
    bool whole;  // a load's rows lie on one page

    // Row r of the unit in Q, O and L.
    __device__ __forceinline__ int out_row(int r) const {
        const int i = a.group_div(r);
        return (it.unit.t0 + i) * a.H + hk * a.group + (r - i * a.group);
    }
    // Keys below this are seen by row r of the unit, within the item.
    __device__ __forceinline__ int row_end(int r) const {
        return min(it.kend, paged_limit(a, it.u, it.unit, a.group_div(r)));
    }
    // Group g of the tile that begins at key0, from K and V alike.
    // kOnce: no other workgroup reads these keys, so they should not displace other lines (16 x 5 tokens
    // of up to 8196 keys 63.6 -> 56.0 us; keys that several workgroups share, 61 tokens of 8253, 26.5
    // -> 32.6).
    template <int N, bool kOnce = false>
    __device__ __forceinline__ void load_groups(const E* src, int key0, int tile_end, int g0,
                                                int step, unsigned char* dst) const {
        const int lane = threadIdx.x & 63;
        const int ld_row = Eng::ld_row(lane);
        if (whole && tile_end <= it.kend) {
            const int row = ld_row * static_cast<int>(rows.pitch);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int g = g0 + step * i;
                const E* base = src + rows.uniform(key0 + Eng::kGroupRows * g);
                const unsigned voff =
                    static_cast<unsigned>((row + Eng::ld_col(lane, g)) * sizeof(E));
                if constexpr (kOnce)
                    lds_dma16_once_s(base, voff, dst + g * Eng::kGroupBytes);
                else
                    lds_dma16_async_s(base, voff, dst + g * Eng::kGroupBytes);
            }
        } else {
            size_t off[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int t = key0 + Eng::kGroupRows * (g0 + step * i) + ld_row;
                off[i] = rows.lane(min(t, it.kend - 1));
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int g = g0 + step * i;
                lds_dma16_async(src + off[i] + Eng::ld_col(lane, g), dst + g * Eng::kGroupBytes);
            }
        }
    }
    // One row's result: its 16-byte piece cc of D, from the unnormalized sums.
    __device__ __forceinline__ static u32x4 finish(const float* x, float inv) {
        u32x4 w;
        if constexpr (std::is_same<T, float>::value) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(x[i] * inv);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = Elem<T>::pack2(x[2 * i] * inv, x[2 * i + 1] * inv);
        }
        return w;
    }

    __device__ __forceinline__ void many_rows(unsigned char* smem) const;
    __device__ __forceinline__ void many_rows_in_turn(unsigned char* smem) const;
    __device__ __forceinline__ void store_many(unsigned char* smem, const f32x16 (&o)[D / 32],
                                               float m, float l, bool on, int orow) const;
    __device__ __forceinline__ void few_rows(unsigned char* smem, float (*s_m)[32],
                                             float (*s_l)[32]) const;
};

// The outputs or partial results of a wave's rows, from its accumulators.
template <class Eng>
__device__ __forceinline__ void PagedWork<Eng>::store_many(unsigned char* smem,
                                                           const f32x16 (&o)[D / 32], float m,
                                                           float l, bool on, int orow) const {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31;
    const int g2 = lane >> 5;
    l = pair_sum(l);
    if (!it.direct) {
        if (!on) return;
        const size_t slot =
            paged_slot_row<PagedShapeOf<Eng>>(a, hk, true, it.slot, wave * 32 + l32);
        float* dst = a.acc + slot * D + 4 * g2;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f32x4 w;
#pragma unroll
                for (int u = 0; u < 4; ++u) w[u] = o[dt][4 * i + u];
                st16(dst + 32 * dt + 8 * i, __builtin_bit_cast(u32x4, w));
            }
        }
        if (g2 == 0) a.ml[slot] = make_float2(m, l);
        return;
    }
    // O rows through LDS, so that a store writes whole rows: 16 bytes a lane.
    constexpr int P = D * static_cast<int>(sizeof(E)) + 16;
    constexpr int kChunks = D * static_cast<int>(sizeof(E)) / 16;  // per row
    static_assert(32 * P <= 2 * Eng::kTile, "the O rows fit the tiles");
    __syncthreads();  // every wave is past its last tile
    unsigned char* stage = smem + wave * 32 * P;
    const bool none = l == 0.0f;  // no key, or every score -inf: O = 0, L = -inf
    const float inv = none ? 0.0f : 1.0f / l;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = none ? 0.0f : o[dt][4 * i + u] * inv;
            unsigned char* dst = stage + l32 * P + (32 * dt + 8 * i + 4 * g2) * sizeof(E);
            if constexpr (std::is_same<T, float>::value) {
                st16(dst, u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]),
                                __float_as_uint(x[2]), __float_as_uint(x[3])});
            } else {
                st8(dst, u32x2{Elem<T>::pack2(x[0], x[1]), Elem<T>::pack2(x[2], x[3])});
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 32 * kChunks / 64; ++i) {
        const int r = (64 * i + lane) / kChunks;
        const int cc = (64 * i + lane) % kChunks;
        const int to = __shfl(orow, r, 64);
        const u32x4 v = ld16(stage + r * P + cc * 16);
        if (to >= 0)
            st16(reinterpret_cast<unsigned char*>(O) + static_cast<size_t>(to) * (D * sizeof(E)) +
                     cc * 16,
                 v);
    }
    if (g2 == 0 && on) L[orow] = none ? -INFINITY : (m + fast_log2(l)) * kLn2;
}

template <class Eng>
__device__ __forceinline__ void PagedWork<Eng>::many_rows(unsigned char* smem) const {
    constexpr int kBlocks = Eng::kStepBlocks;
    constexpr int kStep = 32 * kBlocks;
    constexpr int kBytes = kBlocks * Eng::kTile;  // of a step's K or V
    constexpr int kParts = kBlocks * Eng::kGroups / Eng::kWaves;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31;
    const int g2 = lane >> 5;
    const int row = it.r0 + wave * 32 + l32;
    const bool on = row < it.rows;
    const int orow = on ? out_row(row) : -1;

    typename Eng::Query q;
    Eng::load(q, Q + static_cast<size_t>(on ? orow : 0) * D, on, g2);
    // This lane's keys, and the least and the greatest end of the wave's rows.
    const int kend = on ? row_end(row) : it.kend;
    int least = kend, most = on ? kend : 0;
#pragma unroll
    for (int w = 16; w >= 1; w >>= 1) {
        least = min(least, __shfl_xor(least, w, 64));
        most = max(most, __shfl_xor(most, w, 64));
    }
    const int mask_from = __builtin_amdgcn_readfirstlane(least);
    const int wave_end = __builtin_amdgcn_readfirstlane(most);
    const int nsteps = it.kend > it.kbeg ? (it.kend - it.kbeg + kStep - 1) / kStep : 0;

    unsigned char* const k0 = smem;
    unsigned char* const v0 = smem + kBytes;
    unsigned char* const k1 = smem + 2 * kBytes;
    unsigned char* const v1 = smem + 3 * kBytes;
    auto load = [&](int j, unsigned char* kt, unsigned char* vt) {
        const int key0 = it.kbeg + j * kStep;
        load_groups<kParts>(K, key0, key0 + kStep, wave, Eng::kWaves, kt);
        load_groups<kParts>(V, key0, key0 + kStep, wave, Eng::kWaves, vt);
    };
    const auto lds_at = Eng::offsets(lane);
    f32x16 o[D / 32];
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) o[dt] = f32x16{};
    float m = -INFINITY, l = 0.0f;
    const float cs = fmaxf(a.c, kFltMin);  // scale 0: -inf * 0 would make the masked scores NaN
    auto step = [&](int j, const unsigned char* kt, const unsigned char* vt) {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            const int key0 = it.kbeg + j * kStep + 32 * b;
            if (key0 < wave_end)
                Eng::block(kt + b * Eng::kTile, vt + b * Eng::kTile, lds_at, key0, mask_from, kend, g2,
                           cs, q, o, m, l, [] {});
        }
    };
    // Step j in buffers j & 1: the loads of step j + 1 are issued behind the barrier that ends every
    // wave's reads of step j - 1.
    if (nsteps > 0) load(0, k0, v0);
    for (int j = 0; j < nsteps; j += 2) {
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (j + 1 < nsteps) load(j + 1, k1, v1);
        step(j, k0, v0);
        if (j + 1 >= nsteps) break;
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (j + 2 < nsteps) load(j + 2, k0, v0);
        step(j + 1, k1, v1);
    }

    store_many(smem, o, m, l, on, orow);
}

// The same with the two waves of a SIMD in turn on the matrix and the vector unit. Left to themselves
// they form scores at the same time and then their softmax, so that each unit waits for the other. Here
// waves 4 to 7 (waves 0 to 3 sit on the same SIMDs) start half a step late, and a barrier after each half
// holds them there:
//   half 2 j:      waves 0-3  softmax of S_j                                  waves 4-7  products of step j
//   half 2 j + 1:  waves 0-3  O += V_j^T P_j, S_{j+1} = K_{j+1} Q^T           waves 4-7  softmax of S_j
// K and V tiles rotate through three buffers each. Products j + 1 read V_j and K_{j+1}, in the halves
// 2 j + 1 and 2 j + 2. A wave issues its share of later tiles before its softmax of S_j: waves 0-3 in half
// 2 j, of V_{j+1} and K_{j+2}, whose buffers were last read in half 2 j - 2 (V_{j-2}, K_{j-1}); waves 4-7 in
// half 2 j + 1, one step further, V_{j+2} and K_{j+3}, last read in half 2 j (V_{j-1}, K_j). Behind its next
// softmax it waits until these have landed: half 2 j + 2 or 2 j + 3, before the half that reads them, 2 j + 3
// or 2 j + 5. (8192 tokens of 32 heads over 8, head_dim 64: 870 TFLOP/s, MFMA 33 to 59% busy and the VALU 50
// to 61% over these shapes.)
template <class Eng>
__device__ __forceinline__ void PagedWork<Eng>::many_rows_in_turn(unsigned char* smem) const {
    using Lay = typename Eng::Lay;
    using Frag = typename Eng::Frag;
    constexpr int NW = Eng::kWaves;
    constexpr int kStep = 64;
    constexpr int kBytes = 2 * Eng::kTile;             // of a step's K or V
    constexpr int kParts = 2 * Eng::kGroups / NW;      // loads of a wave per tile
    constexpr int KS = D / 16;
    constexpr int NDT = D / 32;
    constexpr int kMma = 4 * NDT;                      // MFMAs of either product per step
    static_assert(NW == 8 && Eng::kStepBlocks == 2 && 6 * kBytes <= 2 * NW * Eng::kTile, "shape");
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31;
    const int g2 = lane >> 5;
    const int row = it.r0 + wave * 32 + l32;
    const bool on = row < it.rows;
    const int orow = on ? out_row(row) : -1;

    typename Eng::Query q;
    Eng::load(q, Q + static_cast<size_t>(on ? orow : 0) * D, on, g2);
    const int kend = on ? row_end(row) : it.kend;
    int least = kend, most = on ? kend : 0;
#pragma unroll
    for (int w = 16; w >= 1; w >>= 1) {
        least = min(least, __shfl_xor(least, w, 64));
        most = max(most, __shfl_xor(most, w, 64));
    }
    const int mask_from = __builtin_amdgcn_readfirstlane(least);
    const int wave_end = __builtin_amdgcn_readfirstlane(most);
    const int n = it.kend > it.kbeg ? (it.kend - it.kbeg + kStep - 1) / kStep : 0;
    // Steps in which this wave has keys to see.
    const int nw = min(n, wave_end > it.kbeg ? (wave_end - it.kbeg + kStep - 1) / kStep : 0);

    const int k_base[2] = {Lay::row_base(lane, 0), Lay::row_base(lane, 1)};
    const int v_base = Lay::tr_off(lane);
    f32x16 o[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[dt] = f32x16{};
    f32x16 s[2];
    s[0] = s[1] = f32x16{};
    Frag p[4];
    float m = -INFINITY, l = 0.0f;
    const float cs = fmaxf(a.c, kFltMin);  // scale 0: -inf * 0 would make the masked scores NaN

    // A wave's share of a whole tile is kParts neighbouring groups of rows on one page: one scalar base,
    // found by walking the page table a step ahead of K, and V_j comes from where K_j came a step before.
    // (Scalar instructions take their time, 8 cycles where they depend on each other: with a base and a
    // division for each load, the four loads took 950 cycles of each half's 2400; the loads themselves
    // want to be few per half, too. Between the MFMAs they cost as much and delay these.)
    constexpr int kShare = Eng::kGroupRows * kParts;  // rows
    const bool shares_whole = whole && rows.page_size % kShare == 0 && it.kbeg % kShare == 0;
    const int whole_tiles = shares_whole ? (it.kend - it.kbeg) / kStep : 0;
    const unsigned row_bytes = static_cast<unsigned>(rows.pitch * sizeof(E));
    const uint64_t page_bytes = static_cast<uint64_t>(row_bytes) * rows.page_size;
    unsigned voff[kParts];
#pragma unroll
    for (int i = 0; i < kParts; ++i)
        voff[i] = (Eng::ld_row(lane) + Eng::kGroupRows * i) * row_bytes +
                  static_cast<unsigned>(Eng::ld_col(lane, 0) * sizeof(E));
    // Place of this wave's share of the next tile to ask for: entry of the page table, row of the page.
    const int first_key = it.kbeg + kShare * wave;
    int entry = rows.page_div(first_key);
    int in_page = first_key - entry * rows.page_size;
    const int last_entry = rows.page_div(max(first_key, first_key + (whole_tiles - 1) * kStep));
    const int step_pages = rows.page_div(kStep);
    const int step_rows = kStep - step_pages * rows.page_size;
    int page = 0, page_row = 0;  // of the tile asked for
    uint64_t at = 0;             // place of the last whole K tile, in bytes
    auto ask = [&] {
        page = rows.entry(min(entry, last_entry));  // behind the last whole tile: any
        page_row = in_page;
        entry += step_pages;
        in_page += step_rows;
        if (in_page >= rows.page_size) {
            in_page -= rows.page_size;
            ++entry;
        }
    };
    auto place = [&] {
        at = static_cast<uint64_t>(static_cast<unsigned>(page)) * page_bytes +
             static_cast<uint64_t>(static_cast<unsigned>(page_row)) * row_bytes;
    };
    const unsigned lds0 = __builtin_amdgcn_readfirstlane(lds_address(smem)) +
                          static_cast<unsigned>(wave * kParts * Eng::kGroupBytes);
    // lds_dma16_async_s with the LDS address as a number.
    auto load_whole = [&](const E* src, int buffer) {
#pragma unroll
        for (int i = 0; i < kParts; ++i)
            asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                         :
                         : "v"(voff[i]), "s"(reinterpret_cast<const char*>(src) + at),
                           "{m0}"(lds0 + buffer + Eng::kGroupBytes * i)
                         : "memory");
    };
    auto load = [&](const E* src, int j, int buffer) {
        if (j < whole_tiles) {
            load_whole(src, buffer);
        } else {
            const int key0 = it.kbeg + j * kStep;
            load_groups<kParts>(src, key0, key0 + kStep, wave * kParts, 1, smem + buffer);
        }
    };
    auto v_frag = [&](const unsigned char* vt, int i) {
        const unsigned char* at = vt + v_base + (i / NDT) * Lay::kTrRows16 + Lay::dtile_off(i % NDT);
        return tr_frag_at<T>(at, at + Lay::kTrHigh);
    };
    auto k_frag = [&](const unsigned char* kt, int i) {
        return as_frag<T>(
            ld16(kt + k_base[(i % KS) & 1] + (i / KS) * Eng::kTile + Lay::k_off(i % KS)));
    };
    constexpr int kAhead = 4;  // MFMAs ahead of which an operand is read
    auto scores = [&](const unsigned char* kt) {
        Frag f[kMma];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) f[i] = k_frag(kt, i);
#pragma unroll
        for (int i = 0; i < kMma; ++i) {
            if (i + kAhead < kMma) f[i + kAhead] = k_frag(kt, i + kAhead);
            s[i / KS] = Elem<T>::mma(f[i], q.f[i % KS], s[i / KS]);
        }
    };
    // O += V^T P, then the next scores, in one chain. (Behind the last step these come from an old
    // tile and are not used.)
    auto products = [&](const unsigned char* vt, const unsigned char* kt) {
        Frag f[2 * kMma];
        auto frag_of = [&](int i) { return i < kMma ? v_frag(vt, i) : k_frag(kt, i - kMma); };
#pragma unroll
        for (int i = 0; i < kAhead; ++i) f[i] = frag_of(i);
#pragma unroll
        for (int i = 0; i < 2 * kMma; ++i) {
            if (i + kAhead < 2 * kMma) f[i + kAhead] = frag_of(i + kAhead);
            if (i < kMma) {
                o[i % NDT] = Elem<T>::mma(f[i], p[i / NDT], o[i % NDT]);
            } else {
                const int k = i - kMma;
                if (k == 0) s[0] = s[1] = f32x16{};
                s[k / KS] = Elem<T>::mma(f[i], q.f[k % KS], s[k / KS]);
            }
        }
    };
    // The softmax of S_j: masks, the lazily raised maximum, P_j rounded to T, the row sum in fp32.
    auto softmax = [&](int j) {
        const int key0 = it.kbeg + j * kStep;
        if (key0 + kStep > mask_from) {
            const int lim = kend - key0 - 4 * g2;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[t][r] = 32 * t + 8 * (r >> 2) + (r & 3) < lim ? s[t][r] : -INFINITY;
            }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int r = 0; r < 16; r += 2)
                mx = __builtin_elementwise_maximum(__builtin_elementwise_maximum(mx, s[t][r]),
                                                   s[t][r + 1]);
        }
        const float m_new = fmaxf(m, pair_max(mx) * cs);
        const bool grow = m_new > m + kLazyRescale;
        if (__ballot(grow) != 0) {
            const float alpha = grow ? fast_exp2(m_new == -INFINITY ? 0.0f : m - m_new) : 1.0f;
            m = grow ? m_new : m;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) o[dt] *= alpha;
        }
        const float m_use = (m == -INFINITY) ? 0.0f : m;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f32x16& x = s[i >> 1];
            const int r0 = 8 * (i & 1);
#pragma unroll
            for (int r = r0; r < r0 + 8; ++r) x[r] = fast_exp2(fmaf(x[r], cs, -m_use));
#pragma unroll
            for (int r = r0; r < r0 + 8; r += 2) sum += x[r] + x[r + 1];
            p[i] = pack_frag<T>(x[r0], x[r0 + 1], x[r0 + 2], x[r0 + 3], x[r0 + 4], x[r0 + 5],
                                x[r0 + 6], x[r0 + 7]);
        }
        l += sum;
    };
    auto barrier = [] {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };

    if (n > 0) {
        // V_j and K_{j+1}, for j in turn, into the buffers at vd and kd; the loads issued.
        int kd = kBytes, vd = 3 * kBytes;
        auto rotate = [&] {
            kd = kd == 2 * kBytes ? 0 : kd + kBytes;
            vd = vd == 5 * kBytes ? 3 * kBytes : vd + kBytes;
        };
        auto load_kv = [&](int j) {
            int count = 2 * kParts;
            if (j + 1 < whole_tiles) {
                load_whole(V, vd);
                place();
                load_whole(K, kd);
                ask();
            } else {
                if (j < n) load(V, j, vd);
                if (j + 1 < n)
                    load(K, j + 1, kd);
                else
                    count = j < n ? kParts : 0;
            }
            rotate();
            return count;
        };
        // Until only the newest loads, so many, are in flight.
        auto wait_for_older = [&](int newest) {
            if (newest == 2 * kParts)
                wait_loads<2 * kParts>();
            else if (newest == kParts)
                wait_loads<kParts>();
            else
                wait_loads<0>();
        };
        if (whole_tiles > 0) {
            ask();
            place();
            ask();
        }
        const int late = wave >> 2;  // 1: half a step behind
        load(K, 0, 0);
        load_kv(0);
        int newest = 0;
        if (late) newest = load_kv(1);
        wait_for_older(newest);
        barrier();
        scores(smem);
        if (late) barrier();
        int kb = kBytes, vb = 3 * kBytes;  // buffers of K_{j+1} and V_j
        for (int j = 0; j < n; ++j) {
            newest = load_kv(j + 1 + late);
            if (j < nw) softmax(j);
            wait_for_older(newest);
            barrier();
            if (j < nw) {
                __builtin_amdgcn_s_setprio(1);
                products(smem + vb, smem + kb);
                __builtin_amdgcn_s_setprio(0);
            }
            barrier();
            kb = kb == 2 * kBytes ? 0 : kb + kBytes;
            vb = vb == 5 * kBytes ? 3 * kBytes : vb + kBytes;
        }
        if (!late) barrier();  // as many as the others
    }
    store_many(smem, o, m, l, on, orow);
}

template <class Eng>
__device__ __forceinline__ void PagedWork<Eng>::few_rows(unsigned char* smem, float (*s_m)[32],
                                                          float (*s_l)[32]) const {
    constexpr int NW = Eng::kWaves;
    constexpr int kLoads = Eng::kGroups;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31;
    const int g2 = lane >> 5;
    const int row = it.r0 + l32;
    const bool on = row < it.rows;

    typename Eng::Query q;
    Eng::load(q, Q + static_cast<size_t>(on ? out_row(row) : 0) * D, on, g2);
    const int kend = on ? row_end(row) : it.kend;
    int least = kend;
#pragma unroll
    for (int w = 16; w >= 1; w >>= 1) least = min(least, __shfl_xor(least, w, 64));
    const int mask_from = __builtin_amdgcn_readfirstlane(least);
    const int nblk = it.kend > it.kbeg ? (it.kend - it.kbeg + 31) / 32 : 0;

    unsigned char* kt = smem + wave * 2 * Eng::kTile;
    unsigned char* vt = kt + Eng::kTile;
    auto load = [&](const E* src, int b, unsigned char* dst) {
        const int key0 = it.kbeg + 32 * b;
        if (it.of.tiles == 1)
            load_groups<kLoads, true>(src, key0, key0 + 32, 0, 1, dst);
        else
            load_groups<kLoads>(src, key0, key0 + 32, 0, 1, dst);
    };
    // After the Q loads (see the waits of the loop below).
    asm volatile("" ::: "memory");
    if (wave < nblk) {
        load(K, wave, kt);
        load(V, wave, vt);
    }
    const auto lds_at = Eng::offsets(lane);
    f32x16 o[D / 32];
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) o[dt] = f32x16{};
    float m = -INFINITY, l = 0.0f;
    const float cs = fmaxf(a.c, kFltMin);
    // K and V are waited for separately (vmcnt counts a wave's loads in order, kLoads per tile): K
    // before the scores, V before P V; the next K is issued once the scores have read this one, the
    // next V once P V has.
    for (int b = wave; b < nblk; b += NW) {
        const bool next = b + NW < nblk;
        wait_loads<kLoads>();
        Eng::block(kt, vt, lds_at, it.kbeg + 32 * b, mask_from, kend, g2, cs, q, o, m, l, [&] {
            if (next) {
                wait_lds();
                load(K, b + NW, kt);
                wait_loads<kLoads>();
            } else {
                wait_loads<0>();
            }
        });
        if (next) {
            wait_lds();
            load(V, b + NW, vt);
        }
    }

    // Merge: every wave scales its rows to the common max and leaves them in LDS, then the
    // workgroup sums them wave after wave.
    constexpr int P = D + 4;  // pitch of the merge rows (floats)
    static_assert(NW * 32 * P * 4 <= NW * 2 * Eng::kTile, "the merge rows fit the tiles");
    l = pair_sum(l);
    if (g2 == 0) {
        s_m[wave][l32] = m;
        s_l[wave][l32] = l;
    }
    __syncthreads();  // also ends every wave's use of its tiles
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, s_m[w][l32]);
    // No key of this row among the wave's, or every score -inf: such a part has no say, also where 0 times
    // a value made it NaN.
    const bool none = m == -INFINITY;
    const float f = none ? 0.0f : fast_exp2(m - M);
    float* mrg = reinterpret_cast<float*>(smem);
    if (on) {
        float* dst = mrg + (wave * 32 + l32) * P + 4 * g2;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f32x4 w;
#pragma unroll
                for (int u = 0; u < 4; ++u) w[u] = none ? 0.0f : o[dt][4 * i + u] * f;
                st16(dst + 32 * dt + 8 * i, __builtin_bit_cast(u32x4, w));
            }
        }
    }
    __syncthreads();
    constexpr int kPiece = 16 / static_cast<int>(sizeof(E));  // columns of an output's 16 bytes
    constexpr int kPieces = D / kPiece;
#pragma unroll
    for (int i0 = 0; i0 < 32 * kPieces; i0 += 64 * NW) {
        const int i = i0 + threadIdx.x;
        const int r = i / kPieces;
        const int cc = (i % kPieces) * kPiece;
        if (r >= 32 || it.r0 + r >= it.rows) break;
        float ms[NW], MM = -INFINITY, lt = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            ms[w] = s_m[w][r];
            MM = fmaxf(MM, ms[w]);
        }
        float x[kPiece];
#pragma unroll
        for (int u = 0; u < kPiece; ++u) x[u] = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            lt = fmaf(s_l[w][r], ms[w] == -INFINITY ? 0.0f : fast_exp2(ms[w] - MM), lt);
#pragma unroll
            for (int u = 0; u < kPiece; u += 4) {
                const f32x4 y =
                    __builtin_bit_cast(f32x4, ld16(mrg + (w * 32 + r) * P + cc + u));
#pragma unroll
                for (int v = 0; v < 4; ++v) x[u + v] += y[v];
            }
        }
        if (!it.direct) {
            const size_t slot = paged_slot_row<PagedShapeOf<Eng>>(a, hk, false, it.slot, r);
#pragma unroll
            for (int u = 0; u < kPiece; u += 4)
                st16(a.acc + slot * D + cc + u,
                     __builtin_bit_cast(u32x4, f32x4{x[u], x[u + 1], x[u + 2], x[u + 3]}));
            if (cc == 0) a.ml[slot] = make_float2(MM, lt);
            continue;
        }
        const bool none = lt == 0.0f;
        if (none) {
#pragma unroll
            for (int u = 0; u < kPiece; ++u) x[u] = 0.0f;
        }
        const int to = out_row(it.r0 + r);
        st16(O + static_cast<size_t>(to) * D + cc, finish(x, none ? 0.0f : 1.0f / lt));
        if (cc == 0) L[to] = none ? -INFINITY : (MM + fast_log2(lt)) * kLn2;
    }
}

// Second launch bound: waves per SIMD of the workgroups that share a CU.
template <class Eng, bool kShared>
__global__ void __launch_bounds__((64 * Eng::kWaves), (Eng::kPerCu * Eng::kWaves / 4))
    paged_kernel(const typename Mma<typename Eng::T>::elem* __restrict__ Q,
                 const typename Mma<typename Eng::T>::elem* __restrict__ K,
                 const typename Mma<typename Eng::T>::elem* __restrict__ V,
                 typename Mma<typename Eng::T>::elem* __restrict__ O, float* __restrict__ L,
                 PagedArgs a) {
    constexpr int D = Eng::D;
    constexpr int kBytes = Eng::kWaves * 2 * Eng::kTile;
    static_assert(kBytes >= 4 * Eng::kStepBlocks * Eng::kTile, "either kind's tiles");
    __shared__ __attribute__((aligned(1024))) unsigned char smem[kBytes];
    __shared__ float s_m[Eng::kWaves][32];
    __shared__ float s_l[Eng::kWaves][32];
    // The items of a key/value head stay on one XCD where the heads can be dealt out evenly.
    int hk, x;
    head_rank_order(blockIdx.x, a.Hkv, hk, x);
    PagedItem it;
    if constexpr (kShared) {
        it = shared_item<PagedShapeOf<Eng>, GpuWave>(a, x);
    } else {
        // The sequences of more than 64 (see PagedPlan), where they fit.
        PagedSeq* seqs = reinterpret_cast<PagedSeq*>(smem);
        const int per = (a.B + 63) / 64;
        const bool staged = per > 1 && per < kBytes / static_cast<int>(64 * sizeof(PagedSeq));
        if (staged) {
            const int lane = threadIdx.x & 63;
            for (int j = threadIdx.x >> 6; j < per && lane * per + j < a.B; j += Eng::kWaves)
                seqs[lane * (per + 1) + j] = paged_seq(a, lane * per + j);
            __syncthreads();
        }
        it = paged_item<PagedShapeOf<Eng>, GpuWave>(a, x, seqs, staged);
        if (staged) __syncthreads();  // the tiles go to the same place
    }
    if (!it.found) return;
    if (!kShared && a.wgs > 0 && it.first && hk == 0 && threadIdx.x == 0)
        a.units[it.u] = make_int4(it.of.first, it.of.tiles, it.of.chunks, it.many);
    if (!it.direct && it.kend <= it.kbeg) {
        // No keys of this chunk for these rows (a causal mask): nothing but the mark of an empty part.
        const int n = min(it.rows - it.r0, it.many ? PagedShapeOf<Eng>::kTile : 32);
        for (int r = threadIdx.x; r < n; r += 64 * Eng::kWaves)
            a.ml[paged_slot_row<PagedShapeOf<Eng>>(a, hk, it.many, it.slot, r)] =
                make_float2(-INFINITY, 0.0f);
        return;
    }
    const int* table = !kShared     ? a.block_table + static_cast<size_t>(it.u) * a.max_pages
                       : it.u == 0 ? a.prefix_table
                                   : a.block_table + static_cast<size_t>(it.u - 1) * a.max_pages;
    const PagedWork<Eng> work{Q,
                               K + static_cast<size_t>(hk) * D,
                               V + static_cast<size_t>(hk) * D,
                               O,
                               L,
                               a,
                               it,
                               hk,
                               {table, a.page_div, a.page_size,
                                static_cast<size_t>(a.Hkv) * D},
                               // Tiles begin at the unit's first key: behind a prefix, anywhere.
                               a.whole_groups && it.unit.kbeg % Eng::kGroupRows == 0};
    if (std::is_same<typename Eng::T, float>::value || !it.many) {
        work.few_rows(smem, s_m, s_l);
    } else if constexpr (!std::is_same<typename Eng::T, float>::value) {
        if constexpr (Eng::kInTurn)
            work.many_rows_in_turn(smem);
        else
            work.many_rows(smem);
    }
}

// Merges the parts of each row: O = sum O_i 2^(m_i - M) / l with M = max m_i and l = sum l_i
// 2^(m_i - M), L = (M + log2 l) ln 2. D / 4 lanes hold a row, four columns each; kWays groups of them
// take every kWays-th part, kBatch in flight, and are merged through LDS in order. One workgroup per token
// and 256 / (kWays D / 4) query heads.
template <class Eng, int kWays>
__global__ void __launch_bounds__(256)
    paged_combine_kernel(typename Mma<typename Eng::T>::elem* __restrict__ O,
                         float* __restrict__ L, PagedArgs a) {
    using T = typename Eng::T;
    using E = typename Mma<T>::elem;
    using Shape = PagedShapeOf<Eng>;
    constexpr int D = Eng::D;
    constexpr int LPR = D / 4;
    constexpr int kRows = 256 / LPR / kWays;
    constexpr int kBatch = 8;
    __shared__ f32x4 s_acc[256];
    __shared__ float2 s_ml[256 / LPR];
    const int t = blockIdx.x;
    const int slot = threadIdx.x / LPR;
    const int way = slot % kWays;
    const int h = blockIdx.y * kRows + slot / kWays;
    const int part = threadIdx.x % LPR;
    int u = 0;
    if (!a.shared) {
        u = sequence_of(a.starts, a.B, t);
        if (u == a.B) return;  // padding
    }
    const bool on = h < a.H;
    const int hk = a.group_div(on ? h : 0);
    const int g = (on ? h : 0) - hk * a.group;
    // The parts of unit v's row r: `n` of them, from row `at` of acc and ml on, `step` rows apart.
    struct Parts {
        int n;
        size_t at, step;
    };
    auto parts_of = [&](int v, int r) {
        const int4 d = a.units[v];
        if (d.z == 1) return Parts{1, 0, 0};
        const bool many = d.w != 0;
        const int tile = many ? r / Shape::kTile : r / 32;
        const int in = many ? r % Shape::kTile : r % 32;
        const int first = d.x + (a.causal ? d.y - 1 - tile : tile);
        // Where starts that decrease left a unit without items the note is not this call's.
        const bool ok = d.x >= 0 && d.z >= 0 && tile < d.y &&
                        d.x + static_cast<long long>(d.y) * d.z <= (many ? a.max_many : a.max_few);
        return Parts{ok ? d.z : 0, ok ? paged_slot_row<Shape>(a, hk, many, first, in) : 0,
                     static_cast<size_t>(d.y) * (many ? Shape::kTile : a.few_rows)};
    };
    Parts pre{0, 0, 0}, own{0, 0, 0};
    if (a.shared) {
        // Slots as shared_item numbers them.
        const SharedCut& c = a.cut;
        auto cut_parts = [&](bool many, int first, int tiles, int n, int r) {
            const int tile = many ? r / Shape::kTile : r / 32;
            const int in = many ? r % Shape::kTile : r % 32;
            return Parts{n, paged_slot_row<Shape>(a, hk, many, first + tile, in),
                         static_cast<size_t>(tiles) * (many ? Shape::kTile : a.few_rows)};
        };
        pre = cut_parts(c.pre_many, 0, c.pre_tiles, c.pre_chunks, t * a.group + g);
        const int keys = paged_seq_len(a, t) - a.prefix;
        if (keys > 0) {
            const int before = c.pre_many == c.own_many ? c.pre_tiles * c.pre_chunks : 0;
            own = cut_parts(c.own_many, before + t * c.own_chunks * c.own_tiles, c.own_tiles,
                            shared_own_parts(a, keys), g);
        }
    } else {
        own = parts_of(u, (t - a.starts[u]) * a.group + g);
        if (own.n == 1) return;  // written already
    }
    const int parts = on ? pre.n + own.n : 0;
    float M = -INFINITY, l = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int p0 = way; p0 < parts; p0 += kBatch * kWays) {
        float2 v[kBatch];
        f32x4 x[kBatch];
        float M2 = M;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int p = p0 + i * kWays;
            v[i] = make_float2(-INFINITY, 0.0f);
            x[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (p < parts) {
                const size_t s = p < pre.n ? pre.at + p * pre.step
                                           : own.at + (p - pre.n) * own.step;
                v[i] = a.ml[s];
                x[i] = __builtin_bit_cast(f32x4, ld16(a.acc + s * D + 4 * part));
                // No key of this row, or every score -inf: such a part has no say, also where
                // 0 times a value made it NaN.
                if (v[i].x == -INFINITY) x[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) M2 = fmaxf(M2, v[i].x);
        auto weight = [&](float mi) { return mi == -INFINITY ? 0.0f : fast_exp2(mi - M2); };
        const float f0 = weight(M);
        l *= f0;
        acc *= f0;
        M = M2;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const float f = weight(v[i].x);
            l = fmaf(v[i].y, f, l);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = fmaf(x[i][c], f, acc[c]);
        }
    }
    s_acc[threadIdx.x] = acc;
    if (part == 0) s_ml[slot] = make_float2(M, l);
    __syncthreads();
    if (way != 0 || !on) return;
#pragma unroll
    for (int w = 1; w < kWays; ++w) M = fmaxf(M, s_ml[slot + w].x);
    l = 0.0f;
    acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWays; ++w) {
        const float2 v = s_ml[slot + w];
        const f32x4 x = s_acc[threadIdx.x + w * LPR];
        const float f = v.x == -INFINITY ? 0.0f : fast_exp2(v.x - M);
        l = fmaf(v.y, f, l);
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] = fmaf(x[c], f, acc[c]);
    }
    const bool none = l == 0.0f;
    const float inv = none ? 0.0f : 1.0f / l;
    float y[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) y[c] = none ? 0.0f : acc[c] * inv;
    const size_t row = static_cast<size_t>(t) * a.H + h;
    E* dst = O + row * D + 4 * part;
    if constexpr (std::is_same<T, float>::value)
        st16(dst, u32x4{__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]),
                        __float_as_uint(y[3])});
    else
        st8(dst, u32x2{Elem<T>::pack2(y[0], y[1]), Elem<T>::pack2(y[2], y[3])});
    if (part == 0) L[row] = none ? -INFINITY : (M + fast_log2(l)) * kLn2;
}

}  // namespace dev

namespace detail {
namespace {

// Steps and rounds that a chunk has at least: a part of 256 rows is 133 KB to write and to read again.
constexpr int kMinSteps = 6;
// In a shared decode own keys wait for the prefix's items, so these are longer (bf16, 32 heads over 8, us, of 6,
// 8 and 12 steps: 64 sequences behind 2048 keys 41.6, 40.9, 41.6, 128 behind 4000 47.1, 44.1, 41.9, 256 of 2
// key/value heads behind 2000 44.2, 40.5, 42.2, 40 behind 2000 24.2, 25.0, 37.8).
constexpr int kSharedSteps = 8;
constexpr int kMinRounds = 1;

// The sizes of one launch: grid and slots.
template <class Eng>
struct PagedGrid {
    using Shape = dev::PagedShapeOf<Eng>;
    static_assert(dev::is_paged_shape<Shape>(static_cast<dev::PagedShapes*>(nullptr)),
                  "the cut is tested on the host for PagedShapes");
    static constexpr int D = Eng::D;
    int wgs;                     // 0: keys are not cut into chunks
    long long items, many, few;  // per key/value head: items, and slots of either kind
    long long units;
    int kv_heads, few_rows, tokens;
    dev::SharedCut cut;

    PagedGrid(const PagedCall& call, bool shared, bool chunks) {
        kv_heads = call.num_kv_heads;
        tokens = call.num_tokens;
        const int group = call.num_heads / kv_heads;
        wgs = chunks ? (Eng::kPerCu * compute_units() + kv_heads - 1) / kv_heads : 0;
        if (shared) {
            cut = dev::shared_cut<Shape>(call.batch_size, group, call.prefix_len, wgs, kSharedSteps);
            const long long pre = static_cast<long long>(cut.pre_tiles) * cut.pre_chunks;
            const long long own =
                static_cast<long long>(call.batch_size) * cut.own_chunks * cut.own_tiles;
            items = pre + own;
            many = (cut.pre_many ? pre : 0) + (cut.own_many ? own : 0);
            few = items - many;
            units = 0;
            few_rows = cut.pre_many && !cut.own_many && cut.own_tiles == 1 ? group : 32;
            return;
        }
        const dev::PagedTiles tiles =
            dev::paged_tiles<Shape>(call.num_tokens, call.batch_size, group);
        items = tiles.all;
        many = few = 0;
        few_rows = 32;
        units = call.batch_size;
        if (chunks) {
            items = (items + wgs / 2 + wgs) / wgs * wgs;  // paged_room, in 64 bits
            // Items of units with several chunks: at most 3/2 wgs more than tiles (paged_room), and no
            // more tiles than that, as each adds one at least.
            few = std::min(items, 3LL * wgs);
            many = tiles.many ? std::min(few, tiles.many + 2LL * wgs) : 0;
        }
    }
    // A launch has at most 2^32 - 1 threads in x; the merge has a workgroup per token.
    bool too_large() const {
        return items * kv_heads * 64 * Eng::kWaves > 0xffffffffLL ||
               (wgs && 256LL * tokens > 0xffffffffLL);
    }
    size_t slots() const {  // rows of partial results
        return static_cast<size_t>(kv_heads) * (many * Shape::kTile + few * few_rows);
    }
    size_t bytes() const {
        return wgs ? slots() * (D * sizeof(float) + sizeof(float2)) + units * sizeof(int4) : 0;
    }
};

// Whether the tiles alone, at least so many, take three of four workgroup places: chunks cost the partial
// results and the merge (fp32, 512 + 1024 tokens of 8 heads, head_dim 64, 384 tiles for 512 places: 40.7
// -> 31 us without). From num_tokens alone, as the host knows no more: beside
// prompts that fill the chip a token with a long cache has all its keys in one workgroup per key/value head,
// which starts after the prompts' tiles (bf16, 32 heads over 8, head_dim 128, us in one call and in two: 5000
// tokens and one behind 8000 keys 292 and 229, behind 100000 keys 1260 and 302; 4 x 2000 tokens and 32 behind
// 4000 keys 258 and 251).
template <class Eng>
bool fills_chip(const PagedCall& call) {
    const long long rows =
        static_cast<long long>(call.num_tokens) * (call.num_heads / call.num_kv_heads);
    const int tile = rows > Eng::kManyRows ? 32 * Eng::kWaves : 32;
    return 4 * (rows / tile * call.num_kv_heads) >=
           3LL * Eng::kPerCu * compute_units();
}

template <class Eng, bool kShared>
FlashAttentionError run_paged(const PagedCall& call, bool chunks, hipStream_t stream) {
    using T = typename Eng::T;
    using E = typename dev::Mma<T>::elem;
    constexpr int D = Eng::D;
    constexpr bool shared = kShared;
    dev::PagedArgs a{};
    a.block_table = call.block_table;
    a.prefix_table = call.prefix_table;
    a.seq_lens = call.seq_lens;
    a.starts = call.query_starts;
    a.B = call.batch_size;
    a.T = call.num_tokens;
    a.H = call.num_heads;
    a.Hkv = call.num_kv_heads;
    a.group = a.H / a.Hkv;
    a.page_size = call.page_size;
    a.max_pages = call.max_pages;
    a.cap = a.page_size * a.max_pages;
    a.page_div = dev::fast_div(a.page_size);
    a.group_div = dev::fast_div(a.group);
    a.shared = shared;
    a.causal = call.causal;
    a.prefix = call.prefix_len;
    // Loads from a multiple of their rows stay on one page, and their lane offsets fit 32 bits.
    a.whole_groups = a.page_size % Eng::kGroupRows == 0 &&
                     static_cast<long long>(a.Hkv) * D * Eng::kGroupRows * 4 < (1LL << 31);
    a.c = call.scale * dev::kLog2e;
    a.min_steps = kMinSteps;
    a.min_rounds = kMinRounds;

    const PagedGrid<Eng> grid(call, shared, chunks);
    if (grid.too_large()) return FlashAttentionError::INVALID_DIMENSION;
    a.wgs = grid.wgs;
    a.cut = grid.cut;
    a.max_many = static_cast<int>(grid.many);
    a.max_few = static_cast<int>(grid.few);
    a.few_rows = grid.few_rows;
    StreamWorkspace ws(stream, true);
    if (chunks) {
        void* base = call.workspace;
        if (base == nullptr) {
            FlashAttentionError err = ws.alloc(grid.bytes());
            if (err != FlashAttentionError::SUCCESS) return err;
            base = ws.get();
        } else if (call.workspace_bytes < grid.bytes()) {
            return FlashAttentionError::OUT_OF_MEMORY;
        }
        a.acc = static_cast<float*>(base);
        a.ml = reinterpret_cast<float2*>(a.acc + grid.slots() * D);
        a.units = reinterpret_cast<int4*>(a.ml + grid.slots());
    }
    ProfileEvents tok = profile_kernel<T, D>(shared ? "decode_shared" : "forward_paged");
    auto go = [&](auto kernel) {
        launch_kernel(tok, kernel, dim3(static_cast<unsigned>(grid.items * a.Hkv)),
                      dim3(64 * Eng::kWaves), 0, stream, static_cast<const E*>(call.Q),
                      static_cast<const E*>(call.K_cache), static_cast<const E*>(call.V_cache),
                      static_cast<E*>(call.O), call.L, a);
    };
    if constexpr (kShared)
        go(dev::paged_kernel<Eng, true>);
    else
        go(dev::paged_kernel<Eng, false>);
    FlashAttentionError err = from_hip(hipGetLastError());
    if (err != FlashAttentionError::SUCCESS || !chunks) return err;
    tok = profile_kernel<T, D>("paged_combine");
    auto merge = [&](auto kernel, int ways) {
        const int rows = 256 / (D / 4) / ways;
        launch_kernel(tok, kernel,
                      dim3(static_cast<unsigned>(a.T),
                           static_cast<unsigned>((a.H + rows - 1) / rows)),
                      dim3(256), 0, stream, static_cast<E*>(call.O), call.L, a);
    };
    // Few rows have many parts each and want more loads in flight: 61 tokens of 8253 keys, 32 heads,
    // 9.2 -> 7.0 us; 250 tokens 8.8 -> 11.3.
    if (static_cast<long long>(a.T) * a.H * D <= (1 << 19))
        merge(dev::paged_combine_kernel<Eng, 4>, 4);
    else
        merge(dev::paged_combine_kernel<Eng, 1>, 1);
    return from_hip(hipGetLastError());
}

// Workgroups: eight waves (four in fp32), and at head_dim 128 four, two workgroups a CU, where most
// sequences have few rows: the start of one workgroup then hides behind the other. In a shared decode, where
// the batch has few rows or the prefix is not so long that the products over it take most of the time. Kernel
// times, us, eight waves -> four: 16 x 5 tokens of up to 8196 keys 64.5 -> 63.0; 250 tokens of 8442 keys
// 44.3 -> 55.9, 4 x 61 tokens of 8253 keys 38.5 -> 43.1. Shared, 32 heads over 8, up to 300 own keys: 4
// sequences behind 1000 keys 8.3 -> 7.7, 128 behind 500 40.8 -> 31.8, behind 4000 55.0 -> 48.0, behind 16000
// 76.9 -> 78.1, 512 behind 4000 155.7 -> 130.6, behind 16000 227.9 -> 230.5, 128 with up to 512 own keys
// behind 32768 113 -> 124.
template <typename T, int D>
struct PagedEngines {
    static constexpr int kWaves = std::is_same<T, float>::value ? 4 : 8;
    using Rows = dev::PagedEngine<T, D, kWaves>;
    using Few = dev::PagedEngine<T, D, D == 128 ? 4 : kWaves>;
    static bool few(const PagedCall& call, bool shared) {
        return (shared && call.prefix_len <= 8192) ||
               static_cast<long long>(call.num_tokens) * (call.num_heads / call.num_kv_heads) <=
                   static_cast<long long>(shared ? 1 : call.batch_size) * Rows::kManyRows;
    }
};

template <typename T, int D>
FlashAttentionError run_paged_dim(const PagedCall& call, hipStream_t stream) {
    using Engines = PagedEngines<T, D>;
    const bool shared = call.query_starts == nullptr;
    if (shared || !fills_chip<typename Engines::Rows>(call)) {
        // A graph's replays need memory that is theirs: the caller's. (Memory that the graph itself
        // allocates, a recorded hipMallocAsync, was not there in the replay of two graphs in a row.)
        if (call.workspace != nullptr || !stream_capturing(stream)) {
            const bool few = Engines::few(call, shared);
            if (shared)
                return few ? run_paged<typename Engines::Few, true>(call, true, stream)
                           : run_paged<typename Engines::Rows, true>(call, true, stream);
            return few ? run_paged<typename Engines::Few, false>(call, true, stream)
                       : run_paged<typename Engines::Rows, false>(call, true, stream);
        }
        if (shared)
            return PagedGrid<typename Engines::Rows>(call, true, true).too_large()
                       ? FlashAttentionError::INVALID_DIMENSION
                       : FlashAttentionError::OUT_OF_MEMORY;
    }
    return run_paged<typename Engines::Rows, false>(call, false, stream);
}

template <typename T, int D>
long long workspace_of(const PagedCall& call) {
    using Engines = PagedEngines<T, D>;
    const bool shared = call.prefix_len > 0;
    const bool chunks = shared || !fills_chip<typename Engines::Rows>(call);
    auto bytes = [](const auto& grid) {
        return grid.too_large() ? -1 : static_cast<long long>(grid.bytes());
    };
    if (shared) {  // of any prefix
        const long long few = bytes(PagedGrid<typename Engines::Few>(call, true, true));
        const long long rows = bytes(PagedGrid<typename Engines::Rows>(call, true, true));
        return few < 0 || rows < 0 ? -1 : std::max(few, rows);
    }
    if (chunks && Engines::few(call, false))
        return bytes(PagedGrid<typename Engines::Few>(call, false, true));
    return bytes(PagedGrid<typename Engines::Rows>(call, shared, chunks));
}

}  // namespace

template <typename T>
long long paged_workspace(const PagedCall& c) {
    return c.head_dim == 32   ? workspace_of<T, 32>(c)
           : c.head_dim == 64 ? workspace_of<T, 64>(c)
                              : workspace_of<T, 128>(c);
}

template <typename T>
FlashAttentionError launch_paged(const PagedCall& c, hipStream_t stream) {
    switch (c.head_dim) {
        case 32:
            return run_paged_dim<T, 32>(c, stream);
        case 64:
            return run_paged_dim<T, 64>(c, stream);
        case 128:
            return run_paged_dim<T, 128>(c, stream);
    }
    return FlashAttentionError::UNSUPPORTED_HEAD_DIM;
}
#define CUFLASH_PAGED_TYPE(T)                              \
    template long long paged_workspace<T>(const PagedCall&); \
    template FlashAttentionError launch_paged<T>(const PagedCall&, hipStream_t);
CUFLASH_PAGED_TYPE(float)
CUFLASH_PAGED_TYPE(__half)
CUFLASH_PAGED_TYPE(__hip_bfloat16)
#undef CUFLASH_PAGED_TYPE

}  // namespace detail
}  // namespace cuflash
