#pragma once

// How the attention of packed tokens over a paged cache is cut into workgroups
// (flash_attention_forward_paged, flash_attention_decode_shared). How many tokens and keys a sequence
// has is known on the device only, so every workgroup finds its part by itself, from the same sums
// over the sequences. Everything that becomes an address or a loop bound is formed here, in code that
// also compiles for the host, where tests/cpp/test_paged_plan.cpp runs it with every index checked.

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cuflash {
namespace dev {

// n / d for 0 <= n < 2^31 and 1 <= d < 2^31 as a product and a shift: with 2^(s-1) < d <= 2^s and
// mul = ceil(2^(31+s) / d) the product's error, n (mul d - 2^(31+s)) / d < n 2^s / d, stays below
// 2^(31+s) / d.
struct FastDiv {
    uint32_t mul;
    uint32_t shift;
    __host__ __device__ __forceinline__ int operator()(int n) const {
        return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * mul) >> shift);
    }
};
inline FastDiv fast_div(int d) {
    uint32_t s = 0;
    while ((int64_t(1) << s) < d) ++s;
    return {static_cast<uint32_t>(((uint64_t(1) << (31 + s)) + d - 1) / d), 31 + s};
}

// A unit is the tokens of one sequence over its keys; in a shared decode unit 0 is the whole batch
// over the shared keys and unit b + 1 sequence b over its own ones. The rows of a unit are its
// tokens times the query heads of one key/value head (row r: token r / group, head r % group).
//  * More than kManyRows rows: tiles of kTile rows, one 32-row strip per wave, whose waves share the
//    keys, kStep at a time.
//  * Fewer: tiles of 32 rows whose keys are spread over the waves, kRound keys in each round.
// Where the tiles alone do not fill the chip (per_head > 0), the keys of every unit are cut into
// chunks of whole steps or rounds, at most `s` of them, the least s with which the items of one
// key/value head number about per_head: the work of a head is W = sum of tiles times steps, and s =
// W / per_head rounded up gives at most per_head items and one more per tile. Chunks leave partial
// results in slots of their own, numbered like the items.
constexpr int kManyRows = 96;

template <int TILE, int STEP, int ROUND>
struct PagedShape {
    static constexpr int kTile = TILE;
    static constexpr int kStep = STEP;
    static constexpr int kRound = ROUND;
};

struct PagedArgs {
    const int* block_table;   // [B, max_pages]
    const int* prefix_table;  // pages of the shared keys
    const int* seq_lens;      // [B]
    const int* starts;        // [B + 1], not in a shared decode
    int B, T, H, Hkv, group;
    int page_size, max_pages, cap;  // cap = page_size * max_pages
    FastDiv page_div, group_div;
    bool shared, causal;
    bool whole_groups;  // the rows of one load are a divisor of the page's
    int prefix;         // shared keys
    int per_head;       // items per key/value head that the chunks aim at; 0: no chunks
    int min_steps, min_rounds;   // least per chunk
    int max_many, max_few;       // slots per key/value head for the items of either kind
    float c;                     // scale * log2(e)
    float* acc;  // [Hkv, max_many, kTile, D], then [Hkv, max_few, 32, D]
    float2* ml;  // the same without D: m in log2 units, l
};

struct PagedUnit {
    int t0, n;       // tokens
    int kbeg, kend;  // keys
};

__host__ __device__ __forceinline__ int paged_clamp(int x, int lo, int hi) {
    return x < lo ? lo : x > hi ? hi : x;
}
__host__ __device__ __forceinline__ int paged_seq_len(const PagedArgs& a, int b) {
    return paged_clamp(a.seq_lens[b], 0, a.cap);
}
__host__ __device__ __forceinline__ int paged_units(const PagedArgs& a) {
    return a.shared ? a.B + 1 : a.B;
}
__host__ __device__ __forceinline__ PagedUnit paged_unit(const PagedArgs& a, int u) {
    if (a.shared) {
        if (u == 0) return {0, a.B, 0, a.prefix};
        const int len = paged_seq_len(a, u - 1);
        return {u - 1, 1, a.prefix, len > a.prefix ? len : a.prefix};
    }
    const int t0 = paged_clamp(a.starts[u], 0, a.T);
    const int t1 = paged_clamp(a.starts[u + 1], t0, a.T);
    return {t0, t1 - t0, 0, paged_seq_len(a, u)};
}
// Keys that token i of unit u sees: those of the unit below the limit.
__host__ __device__ __forceinline__ int paged_limit(const PagedArgs& a, int u, const PagedUnit& pu,
                                                    int i) {
    if (a.shared && u == 0) {
        const int len = paged_seq_len(a, i);
        return len < pu.kend ? len : pu.kend;
    }
    if (!a.causal) return pu.kend;
    const int lim = pu.kend - pu.n + i + 1;
    return lim > 0 ? lim : 0;
}

// The cut of one launch: chunks of at most s steps, and the items of either kind.
struct PagedCut {
    int s;
    int many, few;
};

// The sums over the units. W: the 64 lanes of a wave, one int each in W::Int.
template <class Shape, class W>
struct PagedPlan {
    using Int = typename W::Int;
    static constexpr int kNoChunks = 0x7fffffff;

    __host__ __device__ static int tiles(int rows) {
        return rows > kManyRows ? (rows + Shape::kTile - 1) / Shape::kTile : (rows + 31) / 32;
    }
    __host__ __device__ static int steps(int rows, int keys) {
        return rows > kManyRows ? keys / Shape::kStep + (keys % Shape::kStep > 0)
                                : keys / Shape::kRound + (keys % Shape::kRound > 0);
    }
    // Chunks of a unit. One without keys still has outputs, but for a shared decode, where the
    // combine writes them.
    __host__ __device__ static int chunks(const PagedArgs& a, int rows, int keys, int s) {
        const int n = steps(rows, keys);
        if (n == 0) return a.shared ? 0 : 1;
        const int least = rows > kManyRows ? a.min_steps : a.min_rounds;
        if (s < least) s = least;
        return s >= n ? 1 : (n + s - 1) / s;
    }
    struct Batch {  // 64 units
        Int rows, keys;
    };
    __host__ __device__ static Batch batch(const PagedArgs& a, int u0) {
        const int units = paged_units(a);
        Batch b;
        b.rows = W::each([&](int lane) {
            return u0 + lane < units ? paged_unit(a, u0 + lane).n * a.group : 0;
        });
        b.keys = W::each([&](int lane) {
            if (u0 + lane >= units) return 0;
            const PagedUnit u = paged_unit(a, u0 + lane);
            return u.kend - u.kbeg;
        });
        return b;
    }
    __host__ __device__ static Int items(const PagedArgs& a, const Batch& b, int s, bool many) {
        return W::map2(b.rows, b.keys, [&](int rows, int keys) {
            return (rows > kManyRows) == many ? tiles(rows) * chunks(a, rows, keys, s) : 0;
        });
    }
    __host__ __device__ static void count(const PagedArgs& a, const Batch& first, PagedCut& cut) {
        cut.many = cut.few = 0;
        for (int u0 = 0; u0 < paged_units(a); u0 += 64) {
            const Batch b = u0 == 0 ? first : batch(a, u0);
            cut.many += W::lane(W::scan(items(a, b, cut.s, true)), 63);
            cut.few += W::lane(W::scan(items(a, b, cut.s, false)), 63);
        }
    }
    // Every workgroup and the combine come to the same cut: integers only.
    __host__ __device__ static PagedCut cut(const PagedArgs& a, const Batch& first) {
        PagedCut c{kNoChunks, 0, 0};
        if (a.per_head > 0) {
            int work = 0;
            for (int u0 = 0; u0 < paged_units(a); u0 += 64) {
                const Batch b = u0 == 0 ? first : batch(a, u0);
                const Int w = W::map2(b.rows, b.keys, [&](int rows, int keys) {
                    const int64_t x = static_cast<int64_t>(tiles(rows)) * steps(rows, keys);
                    return x > (1 << 24) ? 1 << 24 : static_cast<int>(x);
                });
                work += W::lane(W::scan(w), 63);  // at most 2^30
                if (work > 1 << 30) work = 1 << 30;
            }
            c.s = work / a.per_head + 1;
            count(a, first, c);
            // More items than slots (a sum of work above that was cut off): no chunks.
            if (c.many <= a.max_many && c.few <= a.max_few) return c;
            c.s = kNoChunks;
        }
        count(a, first, c);
        return c;
    }
};

// A unit's items in one launch: `first` is the index of its first one among those of its kind; item
// first + chunk * tiles + i is chunk `chunk` of tile i (of tile tiles - 1 - i with a causal mask:
// the longest tiles start first).
struct PagedUnitItems {
    bool many;
    int first, tiles, chunks;
};

// One workgroup's part: rows [r0, r0 + kTile or 32) of unit u's `rows`, keys [kbeg, kend).
struct PagedItem {
    bool found, many;
    bool direct;  // the only part of its rows: outputs, no partial results
    int u, rows, r0;
    int kbeg, kend;
    int index;  // among the items of its kind: the slot
    PagedUnit unit;
};

template <class Shape, class W>
__host__ __device__ __forceinline__ PagedItem paged_item(const PagedArgs& a, int x) {
    using Plan = PagedPlan<Shape, W>;
    PagedItem r{};
    const auto first = Plan::batch(a, 0);
    const PagedCut cut = Plan::cut(a, first);
    if (x >= cut.many + cut.few) return r;
    r.many = x < cut.many;
    r.index = r.many ? x : x - cut.many;
    int before = 0;
    for (int u0 = 0; u0 < paged_units(a); u0 += 64) {
        const auto b = u0 == 0 ? first : Plan::batch(a, u0);
        const auto own = Plan::items(a, b, cut.s, r.many);
        const auto incl = W::scan(own);
        const int i = W::first(incl, [&](int n) { return before + n > r.index; });
        if (i < 0) {
            before += W::lane(incl, 63);
            continue;
        }
        r.found = true;
        r.u = u0 + i;
        r.rows = W::lane(b.rows, i);
        const int keys = W::lane(b.keys, i);
        const int at = r.index - before - (W::lane(incl, i) - W::lane(own, i));
        const int tiles = Plan::tiles(r.rows);
        const int chunks = Plan::chunks(a, r.rows, keys, cut.s);
        const int chunk = at / tiles;
        const int tile = a.causal ? tiles - 1 - (at - chunk * tiles) : at - chunk * tiles;
        r.r0 = tile * (r.many ? Shape::kTile : 32);
        r.direct = chunks == 1 && !a.shared;
        r.unit = paged_unit(a, r.u);
        // (chunks - 1) each <= (chunks - 1) s < steps: the last chunk has keys as well.
        const int each = (Plan::steps(r.rows, keys) + chunks - 1) / chunks;
        const int64_t len = static_cast<int64_t>(each) * (r.many ? Shape::kStep : Shape::kRound);
        const int64_t beg = r.unit.kbeg + chunk * len;
        r.kbeg = static_cast<int>(beg);
        r.kend = beg + len < r.unit.kend ? static_cast<int>(beg + len) : r.unit.kend;
        // With a causal mask, no further than the last row of the tile sees.
        if (a.causal && !a.shared) {
            const int last = (r.many ? Shape::kTile : 32) + r.r0;
            const int lim =
                paged_limit(a, r.u, r.unit, a.group_div((last < r.rows ? last : r.rows) - 1));
            if (lim < r.kend) r.kend = lim;
        }
        return r;
    }
    return r;
}

template <class Shape, class W>
__host__ __device__ __forceinline__ PagedUnitItems
paged_unit_items(const PagedArgs& a, const PagedCut& cut,
                 const typename PagedPlan<Shape, W>::Batch& first, int u) {
    using Plan = PagedPlan<Shape, W>;
    int before_many = 0, before_few = 0;
    for (int u0 = 0;; u0 += 64) {
        const auto b = u0 == 0 ? first : Plan::batch(a, u0);
        const auto many = W::scan(Plan::items(a, b, cut.s, true));
        const auto few = W::scan(Plan::items(a, b, cut.s, false));
        if (u < u0 + 64) {
            const int i = u - u0;
            const int rows = W::lane(b.rows, i);
            PagedUnitItems r;
            r.many = rows > kManyRows;
            r.tiles = Plan::tiles(rows);
            r.chunks = Plan::chunks(a, rows, W::lane(b.keys, i), cut.s);
            r.first = (r.many ? before_many + W::lane(many, i) : before_few + W::lane(few, i)) -
                      r.tiles * r.chunks;
            return r;
        }
        before_many += W::lane(many, 63);
        before_few += W::lane(few, 63);
    }
}

// Row of `acc` and `ml` that item `index`'s row r has.
template <class Shape>
__host__ __device__ __forceinline__ size_t paged_slot_row(const PagedArgs& a, int hk, bool many,
                                                          int index, int r) {
    if (many)
        return (static_cast<size_t>(hk) * a.max_many + index) * Shape::kTile + r;
    return static_cast<size_t>(a.Hkv) * a.max_many * Shape::kTile +
           (static_cast<size_t>(hk) * a.max_few + index) * 32 + r;
}

// Sizes that the host knows: the tiles of either kind that `units` sequences with `tokens` tokens in
// all can have at most.
struct PagedTiles {
    long long many, few;
};
template <class Shape>
inline PagedTiles paged_tiles(long long tokens, long long units, int group) {
    const long long rows = tokens * group;
    const long long with = units < tokens ? units : tokens;  // sequences that have tokens
    const long long big = rows / (kManyRows + 1) < with ? rows / (kManyRows + 1) : with;
    const long long a = rows / 32 + with, b = with * ((kManyRows + 31) / 32);
    return {big ? rows / Shape::kTile + big : 0, a < b ? a : b};
}

}  // namespace dev
}  // namespace cuflash
