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
//  * Fewer: tiles of 32 rows whose keys are spread over the waves, kRound keys in each round. A round
//    brings as many bytes as kRoundCost steps take time for.
// Where the tiles alone do not fill the chip (`wgs` > 0), the keys of every unit are cut into chunks
// that cost at most `s`, with the least s that leaves the items of one key/value head at whole rounds
// of the workgroups that run at once: the next multiple of wgs beyond tiles + wgs / 2. Chunks leave
// partial results in slots of their own, numbered like the items, and the first item of a unit notes
// where they are.
constexpr int kManyRows = 96;

template <int TILE, int STEP, int ROUND, int COST>
struct PagedShape {
    static constexpr int kTile = TILE;
    static constexpr int kStep = STEP;
    static constexpr int kRound = ROUND;
    static constexpr int kRoundCost = COST;
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
    int wgs;            // workgroups per key/value head that run at once; 0: no chunks
    int min_steps, min_rounds;  // least per chunk
    int max_many, max_few;      // slots per key/value head for the items of either kind
    float c;                    // scale * log2(e)
    float* acc;   // [Hkv, max_many, kTile, D], then [Hkv, max_few, 32, D]
    float2* ml;   // the same without D: m in log2 units, l
    int4* units;  // [units]: see PagedUnitItems
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

__host__ __device__ __forceinline__ int paged_room(int tiles, int wgs) {
    return (tiles + wgs / 2 + wgs) / wgs * wgs;
}

// The cut of one launch. W: the 64 lanes of a wave, one int each in W::Int.
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
    // Steps or rounds of a chunk that costs at most s.
    __host__ __device__ static int longest(const PagedArgs& a, bool many, int s) {
        if (many) return s > a.min_steps ? s : a.min_steps;
        s /= Shape::kRoundCost;
        return s > a.min_rounds ? s : a.min_rounds;
    }
    // Chunks of a unit of n steps. One without keys still has outputs, but for a shared decode,
    // where the combine writes them.
    __host__ __device__ static int chunks(const PagedArgs& a, int n, int most) {
        if (n == 0) return a.shared ? 0 : 1;
        return most >= n ? 1 : (n + most - 1) / most;
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
    // Items of every unit.
    __host__ __device__ static Int items(const PagedArgs& a, const Batch& b, int s) {
        const int many = longest(a, true, s), few = longest(a, false, s);
        return W::map2(b.rows, b.keys, [&](int rows, int keys) {
            return tiles(rows) * chunks(a, steps(rows, keys), rows > kManyRows ? many : few);
        });
    }
    __host__ __device__ static Int of_kind(const Batch& b, const Int& items, bool many) {
        return W::map2(b.rows, items,
                       [&](int rows, int n) { return (rows > kManyRows) == many ? n : 0; });
    }
    // f summed over the units.
    template <class F>
    __host__ __device__ static int sum(const PagedArgs& a, const Batch& first, F f) {
        int total = 0;
        for (int u0 = 0; u0 < paged_units(a); u0 += 64)
            total += W::lane(W::scan(f(u0 == 0 ? first : batch(a, u0))), 63);
        return total;
    }
    // The greatest cost of a chunk: integers only, every workgroup comes to the same.
    __host__ __device__ static int cut(const PagedArgs& a, const Batch& first) {
        if (a.wgs == 0) return kNoChunks;
        const int total = sum(a, first, [&](const Batch& b) {
            return W::map2(b.rows, b.keys, [&](int rows, int) { return tiles(rows); });
        });
        int work = 0;
        for (int u0 = 0; u0 < paged_units(a); u0 += 64) {
            const Batch b = u0 == 0 ? first : batch(a, u0);
            const Int w = W::map2(b.rows, b.keys, [&](int rows, int keys) {
                const float x = static_cast<float>(tiles(rows)) *
                                static_cast<float>(steps(rows, keys)) *
                                (rows > kManyRows ? 1 : Shape::kRoundCost);
                return x > 16777216.0f ? 1 << 24 : static_cast<int>(x);  // exact below
            });
            work += W::lane(W::scan(w), 63);  // at most 2^30
            if (work > 1 << 30) work = 1 << 30;
        }
        // Chunks of at most s: at most work / s + tiles items, so the least s that keeps them within
        // the room lies in [work / room, work / (room - tiles)], rounded up. (A round of a few-rows
        // unit cannot be cut, and counts as one chunk of its own: the bound holds for s >= kRoundCost.)
        const int room = paged_room(total, a.wgs);
        int lo = (work + room - 1) / room;
        if (lo < Shape::kRoundCost) lo = Shape::kRoundCost;
        int hi = (work + room - total - 1) / (room - total) + Shape::kRoundCost - 1;
        if (hi < lo) hi = lo;
        auto fits = [&](int s) {
            return sum(a, first, [&](const Batch& b) { return items(a, b, s); }) <= room;
        };
        // With several batches of units every trial reads them all again: the upper end then.
        if (paged_units(a) > 64) lo = hi;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (fits(mid))
                hi = mid;
            else
                lo = mid + 1;
        }
        return lo;
    }
};

// A unit's items in one launch: `first` is the index of its first one among those of its kind; item
// first + chunk * tiles + i is chunk `chunk` of tile i (of tile tiles - 1 - i with a causal mask:
// the longest tiles start first). As noted in PagedArgs::units: {first, tiles, chunks, many}.
struct PagedUnitItems {
    int first, tiles, chunks;
    bool many;
};

// One workgroup's part: rows [r0, r0 + kTile or 32) of unit u's `rows`, keys [kbeg, kend).
struct PagedItem {
    bool found, many;
    bool direct;  // the only part of its rows: outputs, no partial results
    bool first;   // the first item of its unit
    int u, rows, r0;
    int kbeg, kend;
    int index;  // among the items of its kind: the slot
    PagedUnit unit;
    PagedUnitItems of;  // the unit's items
};

template <class Shape, class W>
__host__ __device__ __forceinline__ PagedItem paged_item(const PagedArgs& a, int x) {
    using Plan = PagedPlan<Shape, W>;
    PagedItem r{};
    const auto first = Plan::batch(a, 0);
    const int s = Plan::cut(a, first);
    // Items of many rows come first: they take longest.
    const int units = paged_units(a);
    for (int kind = 0; kind < 2; ++kind) {
        r.many = kind == 0;
        int before = 0;
        for (int u0 = 0; u0 < units; u0 += 64) {
            const auto b = u0 == 0 ? first : Plan::batch(a, u0);
            const auto own = Plan::of_kind(b, Plan::items(a, b, s), r.many);
            const auto incl = W::scan(own);
            const int i = W::first(incl, [&](int n) { return before + n > x; });
            if (i < 0) {
                before += W::lane(incl, 63);
                continue;
            }
            r.u = u0 + i;
            r.rows = W::lane(b.rows, i);
            r.index = x;
            const int slots = r.many ? a.max_many : a.max_few;
            r.found = a.wgs == 0 || before + W::lane(incl, i) <= slots;
            const int keys = W::lane(b.keys, i);
            const int at = x - before - (W::lane(incl, i) - W::lane(own, i));
            r.of.first = x - at;
            r.of.tiles = Plan::tiles(r.rows);
            r.of.many = r.many;
            const int n = Plan::steps(r.rows, keys);
            r.of.chunks = Plan::chunks(a, n, Plan::longest(a, r.many, s));
            const int chunk = at / r.of.tiles;
            const int in = at - chunk * r.of.tiles;
            r.first = at == 0;
            r.r0 = (a.causal ? r.of.tiles - 1 - in : in) * (r.many ? Shape::kTile : 32);
            r.direct = r.of.chunks == 1 && !a.shared;
            r.unit = paged_unit(a, r.u);
            // (chunks - 1) each <= (chunks - 1) most < n: the last chunk has keys as well.
            const int each = (n + r.of.chunks - 1) / r.of.chunks;
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
        x -= before;
    }
    return r;
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
