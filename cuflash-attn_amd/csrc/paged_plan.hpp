#pragma once

// How the attention of packed tokens over a paged cache is cut into workgroups
// (flash_attention_forward_paged, flash_attention_decode_shared). How many tokens and keys a sequence
// has is known on the device only, so every workgroup finds its part by itself, from the same sums
// over the sequences. Everything that becomes an address or a loop bound is formed here, in code that
// also compiles for the host, where tests/cpp/test_paged_plan.cpp runs it with every index checked.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <tuple>
#include <type_traits>

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
// Work comes in items, one workgroup's tile of rows over a chunk of keys:
//  * More than kMany rows: tiles of kTile rows, one 32-row strip per wave, whose waves share the
//    keys, kStep at a time.
//  * Fewer: tiles of 32 rows whose keys are spread over the waves, kRound keys in each round. A round
//    brings as many bytes as kRoundCost steps take time for.
// A shared decode is cut by the host, but for the own keys of a sequence, whose length a workgroup
// reads (SharedCut). In a forward, where the tiles alone do not fill the chip (`wgs` > 0), the keys of
// every unit are cut into chunks that cost at most `s`, with the least s that leaves the items of one
// key/value head at whole rounds of the workgroups that run at once: the next multiple of wgs beyond
// tiles + wgs / 2. The items of units with several chunks leave partial results in slots, numbered in
// their order among their kind, and the first item of a forward's unit notes where they are.
template <int TILE, int STEP, int ROUND, int COST, int MANY>
struct PagedShape {
    static constexpr int kMany = MANY;
    static constexpr int kTile = TILE;
    static constexpr int kStep = STEP;
    static constexpr int kRound = ROUND;
    static constexpr int kRoundCost = COST;
};

// The shapes that paged.hip's engines have: 16 bits with eight and with four waves, fp32.
using PagedShapes = std::tuple<PagedShape<256, 64, 256, 2, 96>, PagedShape<128, 64, 128, 2, 96>,
                               PagedShape<128, 32, 128, 1, 0x7fffffff>>;
template <class Shape, class... Known>
constexpr bool is_paged_shape(const std::tuple<Known...>*) {
    return (std::is_same<Shape, Known>::value || ...);
}

// The cut of a shared decode: unit 0 in `pre_chunks` chunks of pre_len keys; the own keys of every
// sequence in at most own_chunks, of own_least keys or more. Items: unit 0, chunk by chunk, then
// sequence by sequence.
struct SharedCut {
    int pre_tiles, pre_chunks, pre_len;
    int own_tiles, own_chunks, own_least;
    FastDiv own_items_div, own_tiles_div, pre_tiles_div;
    bool pre_many, own_many;
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
    int few_rows;               // rows of a slot for an item of few rows
    float* acc;   // [Hkv, max_many, kTile, D], then [Hkv, max_few, few_rows, D]
    float2* ml;   // the same without D: m in log2 units, l
    int4* units;  // [B], forward: see PagedUnitItems
    SharedCut cut;
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

// Division by a number that is the same for the whole launch, by its reciprocal: n < 2^31. The first
// quotient is off by a few, what remains of n is small, and the second by at most one.
struct UniformDiv {
    int d;
    float r;
    __host__ __device__ __forceinline__ explicit UniformDiv(int by) : d(by) {
#ifdef __HIP_DEVICE_COMPILE__
        r = __builtin_amdgcn_rcpf(static_cast<float>(by));
#else
        r = 1.0f / static_cast<float>(by);
#endif
    }
    __host__ __device__ __forceinline__ int operator()(int n) const {
        int q = static_cast<int>(static_cast<float>(n) * r);
        // In 64 bits where q d may pass 2^31 by the error of q.
        int rest = static_cast<int>(n - static_cast<int64_t>(q) * d);
        const int more = static_cast<int>(static_cast<float>(rest) * r);
        q += more;
        rest -= more * d;
        if (rest < 0) {
            --q;
            rest += d;
        }
        return rest >= d ? q + 1 : q;
    }
};

constexpr int kNoChunks = 0x7fffffff;

// Rows and keys of a sequence in a forward.
struct PagedSeq {
    int rows, keys;
};
__host__ __device__ __forceinline__ PagedSeq paged_seq(const PagedArgs& a, int b) {
    const int t0 = paged_clamp(a.starts[b], 0, a.T);
    return {(paged_clamp(a.starts[b + 1], t0, a.T) - t0) * a.group, paged_seq_len(a, b)};
}

// The cut of one launch, found by every wave for itself: a few hundred instructions and two loads that
// need each other, which every workgroup waits for. W: the 64 lanes of a wave, one int each in W::Int.
// Lane i has the `per` sequences from i per on, the first of them in registers. Where there are several,
// the workgroup has put them side by side in LDS (`seqs`: sequence i per + j at i (per + 1) + j, so that
// the lanes meet different banks), as they are gone through several times: one token each, 32 heads over 8,
// head_dim 128, of 512 sequences with up to 500 keys 309 -> 179 us, of 1024 with up to 60 keys 809 -> 222.
template <class Shape, class W>
struct PagedPlan {
    using Int = typename W::Int;
    struct Most {  // steps, rounds of a chunk
        UniformDiv many, few;
    };

    const PagedArgs& a;
    int per;
    const PagedSeq* seqs;
    bool staged;
    Int rows0, keys0;
    Most most;
    Int many, few;              // items of either kind up to and with the lane's
    Int many_slots, few_slots;  // the lane's items of units with several chunks

    __host__ __device__ __forceinline__ static int up(int x, int by) {
        return static_cast<int>((static_cast<uint32_t>(x) + (by - 1)) / by);
    }
    __host__ __device__ __forceinline__ static int tiles(int rows) {
        return rows > Shape::kMany ? up(rows, Shape::kTile) : up(rows, 32);
    }
    __host__ __device__ __forceinline__ static int steps(int rows, int keys) {
        return rows > Shape::kMany ? up(keys, Shape::kStep) : up(keys, Shape::kRound);
    }
    // Sequence j of a lane.
    __host__ __device__ __forceinline__ PagedSeq seq(int lane, int j) const {
        return staged ? seqs[lane * (per + 1) + j] : paged_seq(a, lane * per + j);
    }
    // Chunks of n steps, items of a unit. A unit with rows but no keys has outputs all the same.
    __host__ __device__ __forceinline__ static int chunks(const Most& m, bool is_many, int n) {
        const UniformDiv& most = is_many ? m.many : m.few;
        return n <= most.d ? 1 : most(n - 1) + 1;
    }
    __host__ __device__ __forceinline__ static int items(const Most& m, int rows, int keys) {
        return tiles(rows) * chunks(m, rows > Shape::kMany, steps(rows, keys));
    }
    // Each lane's sums over its sequences: f(rows, keys, sums) adds to N of them, and nothing where both
    // are 0.
    template <int N, class F>
    __host__ __device__ __forceinline__ void sums(Int (&out)[N], F f) const {
        W::fill(out, rows0, keys0, [&](int lane, int rows, int keys, int (&x)[N]) {
            f(rows, keys, x);
            for (int j = 1; j < per && lane * per + j < a.B; ++j) {
                const PagedSeq s = seq(lane, j);
                f(s.rows, s.keys, x);
            }
        });
    }
    template <class F>
    __host__ __device__ __forceinline__ Int sum(F f) const {
        Int x[1];
        sums(x, [&](int rows, int keys, int* to) { to[0] += f(rows, keys); });
        return x[0];
    }
    // Among lane i's sequences, with f(rows, keys) places each, the one that has place `at`: its number, rows
    // and keys. `at` is left within it; `sum` gains g(rows, keys) of those before it.
    template <class F, class G>
    __host__ __device__ __forceinline__ PagedSeq place(int i, F f, G g, int& u, int& at,
                                                       int& sum) const {
        u = i * per;
        if (per == 1) return {W::lane(rows0, i), W::lane(keys0, i)};
        for (int j0 = 0;; j0 += 64) {
            auto here = [&](int lane) { return j0 + lane < per && u + j0 + lane < a.B; };
            const Int rows = W::each([&](int lane) { return here(lane) ? seq(i, j0 + lane).rows : 0; });
            const Int keys = W::each([&](int lane) { return here(lane) ? seq(i, j0 + lane).keys : 0; });
            const Int n = W::scan(W::map2(rows, keys, f)), m = W::scan(W::map2(rows, keys, g));
            if (at >= W::lane(n, 63) && j0 + 64 < per) {
                at -= W::lane(n, 63);
                sum += W::lane(m, 63);
                continue;
            }
            const int k = W::first(n, [&](int x) { return x > at; });
            if (k > 0) {
                at -= W::lane(n, k - 1);
                sum += W::lane(m, k - 1);
            }
            u += j0 + (k > 0 ? k : 0);
            return {W::lane(rows, k > 0 ? k : 0), W::lane(keys, k > 0 ? k : 0)};
        }
    }
    // Chunks that cost at most s.
    __host__ __device__ __forceinline__ Most at_most(int s) const {
        const int few_s = s / Shape::kRoundCost;
        return {UniformDiv(s > a.min_steps ? s : a.min_steps),
                UniformDiv(few_s > a.min_rounds ? few_s : a.min_rounds)};
    }

    __host__ __device__ __forceinline__ PagedPlan(const PagedArgs& args, const PagedSeq* in_lds,
                                                  bool are_staged)
        : a(args), seqs(in_lds), staged(are_staged), most{UniformDiv(1), UniformDiv(1)} {
        per = (a.B + 63) / 64;
        rows0 = W::each([&](int lane) { return lane * per < a.B ? seq(lane, 0).rows : 0; });
        keys0 = W::each([&](int lane) { return lane * per < a.B ? seq(lane, 0).keys : 0; });
        const int room = choose();
        for (int s = 0;; s = s ? 2 * s : most.many.d) {
            if (s) most = at_most(s);
            Int x[4];
            sums(x, [&](int rows, int keys, int* to) {
                const int n = items(most, rows, keys), slots = n > tiles(rows) ? n : 0;
                const bool is_many = rows > Shape::kMany;
                to[0] += is_many ? n : 0;
                to[1] += is_many ? 0 : n;
                to[2] += is_many ? slots : 0;
                to[3] += is_many ? 0 : slots;
            });
            many = W::scan(x[0]);
            few = W::scan(x[1]);
            many_slots = x[2];
            few_slots = x[3];
            // Only units whose work was cut off (choose) can leave more than there is room for.
            if (a.wgs == 0 || W::lane(many, 63) + W::lane(few, 63) <= room ||
                s > 1 << 28)
                return;
        }
    }

    // Sets the chunks; the room for items.
    __host__ __device__ __forceinline__ int choose() {
        if (a.wgs == 0) {
            most = at_most(kNoChunks);
            return 0;
        }
        // A lane's work, cut off where the sum would pass 2^30.
        const int cap = per > 64 ? (1 << 24) / per : 1 << 18;
        Int x[4];
        sums(x, [&](int rows, int keys, int* to) {
            const bool is_many = rows > Shape::kMany;
            const int n = tiles(rows);
            const float each = static_cast<float>(steps(rows, keys)) *
                               (is_many ? 1 : Shape::kRoundCost);
            const float cost = static_cast<float>(n) * each;
            to[0] += n;
            to[1] += cost > static_cast<float>(cap) ? cap : static_cast<int>(cost);
            to[2] += is_many ? n : 0;
            const int own = n == 0 ? 0 : each < 1e9f ? static_cast<int>(each) : 1000000000;
            to[3] = to[3] > own ? to[3] : own;
        });
        const int total = W::lane(W::scan(x[0]), 63);
        const float work = static_cast<float>(W::lane(W::scan(x[1]), 63));
        // Chunks of at most s: at most work / s + total items, on average work / s + total / 2. So
        // the least s that leaves no more than there is room for lies between work / room and
        // work / (room - total), rounded up (a round is not divided: the bound holds for multiples of
        // its cost). The least of four in between that does is taken.
        const int room = paged_room(total, a.wgs);
        auto over = [&](int items) {
            const float x = work / static_cast<float>(items);
            const int s = x < 1e9f ? static_cast<int>(x) + 1 : 1000000000;
            return s < Shape::kRoundCost ? Shape::kRoundCost : s;
        };
        const int lo = over(room), hi = over(room - total) + Shape::kRoundCost;
        if (total > 4 * a.wgs) {  // a few more or less are nothing beside so many
            most = at_most(hi);
            return room;
        }
        const Most m1 = at_most(lo + (hi - lo) / 4), m2 = at_most(lo + (hi - lo) / 2),
                   m3 = at_most(hi - (hi - lo) / 4);
        Int n[3];
        sums(n, [&](int rows, int keys, int* to) {
            to[0] += items(m1, rows, keys);
            to[1] += items(m2, rows, keys);
            to[2] += items(m3, rows, keys);
        });
        const int n1 = W::lane(W::scan(n[0]), 63), n2 = W::lane(W::scan(n[1]), 63),
                  n3 = W::lane(W::scan(n[2]), 63);
        most = n1 <= room ? m1 : n2 <= room ? m2 : n3 <= room ? m3 : at_most(hi);
        // Where the tiles run all at once and the longest takes no more steps than the rounds of chunks and
        // what these cost beside, there are no chunks. Of many rows: the partial results of as many tiles
        // as run at once are written, read and merged in the time of 16 steps, and a chunk's start and end
        // take that of 4 (bf16, us: 1000 tokens, 32 heads over 8, head_dim 128, 41 -> 36; 6 x 1024 tokens
        // of 12 heads, head_dim 64, 55 -> 42; 3000 tokens of 8 heads, head_dim 128, 70 without, 55 with).
        const int n_many = W::lane(W::scan(x[2]), 63);
        const int beside = n_many > 0 ? 4 + 16 * n_many / a.wgs : 1;
        const int rounds = room / a.wgs;
        if (total <= a.wgs &&
            W::most(x[3]) <= static_cast<int64_t>(rounds) * most.many.d + beside)
            most = at_most(kNoChunks);
        return room;
    }
};

// A unit's items in one launch: `first` is the slot of its first one, where it has several chunks; slot
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
    int slot;  // for its partial results, among those of its kind
    PagedUnit unit;
    PagedUnitItems of;  // the unit's items
};

// Tiles of a unit of many rows, or of few, that have more than `steps` steps or rounds: with a causal mask
// tile t of h rows sees the keys below len - n + min(n, ((t + 1) h - 1) / group + 1), so those from
// (kStep steps - len + n) group / h on.
template <class Shape>
__host__ __device__ __forceinline__ int longer_tiles(const PagedArgs& a, bool many, int rows,
                                                     int keys, int steps) {
    if ((rows > Shape::kMany) != many) return 0;
    const int height = many ? Shape::kTile : 32;
    const int tiles = static_cast<int>((static_cast<uint32_t>(rows) + (height - 1)) / height);
    if (steps < 0) return tiles;
    const int n = a.group_div(rows);
    const int64_t q = static_cast<int64_t>(steps) * (many ? Shape::kStep : Shape::kRound) - keys +
                      (a.causal ? n : 0);
    if (!a.causal) return q < 0 ? tiles : 0;
    if (q < 0) return tiles;
    if (q >= n) return 0;
    return tiles - static_cast<int>(q) * a.group / height;
}

// Tile x in the order of their steps, longest first, of the tiles of all units of many rows, or of few: the
// workgroups of a launch without chunks, where a long tile started last would run on alone (7 prompts of
// 285 to 2001 tokens, head_dim 64: 120.6 -> 114.9 us; 2 of 2048 and 4096, head_dim 32: 96.4 -> 88.0; fp32,
// 1024 + 700 tokens of 8 heads, head_dim 64: 44.5 -> 38.0; 6 of 400 tokens, where it only costs: 46.0 -> 47.9).
// The steps of the tile are the least s with no more than x longer tiles.
template <class Shape, class W>
__host__ __device__ __forceinline__ void tile_by_length(const PagedArgs& a,
                                                        const PagedPlan<Shape, W>& plan, int x,
                                                        PagedItem& r, int& keys, int& tile) {
    const bool many = r.many;
    auto longer = [&](int steps) {
        return W::lane(W::scan(plan.sum([&](int rows, int k) {
                           return longer_tiles<Shape>(a, many, rows, k, steps);
                       })),
                       63);
    };
    int lo = 0, hi = a.cap / (many ? Shape::kStep : Shape::kRound) + 1;
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (longer(mid) <= x)
            hi = mid;
        else
            lo = mid + 1;
    }
    // Its place among those of as many steps.
    int at = x - longer(lo);
    auto as_long = [&](int rows, int k) {
        return longer_tiles<Shape>(a, many, rows, k, lo - 1) -
               longer_tiles<Shape>(a, many, rows, k, lo);
    };
    const auto incl = W::scan(plan.sum(as_long));
    const int i = W::first(incl, [&](int n) { return n > at; });
    at -= i > 0 ? W::lane(incl, i > 0 ? i - 1 : 0) : 0;
    int none = 0;
    const PagedSeq s = plan.place(i, as_long, [](int, int) { return 0; }, r.u, at, none);
    r.rows = s.rows;
    keys = s.keys;
    tile = PagedPlan<Shape, W>::tiles(r.rows) -
           longer_tiles<Shape>(a, many, r.rows, keys, lo) - 1 - at;
}

template <class Shape, class W>
__host__ __device__ __forceinline__ PagedItem paged_item(const PagedArgs& a, int x,
                                                         const PagedSeq* seqs, bool staged) {
    PagedItem r{};
    const PagedPlan<Shape, W> plan(a, seqs, staged);
    using Plan = PagedPlan<Shape, W>;
    // Items of many rows come first: of sequences of like lengths they take longest.
    const int total_many = W::lane(plan.many, 63);
    if (x >= total_many + W::lane(plan.few, 63)) return r;
    r.many = x < total_many;
    if (!r.many) x -= total_many;
    int at = 0, keys = 0, by_length = -1, slot = 0;
    if (a.wgs == 0 && a.B > 1 && (r.many || plan.per == 1)) {
        tile_by_length<Shape, W>(a, plan, x, r, keys, by_length);
    } else {
        const auto& incl = r.many ? plan.many : plan.few;
        const int i = W::first(incl, [&](int n) { return n > x; });
        at = x - (i > 0 ? W::lane(incl, i > 0 ? i - 1 : 0) : 0);
        // Slots before the lane's units.
        if (a.wgs > 0) {
            const auto before = W::scan(r.many ? plan.many_slots : plan.few_slots);
            slot = i > 0 ? W::lane(before, i > 0 ? i - 1 : 0) : 0;
        }
        // The sequence among the lane's.
        auto own = [&](int rows, int n) {
            return (rows > Shape::kMany) == r.many ? Plan::items(plan.most, rows, n) : 0;
        };
        auto slots = [&](int rows, int n) {
            const int x = own(rows, n);
            return x > Plan::tiles(rows) ? x : 0;
        };
        const PagedSeq s = plan.place(i, own, slots, r.u, at, slot);
        r.rows = s.rows;
        keys = s.keys;
    }
    r.unit.n = a.group_div(r.rows);
    r.unit.t0 = paged_clamp(a.starts[r.u], 0, a.T);
    r.unit.kend = keys;
    r.of.first = slot;
    r.slot = slot + at;
    r.of.many = r.many;
    r.of.tiles = Plan::tiles(r.rows);
    int each = Plan::steps(r.rows, keys);
    r.of.chunks = Plan::chunks(plan.most, r.many, each);
    r.found = r.of.chunks == 1 ||
              slot + r.of.tiles * r.of.chunks <= (r.many ? a.max_many : a.max_few);
    const int chunk = r.of.chunks == 1 ? 0 : at / r.of.tiles;
    const int in = at - chunk * r.of.tiles;
    r.first = at == 0;
    const int tile = by_length >= 0 ? by_length : a.causal ? r.of.tiles - 1 - in : in;
    r.r0 = tile * (r.many ? Shape::kTile : 32);
    r.direct = r.of.chunks == 1;
    // (chunks - 1) each <= (chunks - 1) most < steps: the last chunk has keys as well.
    if (r.of.chunks > 1) each = (each + r.of.chunks - 1) / r.of.chunks;
    const int64_t len = static_cast<int64_t>(each) * (r.many ? Shape::kStep : Shape::kRound);
    const int64_t beg = chunk * len;
    r.kbeg = static_cast<int>(beg);
    r.kend = beg + len < r.unit.kend ? static_cast<int>(beg + len) : r.unit.kend;
    // With a causal mask, no further than the last row of the tile sees.
    if (a.causal) {
        const int last = (r.many ? Shape::kTile : 32) + r.r0;
        const int lim =
            paged_limit(a, r.u, r.unit, a.group_div((last < r.rows ? last : r.rows) - 1));
        if (lim < r.kend) r.kend = lim;
    }
    return r;
}

// Keys of each chunk of a sequence's own `keys` in a shared decode.
__host__ __device__ __forceinline__ int shared_own_len(const PagedArgs& a, int keys) {
    const uint32_t part = (static_cast<uint32_t>(keys) + (a.cut.own_chunks - 1)) / a.cut.own_chunks;
    const uint32_t len = (part + 31) / 32 * 32;
    return len > 0x7fffffe0u                                   ? 0x7fffffff
           : len > static_cast<uint32_t>(a.cut.own_least) ? static_cast<int>(len)
                                                          : a.cut.own_least;
}
// Chunks that a sequence's own `keys`, at least one, fill. (keys + len may pass 2^31.)
__host__ __device__ __forceinline__ int shared_own_parts(const PagedArgs& a, int keys) {
    return (keys - 1) / shared_own_len(a, keys) + 1;
}

// The sequence at place i of a batch of at most 64 in few chunks where one has more than 1024 own keys (512 in
// fp32): in the order of the lengths, longest first, every lane counting the sequences before its own (40
// sequences with 17 to 700 own keys in fp32 50.8 -> 48.5 us, 64 with 62 to 4000 101.7 -> 96.4). Shorter ones
// keep their order: the counting costs more than a late long sequence there (64 with 16 to 1024 40.0 -> 46.1).
template <class Shape, class W>
__host__ __device__ __forceinline__ int by_length(const PagedArgs& a, int i) {
    constexpr int kLong = std::min(1024, 4 * Shape::kRoundCost * Shape::kRound);
    const auto len = W::each([&](int lane) { return lane < a.B ? paged_seq_len(a, lane) : -1; });
    if (W::first(len, [&](int n) { return n > a.prefix && n - a.prefix > kLong; }) < 0)
        return i;
    auto place = W::each([](int) { return 0; });
    for (int b = 0; b < a.B; ++b) {
        const int other = W::lane(len, b);
        place = W::map3(len, place, [&](int lane, int own, int n) {
            return n + (other > own || (other == own && b < lane));
        });
    }
    return W::first(W::map3(len, place, [&](int lane, int, int n) { return lane < a.B ? n : -1; }),
                    [&](int n) { return n == i; });
}

// Item x of a shared decode. Its slot among those of its kind: unit 0's come first, and those of sequence
// b stand at b's place, also where the items run in the order of lengths.
template <class Shape, class W>
__host__ __device__ __forceinline__ PagedItem shared_item(const PagedArgs& a, int x) {
    PagedItem r{};
    const SharedCut& c = a.cut;
    const int pre = c.pre_tiles * c.pre_chunks;
    r.slot = x;
    int chunk, tile, len;
    if (x < pre) {
        r.many = c.pre_many;
        r.rows = a.B * a.group;
        chunk = c.pre_tiles_div(x);
        tile = x - chunk * c.pre_tiles;
        len = c.pre_len;
        r.of.tiles = c.pre_tiles;
    } else {
        x -= pre;
        if (x >= a.B * c.own_chunks * c.own_tiles) return r;
        r.many = c.own_many;
        r.rows = a.group;
        int b = c.own_items_div(x);
        x -= b * c.own_chunks * c.own_tiles;
        if (a.B <= 64 && c.own_chunks <= 4) b = by_length<Shape, W>(a, b);
        r.slot = (c.own_many == c.pre_many ? pre : 0) + b * c.own_chunks * c.own_tiles + x;
        chunk = c.own_tiles_div(x);
        tile = x - chunk * c.own_tiles;
        r.u = b + 1;
        r.of.tiles = c.own_tiles;
    }
    r.found = true;
    r.unit = paged_unit(a, r.u);
    if (r.u > 0) len = shared_own_len(a, r.unit.kend - r.unit.kbeg);
    r.r0 = tile * (r.many ? Shape::kTile : 32);
    const int64_t beg = r.unit.kbeg + static_cast<int64_t>(chunk) * len;
    r.kbeg = beg < r.unit.kend ? static_cast<int>(beg) : r.unit.kend;
    r.kend = beg + len < r.unit.kend ? static_cast<int>(beg + len) : r.unit.kend;
    return r;
}

// The cut, for `wgs` workgroups per key/value head at once: unit 0 in items for three of four of them (the
// others start on own keys), of at least min_steps steps or one round; own keys in chunks where the tiles of
// all sequences leave workgroups free, or fill them at most twice: so a long sequence among short ones ends
// sooner (bf16, 32 heads over 8, head_dim 128, us: 8 sequences with up to 8000 own keys 39.6 -> 34.5, 32 with
// up to 3000 50.5 -> 45.2, 64 with up to 4000 112 -> 102; but 40 with up to 500 24.2 -> 24.3, 96 of 4
// key/value heads 27.0 -> 28.3). No more than 16 for that: 4 sequences with up to 200 own keys 11.2 -> 12.0
// with 32.
template <class Shape>
inline SharedCut shared_cut(int B, int group, int prefix, int wgs, int min_steps) {
    SharedCut c{};
    auto tiles = [](long long rows) {
        return static_cast<int>(rows > Shape::kMany ? (rows + Shape::kTile - 1) / Shape::kTile
                                                 : (rows + 31) / 32);
    };
    auto ceil_div = [](long long x, long long by) { return (x + by - 1) / by; };
    const long long rows = static_cast<long long>(B) * group;
    c.pre_many = rows > Shape::kMany;
    c.own_many = group > Shape::kMany;
    c.pre_tiles = tiles(rows);
    c.own_tiles = tiles(group);
    const int unit = c.pre_many ? Shape::kStep : Shape::kRound;
    const long long steps = ceil_div(prefix, unit);
    const long long chunks =
        std::max(1LL, std::min<long long>(ceil_div(3LL * wgs, 4LL * c.pre_tiles),
                                          steps / (c.pre_many ? min_steps : 1)));
    const long long each = std::max(1LL, ceil_div(steps, chunks));
    c.pre_chunks = prefix > 0 ? static_cast<int>(ceil_div(steps, each)) : 0;
    c.pre_len = static_cast<int>(std::min<long long>(each * unit, 0x7fffffffLL));
    const long long own = static_cast<long long>(B) * c.own_tiles;
    c.own_chunks = static_cast<int>(
        std::max({1LL, std::min<long long>(64, wgs / own), std::min<long long>(16, 2LL * wgs / own)}));
    c.own_least = c.own_many ? Shape::kStep * min_steps : Shape::kRound;
    c.pre_tiles_div = fast_div(c.pre_tiles);
    c.own_tiles_div = fast_div(c.own_tiles);
    c.own_items_div = fast_div(c.own_chunks * c.own_tiles);
    return c;
}

// Row of `acc` and `ml` that row r of a slot has.
template <class Shape>
__host__ __device__ __forceinline__ size_t paged_slot_row(const PagedArgs& a, int hk, bool many,
                                                          int slot, int r) {
    if (many)
        return (static_cast<size_t>(hk) * a.max_many + slot) * Shape::kTile + r;
    return static_cast<size_t>(a.Hkv) * a.max_many * Shape::kTile +
           (static_cast<size_t>(hk) * a.max_few + slot) * a.few_rows + r;
}

// What the host knows of a forward: the tiles, of many rows and in all, that `units` sequences with
// `tokens` tokens in all can have at most.
struct PagedTiles {
    long long many, all;
};
template <class Shape>
inline PagedTiles paged_tiles(long long tokens, long long units, int group) {
    const long long rows = tokens * group;
    const long long with = std::min(units, tokens);  // sequences that have tokens
    const long long big = std::min(rows / (Shape::kMany + 1LL), with);
    const long long few = (Shape::kMany + 31LL) / 32;  // most tiles of a unit of few rows
    return {big ? rows / Shape::kTile + big : 0,
            std::min(rows / 32 + with, few * with + (big ? rows / Shape::kTile : 0))};
}

}  // namespace dev
}  // namespace cuflash
