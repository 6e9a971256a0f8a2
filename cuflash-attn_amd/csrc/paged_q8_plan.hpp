#pragma once

// How the attention over an 8-bit paged cache is cut into the parts that waves take. How many tokens and
// keys a sequence has is known on the device only, so every wave finds its part by itself, from the
// same sums over the sequences. Everything that becomes an address or a loop bound is formed here, in code
// that also compiles for the host, where tests/cpp/test_paged_q8_plan.cpp runs it.
//
// The query heads of one key/value head are the rows of a sequence (row r: token r / group, head r %
// group), in tiles of R rows; keys come in grains of 32 << shift. All grains of all tiles stand in one
// line, and wave p of `shares` waves per key/value head takes an equal piece of it, from p share on. So no
// wave has more to do than another, whatever the lengths; a tile that several waves have is merged afterwards,
// from at most two partial results a wave: of the tile that it begins in (slot 0) and, where it reaches
// another that it does not finish, of that (slot 1).
// With a causal mask a later tile sees more keys. Tiles stand in pairs in the line, the first with the last,
// the second with the last but one, so that every pair has as many grains, and where a pair begins is a
// product. (With f(e) = max(0, keys - n + e), convex, and e_i <= (i + 1) R / group + 1 tokens up to tile i, a
// pair has at most f(e_first) + f(e_last) + R / group + 2 keys, and so, in grains of g keys, at most
// 2 + floor(R / (group g)) more than the first pair: the `slack`.)

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "paged_plan.hpp"

namespace cuflash {
namespace dev {

struct Q8PlanArgs {
    const int* seq_lens;  // [B]
    const int* starts;    // [B + 1]; null: one token per sequence
    int B, T, group, cap;
    int shares;  // waves per key/value head
    int shift;   // a grain has 32 << shift keys
    int slack;   // grains between pairs
    int least;   // grains of a share, where there are that many
    bool causal;
    FastDiv group_div;
};

// A sequence's tokens and keys.
struct Q8Seq {
    int t0, n, keys;
};
__host__ __device__ __forceinline__ Q8Seq q8_seq(const Q8PlanArgs& a, int b) {
    const int keys = paged_clamp(a.seq_lens[b], 0, a.cap);
    if (!a.starts) return {b, 1, keys};
    const int t0 = paged_clamp(a.starts[b], 0, a.T);
    return {t0, paged_clamp(a.starts[b + 1], t0, a.T) - t0, keys};
}
// Keys that token i of a sequence sees.
__host__ __device__ __forceinline__ int q8_limit(const Q8PlanArgs& a, const Q8Seq& s, int i) {
    if (!a.causal) return s.keys;
    const int lim = s.keys - s.n + i + 1;
    return lim > 0 ? lim : 0;
}

constexpr int kQ8Line = 1 << 30;  // grains of a line, and waves of a launch, are fewer

// The tiles of a sequence in the line.
template <int R>
struct Q8Line {
    int rows, tiles;
    int pairs;  // the last of them may have one tile; without a mask every one has
    int pair;   // grains from pair to pair
    int size;   // in all
    __host__ __device__ __forceinline__ Q8Line(const Q8PlanArgs& a, const Q8Seq& s) {
        rows = s.n * a.group;
        tiles = tiles_of(a, s);
        const int last = tiles > 0 ? grains(a, keys(a, s, tiles - 1)) : 0;
        if (!a.causal || tiles <= 1) {
            pairs = tiles;
            pair = last;
            size = pairs * pair;
        } else {
            pairs = tiles / 2;
            pair = grains(a, keys(a, s, 0)) + last + a.slack;
            size = pairs * pair;
            if (tiles % 2) size += grains(a, keys(a, s, pairs++));
        }
    }
    __host__ __device__ __forceinline__ static int tiles_of(const Q8PlanArgs& a, const Q8Seq& s) {
        return static_cast<int>((static_cast<uint32_t>(s.n * a.group) + (R - 1)) / R);
    }
    // Keys that the rows of a tile see, and their grains.
    __host__ __device__ __forceinline__ int keys(const Q8PlanArgs& a, const Q8Seq& s, int tile) const {
        const int end = tile < tiles - 1 ? (tile + 1) * R : rows;
        return q8_limit(a, s, a.group_div(end - 1));
    }
    __host__ __device__ __forceinline__ static int grains(const Q8PlanArgs& a, int keys) {
        return static_cast<int>((static_cast<uint32_t>(keys) + ((32u << a.shift) - 1)) >>
                                (5 + a.shift));
    }
    // Where tile begins, among the sequence's grains.
    __host__ __device__ __forceinline__ int begin(const Q8PlanArgs& a, const Q8Seq& s, int tile) const {
        const int other = tiles - 1 - tile;
        if (tile < pairs) return tile * pair;
        return other * pair + grains(a, keys(a, s, other));
    }
    // The tile at place x (0 <= x < size) of the sequence's grains and the grain in it; false: none, up to
    // the next pair.
    __host__ __device__ __forceinline__ bool find(const Q8PlanArgs& a, const Q8Seq& s, int x, int& tile,
                                                  int& grain) const {
        tile = x / pair;
        grain = x - tile * pair;
        const int n = grains(a, keys(a, s, tile));
        if (grain < n) return true;
        const int other = tiles - 1 - tile;
        if (other < pairs) return false;
        grain -= n;
        tile = other;
        return grain < grains(a, keys(a, s, tile));
    }
};

// Sums over the sequences, W: the 64 lanes of a wave. Of sequences b0 + lane, in units of 1 << shift.
template <int R, class W>
__host__ __device__ __forceinline__ typename W::Int q8_sizes(const Q8PlanArgs& a, int b0, int shift = 0) {
    return W::each([&](int lane) {
        if (b0 + lane >= a.B) return 0;
        return Q8Line<R>(a, q8_seq(a, b0 + lane)).size >> shift;
    });
}

// Grains of the whole line, and of a wave's share.
struct Q8Total {
    int grains, share;
};
template <int R, class W>
__host__ __device__ __forceinline__ Q8Total q8_total(const Q8PlanArgs& a) {
    int sum = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const auto sizes = q8_sizes<R, W>(a, b0);
        // Only starts that decrease lead past what q8_set_grains() leaves room for. What comes out then is undefined,
        // but the shares of a sum that wrapped would reach beyond the rows and the workspace. A size is at most the
        // line; where 64 of them may pass 32 bits, they are first summed in units of 64.
        if (W::first(sizes, [](int n) { return n > kQ8Line / 64; }) >= 0 &&
            W::lane(W::scan(q8_sizes<R, W>(a, b0, 6)), 63) > kQ8Line / 64)
            return {0, a.least};
        const int block = W::lane(W::scan(sizes), 63);
        if (block > kQ8Line - sum) return {0, a.least};
        sum += block;
    }
    const int share = (sum + (a.shares - 1)) / a.shares;
    return {sum, share > a.least ? share : a.least};
}

// The sequence that has place x of the line (x < total), and where it begins.
template <int R, class W>
__host__ __device__ __forceinline__ int q8_sequence_at(const Q8PlanArgs& a, int x, int& begin) {
    begin = 0;
    for (int b0 = 0;; b0 += 64) {
        const auto incl = W::scan(q8_sizes<R, W>(a, b0));
        const int i = W::first(incl, [&](int n) { return n > x - begin; });
        if (i >= 0 || b0 + 64 >= a.B) {
            const int k = i > 0 ? i : 0;
            if (k > 0) begin += W::lane(incl, k - 1);
            return b0 + k;
        }
        begin += W::lane(incl, 63);
    }
}
// Where sequence b begins in the line.
template <int R, class W>
__host__ __device__ __forceinline__ int q8_begin_of(const Q8PlanArgs& a, int b) {
    int begin = 0;
    for (int b0 = 0; b0 < b; b0 += 64) {
        const auto incl = W::scan(q8_sizes<R, W>(a, b0));
        begin += W::lane(incl, b - b0 < 64 ? b - b0 - 1 : 63);
    }
    return begin;
}

// Where one launch does everything, a workgroup has a tile: tile x of all sequences', in their order; false: there
// are fewer.
template <int R, class W>
__host__ __device__ __forceinline__ bool q8_tile_at(const Q8PlanArgs& a, int x, int& b, int& tile) {
    if (!a.starts) {
        const int each = static_cast<int>((static_cast<uint32_t>(a.group) + (R - 1)) / R);
        b = x / each;
        tile = x - b * each;
        return b < a.B;
    }
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const auto incl = W::scan(W::each([&](int lane) {
            return b0 + lane < a.B ? Q8Line<R>::tiles_of(a, q8_seq(a, b0 + lane)) : 0;
        }));
        const int i = W::first(incl, [&](int n) { return n > x; });
        if (i >= 0) {
            b = b0 + i;
            tile = x - (i > 0 ? W::lane(incl, i - 1) : 0);
            return true;
        }
        x -= W::lane(incl, 63);
    }
    return false;
}
// No launch has more of them.
inline long long q8_most_tiles(const Q8PlanArgs& a, int rows_per_tile) {
    if (!a.starts) return static_cast<long long>(a.B) * ((a.group + rows_per_tile - 1) / rows_per_tile);
    return static_cast<long long>(a.T) * a.group / rows_per_tile + a.B;
}

// The part of a wave: tile by tile, rows from r0 on of sequence b over its keys [kbeg, kend).
struct Q8Segment {
    Q8Seq seq;
    int b, rows, r0;
    int kbeg, kend;
    int slot;  // of the partial result; -1: the whole tile
};
template <int R, class W>
struct Q8Walk {
    int x, begin, end;  // places of the line
    int b, first;       // the sequence at x, and where it begins
    __host__ __device__ __forceinline__ Q8Walk(const Q8PlanArgs& a, int p) {
        const Q8Total total = q8_total<R, W>(a);
        x = begin = p * total.share;
        end = total.grains - begin < total.share ? total.grains : begin + total.share;
        b = first = 0;
        if (begin < end) b = q8_sequence_at<R, W>(a, begin, first);
    }
    __host__ __device__ __forceinline__ bool next(const Q8PlanArgs& a, Q8Segment& to) {
        while (x < end && b < a.B) {
            const Q8Seq s = q8_seq(a, b);
            const Q8Line<R> line(a, s);
            const int in = x - first;
            if (in >= line.size) {
                first += line.size;
                ++b;
                continue;
            }
            int tile, grain;
            if (!line.find(a, s, in, tile, grain)) {
                const int pair = (in / line.pair + 1) * line.pair;
                x = first + (pair < line.size ? pair : line.size);
                continue;
            }
            const int keys = line.keys(a, s, tile);
            const int grains = Q8Line<R>::grains(a, keys);
            const int take = grains - grain < end - x ? grains - grain : end - x;
            const int64_t kend = static_cast<int64_t>(grain + take) << (5 + a.shift);
            to.seq = s;
            to.b = b;
            to.rows = line.rows;
            to.r0 = tile * R;
            to.kbeg = grain << (5 + a.shift);
            to.kend = kend < keys ? static_cast<int>(kend) : keys;
            to.slot = take == grains ? -1 : grain == 0 && x > begin ? 1 : 0;
            x += take;
            return true;
        }
        return false;
    }
};

// Rows of a sequence that lie in tiles without a key: the first ones.
template <int R>
__host__ __device__ __forceinline__ int q8_rows_without_keys(const Q8PlanArgs& a, const Q8Seq& s) {
    if (s.keys == 0) return s.n * a.group;
    if (!a.causal || s.n <= s.keys) return 0;
    return (s.n - s.keys) * a.group / R * R;
}

// The waves that have a part of a tile, `from` .. `to`, and the slot of wave `from`'s; from > to: the tile
// has no keys (or, with starts that decrease, no wave).
struct Q8Parts {
    int from, to, slot;
};
__host__ __device__ __forceinline__ Q8Parts q8_parts(const Q8PlanArgs& a, const Q8Total& total, int begin,
                                                     int grains) {
    if (grains == 0 || begin < 0 || begin > kQ8Line) return {0, -1, 0};
    const int from = begin / total.share, to = (begin + grains - 1) / total.share;
    if (to >= a.shares) return {0, -1, 0};
    return {from, to, begin > from * total.share ? 1 : 0};
}

// The grains of a launch, of 32 << least keys or more, so that by what the host knows the line has less than 2^30 of
// them. With the largest, of 2^31 keys, a tile is one grain, and between pairs of tiles, of which a sequence of r rows
// has at most r / R, stand `slack` more. false: more than 2^30 even so, or so many sequences that their number, 64 at
// a time, passes 32 bits.
inline bool q8_set_grains(Q8PlanArgs& a, int rows_per_tile, int least) {
    const long long full = static_cast<long long>(a.T) * a.group / rows_per_tile;
    if (a.B > 0x7fffffff - 63) return false;
    for (a.shift = least;; ++a.shift) {
        a.slack = 2 + static_cast<int>(rows_per_tile / (static_cast<long long>(a.group) << (5 + a.shift)));
        if ((full + 2LL * a.B) * (((a.cap + 31LL) / 32 >> a.shift) + 1 + a.slack) < kQ8Line) return true;
        if (a.shift >= 26) break;
    }
    if (!a.starts) return q8_most_tiles(a, rows_per_tile) <= kQ8Line;
    return full * (1 + (a.causal ? a.slack : 0)) + (a.B < a.T ? a.B : a.T) <= kQ8Line;
}

}  // namespace dev
}  // namespace cuflash
