// The cut of an attention over an 8-bit paged cache into waves (cuflash-attn_amd/csrc/paged_q8_plan.hpp)
// on the host: the code that the kernels run, over random launches, tokens and lengths. No GPU call is made.
//
// Checked for each launch: every grain of keys of every tile of rows is met by one wave, no wave goes beyond
// its share, a partial result's slot is its own, and the merge finds exactly the parts that were left, whole
// tiles being found as whole. Arguments: the number of launches, the seed.

#include <algorithm>
#include <array>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <tuple>
#include <vector>

#include "paged_q8_plan.hpp"

namespace {

using namespace cuflash::dev;

struct HostWave {
    using Int = std::array<int, 64>;
    template <class F>
    static Int each(F f) {
        Int v;
        for (int i = 0; i < 64; ++i) v[i] = f(i);
        return v;
    }
    static Int scan(Int v) {
        for (int i = 0; i < 64; ++i)
            if (v[i] < 0 || (i && __builtin_add_overflow(v[i], v[i - 1], &v[i]))) std::abort();
        return v;
    }
    static int lane(const Int& v, int i) {
        if (i < 0 || i >= 64) std::abort();
        return v[i];
    }
    template <class F>
    static int first(const Int& v, F f) {
        for (int i = 0; i < 64; ++i)
            if (f(v[i])) return i;
        return -1;
    }
};

int g_case = 0;
#define CHECK(cond)                                                            \
    do {                                                                       \
        if (!(cond)) {                                                         \
            std::printf("launch %d, line %d: %s\n", g_case, __LINE__, #cond); \
            std::exit(1);                                                      \
        }                                                                      \
    } while (0)

int spread(std::mt19937& rng, int lo, int hi) {  // over the logarithm
    std::uniform_real_distribution<double> u(std::log(double(lo)), std::log(double(hi) + 1.0));
    return std::min(hi, std::max(lo, int(std::exp(u(rng)))));
}

template <int R>
bool launch(std::mt19937& rng) {  // whether a tile was cut
    auto pick = [&](int n) { return int(rng() % unsigned(n)); };
    Q8PlanArgs a{};
    a.group = std::array<int, 7>{1, 2, 3, 4, 8, 16, 40}[pick(7)];
    a.group_div = fast_div(a.group);
    a.causal = pick(2);
    const bool far = pick(10) == 0;  // keys up to the limit
    a.B = far ? 1 + pick(3) : std::array<int, 6>{1, 2, 7, 64, 65, 200}[pick(6)];
    a.cap = far ? 0x7fffffff - 1023 : spread(rng, 1, a.B > 10 ? 500 : 5000);
    a.shares = spread(rng, 1, 2048);
    a.least = 1 + pick(3) * pick(4);
    const bool decode = pick(3) == 0;
    std::vector<int> lens, starts{0};
    const int most = far ? 6 : spread(rng, 1, a.B > 10 ? 20 : 300);
    for (int b = 0; b < a.B; ++b) {
        const int n = pick(8) == 0 ? 0 : 1 + pick(most);
        starts.push_back(starts.back() + n);
        lens.push_back(pick(9) == 0 ? 0 : far ? a.cap - pick(1000) : 1 + pick(a.cap + 3) - pick(2));
    }
    a.seq_lens = lens.data();
    a.starts = decode ? nullptr : starts.data();
    a.T = decode ? a.B : std::max(1, starts.back() + (pick(4) == 0 ? 5 : 0) - (pick(6) == 0 ? 1 : 0));
    const int least = R == 256 ? 1 : pick(5) == 0 ? 1 + pick(2) : 0;
    q8_set_grains(a, R, least);
    CHECK(far || a.shift == least);

    const Q8Total total = q8_total<R, HostWave>(a);
    int sum = 0;
    for (int b = 0; b < a.B; ++b) {
        CHECK((q8_begin_of<R, HostWave>(a, b) == sum));
        sum += Q8Line<R>(a, q8_seq(a, b)).size;
    }
    CHECK(sum == total.grains && sum < kQ8Line);
    CHECK(static_cast<long long>(total.share) * a.shares >= sum);

    using Key = std::tuple<int, int>;  // sequence, tile
    std::map<Key, std::vector<std::array<int, 4>>> met;  // kbeg, kend, wave, slot
    bool cut = false;
    for (int p = 0; p < a.shares; ++p) {
        Q8Walk<R, HostWave> walk(a, p);
        Q8Segment s;
        int grains = 0, steps = 0;
        std::array<bool, 2> used{};
        while (walk.next(a, s)) {
            CHECK(++steps <= total.share);
            CHECK(s.b >= 0 && s.b < a.B && s.r0 >= 0 && s.r0 % R == 0 && s.r0 < s.rows);
            const Q8Seq q = q8_seq(a, s.b);
            CHECK(q.t0 == s.seq.t0 && q.n == s.seq.n && s.rows == q.n * a.group);
            CHECK(s.kbeg >= 0 && s.kbeg < s.kend && s.kend <= q.keys && s.kbeg % 32 == 0);
            grains += (s.kend - s.kbeg - 1) / (32 << a.shift) + 1;
            if (s.slot >= 0) {
                CHECK(s.slot < 2 && !used[s.slot] && (s.slot == 0 || p < a.shares - 1));
                used[s.slot] = true;
                cut = true;
            }
            met[{s.b, s.r0 / R}].push_back({s.kbeg, s.kend, p, s.slot});
        }
        CHECK(grains <= total.share);
    }
    int tiles = 0;
    for (int b = 0; b < a.B; ++b) {
        const Q8Seq q = q8_seq(a, b);
        const Q8Line<R> line(a, q);
        // A workgroup a tile: the tiles in their order, and none behind them.
        for (int tile = 0; tile < line.tiles; ++tile, ++tiles) {
            int at_b = -1, at = -1;
            CHECK((q8_tile_at<R, HostWave>(a, tiles, at_b, at)) && at_b == b && at == tile);
        }
        CHECK(line.tiles == (q.n * a.group + R - 1) / R);
        const int without = q8_rows_without_keys<R>(a, q);
        for (int tile = 0; tile < line.tiles; ++tile) {
            CHECK((line.keys(a, q, tile) == 0) == (tile * R < without));
            // The keys that some row of the tile sees.
            int keys = 0;
            for (int r = tile * R; r < std::min((tile + 1) * R, line.rows); ++r)
                keys = std::max(keys, q8_limit(a, q, r / a.group));
            CHECK(keys == line.keys(a, q, tile));
            const Q8Parts parts =
                q8_parts(a, total, q8_begin_of<R, HostWave>(a, b) + line.begin(a, q, tile),
                         Q8Line<R>::grains(a, keys));
            const auto& got = met[{b, tile}];  // in the order of the waves
            CHECK(int(got.size()) == parts.to - parts.from + 1);
            int at = 0;
            for (size_t i = 0; i < got.size(); ++i) {
                CHECK(got[i][0] == at);
                at = got[i][1];
                CHECK(got[i][2] == parts.from + int(i));
                CHECK(got[i][3] == (got.size() == 1 ? -1 : i == 0 ? parts.slot : 0));
            }
            CHECK(at == keys);
            // The merge by shares finds a cut tile from the share that it begins in.
            if (got.size() > 1) {
                const int end = std::min((parts.from + 1) * total.share, total.grains);
                int first = 0, in = 0, grain = 0;
                CHECK((q8_sequence_at<R, HostWave>(a, end - 1, first) == b));
                CHECK(line.find(a, q, end - 1 - first, in, grain) && in == tile);
                CHECK(end - 1 - grain == first + line.begin(a, q, tile));
            }
        }
    }
    int none_b, none;
    CHECK(!(q8_tile_at<R, HostWave>(a, tiles, none_b, none)) && tiles <= q8_most_tiles(a, R));
    return cut;
}

// Starts that decrease: every wave ends, and stays inside the tensors.
template <int R>
void disorder(std::mt19937& rng) {
    auto pick = [&](int n) { return int(rng() % unsigned(n)); };
    Q8PlanArgs a{};
    a.group = 1 + pick(8);
    a.group_div = fast_div(a.group);
    a.causal = pick(2);
    a.B = 1 + pick(6);
    a.cap = 1 + pick(3000);
    a.T = 1 + pick(40);
    a.shares = 1 + pick(600);
    a.least = 1 + pick(3);
    std::vector<int> lens, starts;
    for (int b = 0; b <= a.B; ++b) {
        lens.push_back(pick(2 * a.cap) - 5);
        starts.push_back(pick(2 * a.T) - 5);
    }
    a.seq_lens = lens.data();
    a.starts = starts.data();
    q8_set_grains(a, R, R == 256 ? 1 : 0);
    for (int x = 0; x < q8_most_tiles(a, R); ++x) {
        int b, tile;
        if (!q8_tile_at<R, HostWave>(a, x, b, tile)) break;
        const Q8Seq s = q8_seq(a, b);
        const Q8Line<R> line(a, s);
        CHECK(b >= 0 && b < a.B && tile >= 0 && tile < line.tiles && s.t0 + s.n <= a.T);
        CHECK(line.keys(a, s, tile) >= 0 && line.keys(a, s, tile) <= a.cap);
    }
    const Q8Total total = q8_total<R, HostWave>(a);
    for (int p = 0; p < a.shares; ++p) {
        Q8Walk<R, HostWave> walk(a, p);
        Q8Segment s;
        int steps = 0;
        while (walk.next(a, s)) {
            CHECK(++steps <= total.share);
            CHECK(s.seq.t0 >= 0 && s.seq.t0 + s.seq.n <= a.T && s.r0 < s.rows);
            CHECK(s.kbeg >= 0 && s.kbeg < s.kend && s.kend <= a.cap && s.slot < 2);
        }
    }
}

}  // namespace

int main(int argc, char** argv) {
    const int launches = argc > 1 ? std::atoi(argv[1]) : 1000;
    std::mt19937 rng(argc > 2 ? std::atoi(argv[2]) : 1);
    int cut = 0;
    for (g_case = 0; g_case < launches; ++g_case) {
        const int kind = g_case % 3;
        cut += kind == 0 ? launch<16>(rng) : kind == 1 ? launch<32>(rng) : launch<256>(rng);
        kind == 0 ? disorder<32>(rng) : kind == 1 ? disorder<16>(rng) : disorder<256>(rng);
    }
    CHECK(cut > launches / 3);
    std::printf("%d launches, %d with tiles that several waves have\n", launches, cut);
    return 0;
}
