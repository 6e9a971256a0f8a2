// The cut of a paged attention into workgroups (cuflash-attn_amd/csrc/paged_plan.hpp) on the host: the
// code that the kernels run, over random launches, tokens and lengths, with every index that becomes an
// address checked against the array it goes to. No GPU call is made.
//
// Checked for each launch: every row of every unit meets every key it sees in exactly one item; items
// are numbered below the grid and partial results below the slots; direct items are the only ones of
// their rows; the combine finds the slot that an item wrote; items of causal tiles end where their last
// row's keys do; fast_div divides.
//
// Arguments: the number of launches, the seed.

#include <algorithm>
#include <array>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <vector>

#include "paged_plan.hpp"

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
    template <class F>
    static Int map3(const Int& x, const Int& y, F f) {
        return each([&](int i) { return f(i, x[i], y[i]); });
    }
    template <class F>
    static Int map2(const Int& x, const Int& y, F f) {
        return each([&](int i) { return f(x[i], y[i]); });
    }
    template <int N, class F>
    static void fill(Int (&out)[N], const Int& x, const Int& y, F f) {
        for (int i = 0; i < 64; ++i) {
            int sums[N] = {};
            f(i, x[i], y[i], sums);
            for (int j = 0; j < N; ++j) out[j][i] = sums[j];
        }
    }
    static Int scan(Int v) {
        for (int i = 1; i < 64; ++i) {
            if (v[i] < 0 || __builtin_add_overflow(v[i], v[i - 1], &v[i])) std::abort();
        }
        return v;
    }
    static int most(const Int& v) { return std::max(0, *std::max_element(v.begin(), v.end())); }
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

template <class Shape, bool kShared>
bool launch(std::mt19937& rng) {  // whether something was cut into chunks
    auto pick = [&](int n) { return int(rng() % unsigned(n)); };
    PagedArgs a{};
    a.Hkv = std::array<int, 4>{1, 2, 8, 12}[pick(4)];
    a.group = std::array<int, 6>{1, 2, 3, 4, 8, 40}[pick(6)];
    a.H = a.Hkv * a.group;
    a.group_div = fast_div(a.group);
    a.page_size = std::array<int, 6>{1, 6, 16, 24, 64, 256}[pick(6)];
    a.page_div = fast_div(a.page_size);
    a.B = spread(rng, 1, pick(300) == 0 ? 6000 : pick(10) == 0 ? 600 : 200);
    a.max_pages = spread(rng, 1, std::max(1, 40000 / a.page_size));
    a.cap = a.page_size * a.max_pages;
    a.shared = kShared;
    a.causal = !a.shared && pick(3) > 0;
    a.min_steps = 1 + pick(8);
    a.min_rounds = 1 + pick(2);
    std::vector<int> lens(a.B), starts(a.B + 1);
    const int most = spread(rng, 1, a.shared ? 1 : 3000);
    const int kind = pick(4);
    for (int b = 0; b < a.B; ++b) {
        const int n = a.shared ? 1 : kind == 0 ? pick(2) : kind == 1 ? (b == 0 ? most : 1)
                                                         : pick(most + 1);
        starts[b + 1] = starts[b] + n;
        lens[b] = pick(5) == 0 ? pick(40) : spread(rng, 1, a.cap);
        if (pick(3) > 0) lens[b] = std::max(lens[b], n);
        if (pick(20) == 0) lens[b] = -pick(9);
        if (pick(20) == 0) lens[b] = a.cap + pick(1000);
    }
    a.T = starts[a.B];
    if (a.T == 0) return false;
    if (!a.shared && pick(4) == 0) a.T += pick(50);        // padding
    if (!a.shared && pick(8) == 0) a.T = std::max(1, a.T - pick(50));  // starts past the tokens
    a.seq_lens = lens.data();
    a.starts = starts.data();
    a.prefix = a.shared && rng() % 8 ? spread(rng, 1, a.cap) : 0;

    // As the workgroups put them into LDS.
    const bool staged = !a.shared && pick(4) != 0;
    const int per = (a.B + 63) / 64;
    std::vector<PagedSeq> seqs(staged ? 64 * (per + 1) : 0, PagedSeq{1 << 20, 1 << 20});
    for (int b = 0; staged && b < a.B; ++b) seqs[b / per * (per + 1) + b % per] = paged_seq(a, b);

    PagedTiles t{};
    int items, room;
    if constexpr (kShared) {
        a.wgs = spread(rng, 1, 300);
        a.cut = shared_cut<Shape>(a.B, a.group, a.prefix, a.wgs, a.min_steps);
        const SharedCut& c = a.cut;
        const int pre = c.pre_tiles * c.pre_chunks, own = a.B * c.own_chunks * c.own_tiles;
        CHECK(c.pre_len > 0 && int64_t(c.pre_len) * c.pre_chunks >= a.prefix);
        CHECK(int64_t(c.pre_len) * (c.pre_chunks - 1) < a.prefix);
        a.max_many = (c.pre_many ? pre : 0) + (c.own_many ? own : 0);
        a.max_few = pre + own - a.max_many;
        a.few_rows = c.pre_many && !c.own_many && c.own_tiles == 1 ? a.group : 32;
        items = room = pre + own;
        // The workspace's bound, for any prefix.
        const SharedCut most = shared_cut<Shape>(a.B, a.group, 1 << 30, a.wgs, a.min_steps);
        CHECK(c.pre_chunks <= most.pre_chunks && c.own_chunks == most.own_chunks);
    } else {
        t = paged_tiles<Shape>(a.T, a.B, a.group);
        a.wgs = pick(4) == 0 ? 0 : spread(rng, 1, 300);
        room = a.wgs ? paged_room(int(t.all), a.wgs) : int(t.all);
        a.max_few = a.wgs ? std::min(room, 3 * a.wgs) : 0;
        a.max_many = t.many > 0 ? int(std::min<long long>(a.max_few, t.many + 2LL * a.wgs)) : 0;
        a.few_rows = 32;
        const PagedPlan<Shape, HostWave> plan(a, nullptr, false);
        items = HostWave::lane(plan.many, 63) + HostWave::lane(plan.few, 63);
    }
    CHECK(items <= room);
    const int units = a.shared ? a.B + 1 : a.B;
    std::vector<int4> noted(units, make_int4(-1, -1, -1, -1));
    bool chunked = false;
    int64_t longest[2] = {int64_t(1) << 40, int64_t(1) << 40};  // without chunks: longest tiles first
    // (unit, tile row) -> the key ranges of its items; slots taken.
    std::map<std::pair<int, int>, std::vector<std::array<int, 2>>> met;
    std::map<std::pair<bool, int>, int> slots;
    const int grid = room;
    for (int x = 0; x < grid + 3; ++x) {
        PagedItem it;
        if constexpr (kShared)
            it = shared_item<Shape, HostWave>(a, x);
        else
            it = paged_item<Shape, HostWave>(a, x, seqs.data(), staged);
        CHECK(it.found == (x < items));
        if (!it.found) continue;
        CHECK(x < grid);
        CHECK(it.u >= 0 && it.u < units);
        const PagedUnit u = paged_unit(a, it.u);
        CHECK(u.t0 >= 0 && u.n > 0 && u.t0 + u.n <= a.T && it.rows == u.n * a.group);
        CHECK(it.many == (it.rows > Shape::kMany));
        const int tile = it.many ? Shape::kTile : 32;
        CHECK(it.r0 >= 0 && it.r0 % tile == 0 && it.r0 < it.rows);
        CHECK(it.kbeg >= u.kbeg && it.kend <= u.kend);
        if (!kShared && a.wgs == 0 && a.B > 1 && (it.many || a.B <= 64)) {
            const int step = it.many ? Shape::kStep : Shape::kRound;
            const int64_t n = (std::max(0, it.kend) + step - 1) / step;
            CHECK(n <= longest[it.many]);
            longest[it.many] = n;
        }
        if (!it.direct) CHECK(it.slot >= 0 && it.slot < (it.many ? a.max_many : a.max_few));
        if (!it.direct) {
            const int taken = ++slots[{it.many, it.slot}];
            CHECK(taken == 1);
        }
        const int last = a.group_div(std::min(it.rows, it.r0 + tile) - 1);
        if (a.causal) CHECK(it.kend <= paged_limit(a, it.u, u, last));
        // Parts of the unit's rows, as the combine counts them.
        PagedUnitItems ui = it.of;
        if (kShared) {
            const SharedCut& c = a.cut;
            const int keys = u.kend - u.kbeg;
            const int pre = c.pre_tiles * c.pre_chunks;
            ui.many = it.u == 0 ? c.pre_many : c.own_many;
            ui.chunks = it.u == 0 ? c.pre_chunks : keys / shared_own_len(a, keys) + (keys % shared_own_len(a, keys) > 0);
            ui.first = it.u == 0 ? 0
                                 : (c.pre_many == c.own_many ? pre : 0) +
                                       (it.u - 1) * c.own_chunks * c.own_tiles;
            CHECK(ui.chunks <= (it.u == 0 ? c.pre_chunks : c.own_chunks));
            // Chunks past a sequence's keys are empty items that nobody reads.
            if (it.slot - ui.first >= ui.chunks * ui.tiles) {
                CHECK(it.kbeg >= it.kend);
                continue;
            }
            noted[it.u] = make_int4(ui.first, ui.tiles, ui.chunks, ui.many);
        }
        auto& ranges = met[{it.u, it.r0}];
        CHECK(!it.direct || ranges.empty());
        ranges.push_back({it.kbeg, it.kend});
        if (it.first && a.wgs > 0) {
            CHECK(noted[it.u].x == -1);
            noted[it.u] = make_int4(ui.first, ui.tiles, ui.chunks, ui.many);
        }
        CHECK(ui.many == it.many);
        CHECK(it.direct == (ui.chunks == 1 && !a.shared));
        chunked |= ui.chunks > 1;
        const int i = it.r0 / tile;
        const int at = it.slot - ui.first;
        if (it.direct) continue;  // no slot
        CHECK(at >= 0 && at < ui.tiles * ui.chunks);
        CHECK(at % ui.tiles == (a.causal ? ui.tiles - 1 - i : i));
        const int used = std::min(tile, it.rows - it.r0);
        CHECK(it.many || used <= a.few_rows);
        const size_t row = paged_slot_row<Shape>(a, a.Hkv - 1, it.many, it.slot, used - 1);
        CHECK(row < static_cast<size_t>(a.Hkv) * a.max_many * Shape::kTile +
                        static_cast<size_t>(a.Hkv) * a.max_few * a.few_rows);
    }
    for (int u = 0; u < units; ++u) {
        const PagedUnit pu = paged_unit(a, u);
        const int rows = pu.n * a.group;
        const int tile = rows > Shape::kMany ? Shape::kTile : 32;
        // What the combine finds: noted by the unit's first item, but where there is none.
        const int4 n = noted[u];
        PagedUnitItems ui = n.x >= 0 ? PagedUnitItems{n.x, n.y, n.z, n.w != 0}
                                           : PagedUnitItems{0, 0, 0, false};
        if (!kShared && a.wgs == 0) ui = PagedUnitItems{0, 0, pu.n > 0 ? 1 : 0, false};
        else if (n.x < 0) CHECK(pu.n == 0 || (a.shared && pu.kend == pu.kbeg));
        if (n.x >= 0 && (kShared || a.wgs > 0)) {
            CHECK(ui.tiles == (rows + tile - 1) / tile && ui.many == (rows > Shape::kMany));
            CHECK(ui.chunks <= 1 || ui.first + ui.tiles * ui.chunks <= (ui.many ? a.max_many : a.max_few));
        }
        for (int r0 = 0; r0 < rows; r0 += tile) {
            auto ranges = met[{u, r0}];
            CHECK(int(ranges.size()) == ui.chunks);
            std::sort(ranges.begin(), ranges.end());
            int at = pu.kbeg;  // keys below `at` are met
            for (auto& k : ranges) {
                if (k[1] <= k[0]) continue;
                CHECK(k[0] == at);
                at = k[1];
            }
            for (int r : {r0, std::min(rows, r0 + tile) - 1}) {
                const int lim = paged_limit(a, u, pu, a.group_div(r));
                CHECK(lim <= at || lim <= pu.kbeg);
                CHECK(lim <= pu.kend && lim >= 0);
            }
        }
    }
    return chunked;
}

}  // namespace

int main(int argc, char** argv) {
    const int n = argc > 1 ? std::atoi(argv[1]) : 1000;
    std::mt19937 rng(argc > 2 ? std::atoi(argv[2]) : 1);
    for (int i = 0; i < 200000; ++i) {
        const int d = 1 + int(rng() >> (1 + rng() % 31)), v = int(rng() >> 1);
        const FastDiv f = fast_div(std::max(1, d));
        const UniformDiv u(std::max(1, d));
        for (int x : {v, 0x7fffffff, 0, v / d * d, std::max(0, v / d * d - 1)}) CHECK(u(x) == x / d);
        for (int x : {v, 0x7fffffff, 0, v / d * d, std::max(0, v / d * d - 1)}) CHECK(f(x) == x / d);
    }
    int chunked = 0;
    for (g_case = 0; g_case < n; ++g_case) {
        using A = PagedShape<256, 64, 256, 2, 96>;
        using B = PagedShape<128, 32, 128, 1, 0x7fffffff>;
        const int kind = rng() % 6;
        chunked += kind == 0   ? launch<A, true>(rng)
                   : kind == 1 ? launch<B, true>(rng)
                   : kind % 2  ? launch<A, false>(rng)
                               : launch<B, false>(rng);
    }
    std::printf("%d launches, %d of them with chunks\n", n, chunked);
    return chunked > n / 10 ? 0 : 1;
}
