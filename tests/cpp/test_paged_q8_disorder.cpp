// Starts that decrease, of so many tokens and sequences that the grains of all of them pass 32 bits: the cut of an
// attention over an 8-bit paged cache (cuflash-attn_amd/csrc/paged_q8_plan.hpp) on the host, with sums that wrap as the
// GPU's do. What such a call computes is undefined; checked is that every wave ends and that rows, keys and partial
// results stay inside the tensors and the workspace. No GPU call is made. Arguments: the number of launches, the seed.

#include <algorithm>
#include <array>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "paged_q8_plan.hpp"

namespace {

using namespace cuflash::dev;

struct WrappingWave {
    using Int = std::array<int, 64>;
    template <class F>
    static Int each(F f) {
        Int v;
        for (int i = 0; i < 64; ++i) v[i] = f(i);
        return v;
    }
    static Int scan(Int v) {
        for (int i = 1; i < 64; ++i)
            v[i] = static_cast<int>(static_cast<unsigned>(v[i]) + static_cast<unsigned>(v[i - 1]));
        return v;
    }
    static int lane(const Int& v, int i) { return v[i]; }
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

template <int R>
void launch(std::mt19937& rng) {
    auto pick = [&](int n) { return int(rng() % unsigned(n)); };
    Q8PlanArgs a{};
    a.group = 1 << pick(5);
    a.group_div = fast_div(a.group);
    a.causal = pick(2);
    a.B = 2 + pick(700);
    a.T = (1 << (18 + pick(4))) + pick(1000);
    a.cap = 1 + pick(1 << (6 + pick(14)));
    a.shares = 1 + pick(2048);
    a.least = 1 + pick(4);
    // Every second sequence, or most, has all tokens or nearly all.
    std::vector<int> lens, starts;
    for (int b = 0; b <= a.B; ++b) {
        lens.push_back(a.cap - pick(std::min(a.cap, 9)));
        starts.push_back(b % 2 ? a.T - pick(9) : pick(20) == 0 ? pick(a.T) : 0);
    }
    a.seq_lens = lens.data();
    a.starts = starts.data();
    if (!q8_set_grains(a, R, R == 256 ? 1 : 0)) return;
    const Q8Total total = q8_total<R, WrappingWave>(a);
    CHECK(total.grains >= 0 && total.grains <= kQ8Line && total.share >= a.least);
    for (int p = 0; p < a.shares; p += 1 + pick(1 + a.shares / 20)) {
        for (int q : {p, a.shares - 1 - p}) {
            Q8Walk<R, WrappingWave> walk(a, q);
            Q8Segment s;
            // A share may have millions of tiles: its first ones, and the last.
            for (int steps = 0; walk.next(a, s); ++steps) {
                CHECK(s.b >= 0 && s.b < a.B);
                CHECK(s.seq.t0 >= 0 && s.seq.n >= 0 && s.seq.t0 + s.seq.n <= a.T);
                CHECK(s.rows == s.seq.n * a.group && s.r0 >= 0 && s.r0 < s.rows);
                CHECK(s.kbeg >= 0 && s.kbeg < s.kend && s.kend <= a.cap);
                CHECK(s.slot < 2 && (s.slot < 1 || q < a.shares - 1));
                if (steps == 300 && walk.end - walk.x > 1 << 14) walk.x = walk.end - (1 << 13);
                if (steps > 20000) break;
                while (walk.b + 1 < a.B && walk.x - walk.first >= Q8Line<R>(a, q8_seq(a, walk.b)).size)
                    walk.first += Q8Line<R>(a, q8_seq(a, walk.b++)).size;
            }
        }
    }
    for (int i = 0; i < 200; ++i) {
        const int b = pick(a.B);
        const Q8Seq s = q8_seq(a, b);
        if (s.n == 0) continue;
        const Q8Line<R> line(a, s);
        const int tile = pick(line.tiles);
        const Q8Parts parts = q8_parts(a, total, q8_begin_of<R, WrappingWave>(a, b) + line.begin(a, s, tile),
                                       Q8Line<R>::grains(a, line.keys(a, s, tile)));
        CHECK(parts.from >= 0 && parts.to < a.shares && (parts.slot == 0 || parts.from < a.shares));
    }
}

}  // namespace

int main(int argc, char** argv) {
    const int launches = argc > 1 ? std::atoi(argv[1]) : 100;
    std::mt19937 rng(argc > 2 ? std::atoi(argv[2]) : 1);
    for (g_case = 0; g_case < launches; ++g_case)
        g_case % 3 == 0 ? launch<16>(rng) : g_case % 3 == 1 ? launch<32>(rng) : launch<256>(rng);
    return 0;
}
