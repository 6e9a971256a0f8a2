// The cut of the paged attentions (cuflash-attn_amd/csrc/paged_plan.hpp) on the host, for every shape that
// the kernels have: the launches of test_paged_plan.cpp; lengths near the documented limit of 2^31 - 1024
// keys; and so many query heads over a key/value head that a sequence of a shared decode has many rows of
// its own. No GPU call is made.
//
// Checked: every key of a unit lies in exactly one chunk; partial results go to slots of their own below
// those of the launch, where the combine finds them; the combine counts just the chunks that have keys.
//
// Arguments: the number of random launches, the seed.

#define main paged_plan_main  // for its HostWave, CHECK, spread and launch
#include "test_paged_plan.cpp"
#undef main

namespace {

constexpr int kMost = 0x7fffffff - 1023;

// Sequences with lens[b] keys behind `prefix` shared ones, for wgs workgroups per key/value head.
template <class Shape>
void check_shared(std::vector<int> lens, int prefix, int group, int wgs, int min_steps) {
    PagedArgs a{};
    a.B = a.T = static_cast<int>(lens.size());
    a.Hkv = 1;
    a.H = a.group = group;
    a.group_div = fast_div(group);
    a.cap = kMost;
    a.shared = true;
    a.wgs = wgs;
    a.prefix = prefix;
    a.seq_lens = lens.data();
    a.cut = shared_cut<Shape>(a.B, group, prefix, wgs, min_steps);
    const SharedCut& c = a.cut;
    const int pre = c.pre_tiles * c.pre_chunks, own = c.own_chunks * c.own_tiles;
    a.max_many = (c.pre_many ? pre : 0) + (c.own_many ? a.B * own : 0);
    a.max_few = pre + a.B * own - a.max_many;
    a.few_rows = c.pre_many && !c.own_many && c.own_tiles == 1 ? group : 32;
    // Keys up to which the parts of each unit's first tile reach, and how many parts have keys.
    std::vector<int> at(a.B + 1, prefix), parts(a.B + 1, 0);
    at[0] = 0;
    std::vector<bool> taken[2] = {std::vector<bool>(a.max_few), std::vector<bool>(a.max_many)};
    for (int x = 0; x < pre + a.B * own; ++x) {
        const PagedItem it = shared_item<Shape, HostWave>(a, x);
        CHECK(it.found && !it.direct && it.u >= 0 && it.u <= a.B);
        CHECK(it.kbeg >= 0 && it.kend <= it.unit.kend);
        CHECK(it.many == (it.u == 0 ? c.pre_many : c.own_many));
        CHECK(it.slot >= 0 && it.slot < (it.many ? a.max_many : a.max_few));
        CHECK(!taken[it.many][it.slot]);
        taken[it.many][it.slot] = true;
        const int tile = it.many ? Shape::kTile : 32;
        CHECK(it.r0 % tile == 0 && it.r0 < it.rows);
        CHECK(it.many || std::min(32, it.rows - it.r0) <= a.few_rows);
        if (it.kbeg >= it.kend) continue;
        const int first = it.u == 0 ? 0 : (c.own_many == c.pre_many ? pre : 0) + (it.u - 1) * own;
        const int tiles = it.u == 0 ? c.pre_tiles : c.own_tiles;
        const int chunk = (it.slot - first) / tiles;
        CHECK(it.slot == first + chunk * tiles + it.r0 / tile);
        if (it.r0 != 0) continue;
        CHECK(chunk == parts[it.u]);
        CHECK(it.kbeg == at[it.u]);  // chunk after chunk
        at[it.u] = it.kend;
        ++parts[it.u];
    }
    CHECK(at[0] == prefix && parts[0] == c.pre_chunks);
    for (int b = 0; b < a.B; ++b) {
        const int keys = paged_seq_len(a, b) - prefix;
        CHECK(at[b + 1] == std::max(prefix, paged_seq_len(a, b)));
        if (keys > 0) CHECK(shared_own_parts(a, keys) == parts[b + 1]);
    }
}

// Sequences with tokens[b] new tokens and lens[b] keys in a forward.
template <class Shape>
void check_forward(const std::vector<int>& tokens, std::vector<int> lens, int group, int wgs,
                   bool causal) {
    PagedArgs a{};
    a.B = static_cast<int>(lens.size());
    std::vector<int> starts(a.B + 1);
    for (int b = 0; b < a.B; ++b) starts[b + 1] = starts[b] + tokens[b];
    a.T = starts[a.B];
    if (a.T == 0) return;
    a.Hkv = 1;
    a.H = a.group = group;
    a.group_div = fast_div(group);
    a.cap = kMost;
    a.causal = causal;
    a.wgs = wgs;
    a.min_steps = 6;
    a.min_rounds = 1;
    a.few_rows = 32;
    a.seq_lens = lens.data();
    a.starts = starts.data();
    const PagedTiles t = paged_tiles<Shape>(a.T, a.B, group);
    const int room = wgs ? paged_room(int(t.all), wgs) : int(t.all);
    a.max_few = wgs ? std::min(room, 3 * wgs) : 0;
    a.max_many = t.many > 0 ? int(std::min<long long>(a.max_few, t.many + 2LL * wgs)) : 0;
    std::vector<int> at(a.B, 0);  // keys that the chunks of each unit's last tile reach
    std::vector<bool> taken[2] = {std::vector<bool>(a.max_few), std::vector<bool>(a.max_many)};
    for (int x = 0; x < room; ++x) {
        const PagedItem it = paged_item<Shape, HostWave>(a, x, nullptr, false);
        if (!it.found) continue;
        CHECK(it.u >= 0 && it.u < a.B && it.kbeg >= 0 && it.kend <= paged_seq_len(a, it.u));
        if (!it.direct) {
            CHECK(it.slot >= 0 && it.slot < (it.many ? a.max_many : a.max_few));
            CHECK(!taken[it.many][it.slot]);
            taken[it.many][it.slot] = true;
        }
        if (it.r0 + (it.many ? Shape::kTile : 32) < it.rows || it.kbeg >= it.kend) continue;
        CHECK(it.kbeg == at[it.u]);
        at[it.u] = it.kend;
    }
    for (int b = 0; b < a.B; ++b) CHECK(at[b] == (tokens[b] ? paged_seq_len(a, b) : 0));
}

template <class Shape>
void check_shape(std::mt19937& rng, int n) {
    for (g_case = 0; g_case < n; ++g_case) {
        launch<Shape, true>(rng);
        launch<Shape, false>(rng);
    }
    for (g_case = 0; g_case < 3; ++g_case) {
        check_shared<Shape>({kMost}, 77, 4, 128, 8);  // chunks of a 64th
        check_shared<Shape>(std::vector<int>(600, (1 << 30) + 200), 100, 4, 64, 8);  // one chunk
        check_shared<Shape>({kMost, 0, 100, kMost - 1, (1 << 30) + 1}, g_case, 128, 64, 8);
        check_shared<Shape>({kMost, kMost}, kMost, 1, 512, 8);  // a prefix as long as the limit
        check_forward<Shape>({1}, {kMost}, 4, 64, true);
        check_forward<Shape>({1, 40, 0, 300}, {kMost, kMost, kMost, 1 << 30}, 8, 128, g_case > 0);
    }
    for (; g_case < n; ++g_case) {
        const bool long_keys = rng() % 2;
        const int most = long_keys ? kMost : 20000;
        std::vector<int> lens(spread(rng, 1, 300)), tokens(lens.size());
        for (int& x : lens) x = rng() % 3 ? most - int(rng() % 4000) : spread(rng, 1, most);
        for (int& x : tokens) x = rng() % 4 ? 1 : spread(rng, 1, 600);
        const int group = rng() % 2 ? std::array<int, 3>{97, 128, 300}[rng() % 3] : 1 + int(rng() % 96);
        check_shared<Shape>(lens, rng() % 4 ? spread(rng, 1, most) : 0, group, spread(rng, 1, 600),
                            1 + int(rng() % 8));
        check_forward<Shape>(tokens, lens, 1 + int(rng() % 40), rng() % 4 ? spread(rng, 1, 300) : 0,
                             rng() % 3);
    }
}

template <class... Shapes>
void check_shapes(std::mt19937& rng, int n, const std::tuple<Shapes...>*) {
    (check_shape<Shapes>(rng, n), ...);
}

}  // namespace

int main(int argc, char** argv) {
    const int n = argc > 1 ? std::atoi(argv[1]) : 100;
    std::mt19937 rng(argc > 2 ? std::atoi(argv[2]) : 1);
    check_shapes(rng, n, static_cast<PagedShapes*>(nullptr));
    std::printf("%d launches of each kind and shape\n", n);
    return 0;
}
