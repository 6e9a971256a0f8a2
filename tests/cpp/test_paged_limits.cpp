// The cut of a shared decode (cuflash-attn_amd/csrc/paged_plan.hpp) on the host where lengths come near
// the documented limit of 2^31 - 1024 keys: every key of a sequence lies in exactly one chunk, and the
// combine counts just the chunks that have keys. No GPU call is made.
//
// Arguments: the number of random launches, the seed.

#define main paged_plan_main  // for its HostWave, CHECK and spread
#include "test_paged_plan.cpp"
#undef main

namespace {

// Sequences with lens[b] keys behind `prefix` shared ones, for wgs workgroups per key/value head.
template <class Shape>
void check(std::vector<int> lens, int prefix, int group, int wgs, int min_steps) {
    PagedArgs a{};
    a.B = a.T = static_cast<int>(lens.size());
    a.Hkv = 1;
    a.H = a.group = group;
    a.group_div = fast_div(group);
    a.cap = 0x7fffffff - 1023;
    a.shared = true;
    a.wgs = wgs;
    a.prefix = prefix;
    a.seq_lens = lens.data();
    a.cut = shared_cut<Shape>(a.B, group, prefix, wgs, min_steps);
    const SharedCut& c = a.cut;
    const int pre = c.pre_tiles * c.pre_chunks, own = c.own_chunks * c.own_tiles;
    // Keys up to which the parts of each unit's tiles reach, and how many parts have keys.
    std::vector<int> at(a.B + 1, prefix), parts(a.B + 1, 0);
    at[0] = 0;
    for (int x = 0; x < pre + a.B * own; ++x) {
        const PagedItem it = shared_item<Shape, HostWave>(a, x);
        CHECK(it.found && it.u >= 0 && it.u <= a.B);
        CHECK(it.kbeg >= 0 && it.kend <= it.unit.kend);
        if (it.r0 != 0 || it.kbeg >= it.kend) continue;
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

template <class Shape>
void check_all(std::mt19937& rng, int n) {
    const int most = 0x7fffffff - 1023;
    for (g_case = 0; g_case < 3; ++g_case) {
        check<Shape>({most}, 77, 4, 128, 8);  // chunks of a 64th
        check<Shape>(std::vector<int>(600, (1 << 30) + 200), 100, 4, 64, 8);  // one chunk
        check<Shape>({most, 0, 100, most - 1, (1 << 30) + 1}, g_case, 128, 64, 8);
        check<Shape>({most, most}, most, 1, 512, 8);  // a prefix as long as the limit
    }
    for (; g_case < n; ++g_case) {
        std::vector<int> lens(spread(rng, 1, 300));
        for (int& x : lens) x = rng() % 3 ? most - int(rng() % 4000) : spread(rng, 1, most);
        check<Shape>(lens, rng() % 4 ? spread(rng, 1, most) : 0, 1 + int(rng() % 140),
                     spread(rng, 1, 600), 1 + int(rng() % 8));
    }
}

}  // namespace

int main(int argc, char** argv) {
    const int n = argc > 1 ? std::atoi(argv[1]) : 100;
    std::mt19937 rng(argc > 2 ? std::atoi(argv[2]) : 1);
    check_all<PagedShape<256, 64, 256, 2, 96>>(rng, n);
    check_all<PagedShape<128, 64, 128, 2, 96>>(rng, n);
    check_all<PagedShape<128, 32, 128, 1, 0x7fffffff>>(rng, n);
    std::printf("%d launches of each shape\n", n);
    return 0;
}
