// How many tiles an attention over an 8-bit paged cache may have (q8_set_grains() in
// cuflash-attn_amd/csrc/paged_q8_plan.hpp), on the host: launches of up to 2^31 - 1 tokens are told to fit into the
// line of 2^30 grains only if they do, with the lengths that fill it most, and ordinary ones are not refused. No GPU
// call is made.

#include <algorithm>
#include <cstdio>
#include <cstdlib>

#include "paged_q8_plan.hpp"

namespace {

using namespace cuflash::dev;

#define CHECK(cond)                                              \
    do {                                                         \
        if (!(cond)) {                                           \
            std::printf("line %d: %s\n", __LINE__, #cond);       \
            std::exit(1);                                        \
        }                                                        \
    } while (0)

// The line of B sequences (a decode, or with T tokens dealt out evenly) that all have cap keys. They are of at most
// two kinds, so one of each is formed.
template <int R>
long long line_of(Q8PlanArgs a) {
    int keys = a.cap;
    a.seq_lens = &keys;
    if (!a.starts) {
        a.starts = nullptr;
        return Q8Line<R>(a, q8_seq(a, 0)).size * static_cast<long long>(a.B);
    }
    const int used = std::min(a.B, a.T), n = a.T / used, more = a.T % used;
    auto size = [&](int tokens) {
        const int starts[2] = {0, tokens};
        Q8PlanArgs b = a;
        b.starts = starts;
        return static_cast<long long>(Q8Line<R>(b, q8_seq(b, 0)).size);
    };
    return size(n) * (used - more) + (more ? size(n + 1) * more : 0);
}

template <int R>
bool fits(long long B, long long T, int group, int cap, bool decode, bool causal) {
    static const int kStarts = 0;
    Q8PlanArgs a{};
    a.B = static_cast<int>(B);
    a.T = static_cast<int>(T);
    a.group = group;
    a.group_div = fast_div(group);
    a.cap = cap;
    a.causal = causal;
    a.shares = 2048;
    a.starts = decode ? nullptr : &kStarts;
    const bool fit = q8_set_grains(a, R, R == 256 ? 1 : 0);
    if (fit) CHECK(line_of<R>(a) <= kQ8Line);
    return fit;
}

template <int R>
void check() {
    constexpr long long kMost = 0x7fffffff;
    for (int cap : {1, 1025, 100000, 0x7fffffff - 1023}) {
        // One token of one head each: a tile a sequence.
        CHECK(fits<R>(1LL << 30, 1LL << 30, 1, cap, true, false));
        CHECK(!fits<R>((1LL << 30) + 1, (1LL << 30) + 1, 1, cap, true, false));
        CHECK(!fits<R>(kMost, kMost, 1, cap, true, false));
        for (bool causal : {false, true}) {
            CHECK(fits<R>(900000000, 900000000, 1, cap, false, causal));
            CHECK(!fits<R>((1LL << 30) + 1, (1LL << 30) + 1, 1, cap, false, causal));
            // Many tokens in few sequences, sequences without tokens, many heads.
            for (long long B : {1, 2, 1000, 1 << 20, 1 << 29}) {
                CHECK(fits<R>(B, kMost, 1, cap, false, causal));
                CHECK(fits<R>(B, kMost / 64, 64, cap, false, causal));
                CHECK(fits<R>(B, 1, 65535, cap, false, causal));
            }
            CHECK(fits<R>(kMost - 63, 5, 7, cap, false, causal));
            CHECK(!fits<R>(kMost - 62, 5, 7, cap, false, causal));
        }
        for (int group : {1, 8, 40}) CHECK(fits<R>(kMost / group / 8, kMost / group / 8, group, cap, true, false));
    }
}

}  // namespace

int main() {
    check<16>();
    check<32>();
    check<256>();
    return 0;
}
