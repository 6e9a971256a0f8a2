#pragma once

// What the attention kernels over an 8-bit paged cache have in common (attention_q8.hip: a wave takes a
// share of the keys; prompt_q8.hip: a workgroup does): arguments, partial results and their merge.

#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "launch.hpp"
#include "paged_q8_launch.hpp"
#include "paged_q8_plan.hpp"
#include "profile.hpp"
#include "q8.hpp"
#include "softmax.hpp"
#include "wave.hpp"

namespace cuflash {
namespace dev {

struct AttentionQ8Args {
    Q8PlanArgs plan;
    const int* block_table;  // [B, max_pages]
    int H, Hkv;
    int page_size, max_pages;
    uint64_t page_bytes, page_exps;  // codes and exponents of a page
    FastDiv page_div;
    float c;          // scale * log2(e)
    int slot_rows;    // rows of a partial result
    float* acc;       // [2 shares - 1, Hkv, slot_rows, D]: the last share has no second part
    float2* ml;       // the same without D: m in log2 units, l
};

// The row in acc and ml of row r of a tile, of wave (or workgroup) p.
__device__ __forceinline__ size_t q8_slot_row(const AttentionQ8Args& a, int p, int slot, int hk, int r) {
    return ((static_cast<size_t>(p) * 2 + slot) * a.Hkv + hk) * a.slot_rows + r;
}

// A row's parts on their way into one: O = sum O_i 2^(m_i - M) / l with M = max m_i and l = sum l_i
// 2^(m_i - M), L = (M + log2 l) ln 2. A lane has four columns.
struct Q8Merge {
    float M = -INFINITY, l = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    // N parts, v = (m, l) each. One without a key of the row, or whose scores are all -inf, has no say, also
    // where 0 times a value made it NaN.
    template <int N>
    __device__ __forceinline__ void add(const float2 (&v)[N], const f32x4 (&x)[N]) {
        float M2 = M;
#pragma unroll
        for (int i = 0; i < N; ++i) M2 = fmaxf(M2, v[i].x);
        auto weight = [&](float mi) { return mi == -INFINITY ? 0.0f : fast_exp2(mi - M2); };
        const float f0 = weight(M);
        l *= f0;
        acc *= f0;
        M = M2;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float f = weight(v[i].x);
            l = fmaf(v[i].y, f, l);
#pragma unroll
            for (int c = 0; c < 4; ++c)
                acc[c] = v[i].x == -INFINITY ? acc[c] : fmaf(x[i][c], f, acc[c]);
        }
    }
    // The lane's columns, from `to` on, and (once a row) L.
    template <typename T>
    __device__ __forceinline__ void store(typename Mma<T>::elem* to, float* L, bool first) const {
        const bool none = l == 0.0f;
        const float inv = none ? 0.0f : 1.0f / l;
        float y[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] = none ? 0.0f : acc[c] * inv;
        if constexpr (std::is_same<T, float>::value)
            st16(to, u32x4{__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]),
                           __float_as_uint(y[3])});
        else
            st8(to, u32x2{Elem<T>::pack2(y[0], y[1]), Elem<T>::pack2(y[2], y[3])});
        if (first) *L = none ? -INFINITY : (M + fast_log2(l)) * kLn2;
    }
};

// The merge, row by row: one workgroup per token and gridDim.y-th part of its heads. D / 4 lanes have a row,
// and kWays groups of them every kWays-th part of it; they are merged through LDS in order.
template <typename T, int D, int R, int kWays, int kThreads>
__global__ void __launch_bounds__(kThreads)
    combine_q8_kernel(typename Mma<T>::elem* __restrict__ O, float* __restrict__ L,
                      AttentionQ8Args a) {
    constexpr int LPR = D / 4;
    constexpr int kRows = kThreads / LPR / kWays;  // at a time
    constexpr int kBatch = 4;
    __shared__ f32x4 s_acc[kThreads];
    __shared__ float2 s_ml[kThreads / LPR];
    const int t = blockIdx.x;
    const int slot = threadIdx.x / LPR;
    const int way = slot % kWays;
    const int part = threadIdx.x % LPR;
    const int b = a.plan.starts ? sequence_of(a.plan.starts, a.plan.B, t) : t;
    if (b == a.plan.B) return;  // padding
    const Q8Seq s = q8_seq(a.plan, b);
    if (t - s.t0 >= s.n) return;  // starts that decrease
    const Q8Total total = q8_total<R, GpuWave>(a.plan);
    const int first = q8_begin_of<R, GpuWave>(a.plan, b);
    const Q8Line<R> line(a.plan, s);
    for (int h0 = blockIdx.y * kRows; h0 < a.H; h0 += gridDim.y * kRows) {
        const int h = h0 + slot / kWays;
        const bool on = h < a.H;
        const int hk = a.plan.group_div(on ? h : 0);
        const int r = (t - s.t0) * a.plan.group + ((on ? h : 0) - hk * a.plan.group);
        const int tile = r / R;
        const Q8Parts parts =
            q8_parts(a.plan, total, first + line.begin(a.plan, s, tile),
                     Q8Line<R>::grains(a.plan, line.keys(a.plan, s, tile)));
        const bool mine = on && parts.from != parts.to;  // else written already
        Q8Merge sum;
        for (int p0 = parts.from + way; mine && p0 <= parts.to; p0 += kBatch * kWays) {
            float2 v[kBatch];
            f32x4 x[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int p = p0 + i * kWays;
                v[i] = make_float2(-INFINITY, 0.0f);
                x[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if (p <= parts.to) {
                    const size_t at =
                        q8_slot_row(a, p, p == parts.from ? parts.slot : 0, hk, r - tile * R);
                    v[i] = a.ml[at];
                    x[i] = __builtin_bit_cast(f32x4, ld16(a.acc + at * D + 4 * part));
                }
            }
            sum.add(v, x);
        }
        if constexpr (kWays > 1) {
            s_acc[threadIdx.x] = sum.acc;
            if (part == 0) s_ml[slot] = make_float2(sum.M, sum.l);
            __syncthreads();
            if (way == 0) {
                sum = Q8Merge();
                constexpr int kAtOnce = kWays < 4 ? kWays : 4;
                for (int w0 = 0; w0 < kWays; w0 += kAtOnce) {
                    float2 v[kAtOnce];
                    f32x4 x[kAtOnce];
#pragma unroll
                    for (int w = 0; w < kAtOnce; ++w) {
                        v[w] = s_ml[slot + w0 + w];
                        x[w] = s_acc[threadIdx.x + (w0 + w) * LPR];
                    }
                    sum.add(v, x);
                }
            }
        }
        if (mine && way == 0) {
            const size_t row = static_cast<size_t>(t) * a.H + h;
            sum.store<T>(O + row * D + 4 * part, L + row, part == 0);
        }
        if constexpr (kWays > 1) __syncthreads();  // before the next rows'
    }
}

// The merge where there are many rows, most of them whole: by share, as every cut tile begins in one. A
// workgroup has kMergeRows rows of the tile that share blockIdx.x begins and does not finish, if it does; those
// behind the shares write the rows of tiles without a key.
constexpr int kMergeRows = 32;
template <typename T, int D, int R>
__global__ void __launch_bounds__(256)
    merge_q8_kernel(typename Mma<T>::elem* __restrict__ O, float* __restrict__ L,
                    AttentionQ8Args a) {
    constexpr int LPR = D / 4;
    constexpr int kRows = 256 / LPR;  // at a time
    constexpr int kBatch = 4;
    const int hk = blockIdx.y;
    const int part = threadIdx.x % LPR;
    auto row_of = [&](const Q8Seq& s, int r) {
        const int i = a.plan.group_div(r);
        return static_cast<size_t>(s.t0 + i) * a.H + hk * a.plan.group + (r - i * a.plan.group);
    };
    if (static_cast<int>(blockIdx.x) >= a.plan.shares) {
        const int each = gridDim.x - a.plan.shares;
        for (int b = blockIdx.x - a.plan.shares; b < a.plan.B; b += each) {
            const Q8Seq s = q8_seq(a.plan, b);
            const int n = q8_rows_without_keys<R>(a.plan, s);
            for (int r = blockIdx.z * kRows + threadIdx.x / LPR; r < n; r += gridDim.z * kRows) {
                const size_t row = row_of(s, r);
                Q8Merge().store<T>(O + row * D + 4 * part, L + row, part == 0);
            }
        }
        return;
    }
    const int p = blockIdx.x;
    const Q8Total total = q8_total<R, GpuWave>(a.plan);
    const int end = min((p + 1) * total.share, total.grains);
    if (p * total.share >= end) return;
    int first, tile, grain;
    const int b = q8_sequence_at<R, GpuWave>(a.plan, end - 1, first);
    const Q8Seq s = q8_seq(a.plan, b);
    const Q8Line<R> line(a.plan, s);
    if (end - 1 - first >= line.size || !line.find(a.plan, s, end - 1 - first, tile, grain)) return;
    const Q8Parts parts = q8_parts(a.plan, total, end - 1 - grain,
                                   Q8Line<R>::grains(a.plan, line.keys(a.plan, s, tile)));
    if (parts.from != p || parts.to == p) return;
    const int z = blockIdx.z * kMergeRows;
    const int rows = min(min(line.rows - tile * R, R), z + kMergeRows);
    for (int r = z + threadIdx.x / LPR; r < rows; r += kRows) {
        Q8Merge sum;
        for (int p0 = parts.from; p0 <= parts.to; p0 += kBatch) {
            float2 v[kBatch];
            f32x4 x[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                v[i] = make_float2(-INFINITY, 0.0f);
                x[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if (p0 + i <= parts.to) {
                    const size_t at =
                        q8_slot_row(a, p0 + i, p0 + i == parts.from ? parts.slot : 0, hk, r);
                    v[i] = a.ml[at];
                    x[i] = __builtin_bit_cast(f32x4, ld16(a.acc + at * D + 4 * part));
                }
            }
            sum.add(v, x);
        }
        const size_t row = row_of(s, tile * R + r);
        sum.store<T>(O + row * D + 4 * part, L + row, part == 0);
    }
}

}  // namespace dev

namespace detail {

// How one kernel takes a launch: tiles of `rows` rows, `shares` equal parts of all keys per key/value head.
struct Q8Grid {
    int rows, shares;
    int least_shift;  // grains of at least 32 << least_shift keys
    int least;        // such grains of a share
    int slot_rows;    // of a partial result
    int heads, kv_heads, head_dim, tokens;

    Q8Grid(const PagedCall& c, int tile_rows, int parts, int shift, int grains)
        : rows(tile_rows), shares(std::max(1, parts)), least_shift(shift), least(grains), heads(c.num_heads),
          kv_heads(c.num_kv_heads), head_dim(c.head_dim), tokens(c.num_tokens) {
        const long long group = c.num_heads / c.num_kv_heads;
        slot_rows = static_cast<int>(
            std::min<long long>(rows, c.query_starts ? group * c.num_tokens : group));
    }
    size_t slots() const {
        return (static_cast<size_t>(shares) * 2 - 1) * kv_heads * slot_rows;
    }
    size_t bytes() const { return slots() * (head_dim * sizeof(float) + sizeof(float2)); }
    // Many rows, of which few are cut: the merge goes by shares, else by tokens and heads.
    bool by_share() const { return static_cast<long long>(tokens) * heads >= kByShare; }
    static constexpr long long kByShare = 1 << 13;
    // fits: whether all tiles find their place in one line (paged_q8_plan.hpp).
    dev::AttentionQ8Args args(const PagedCall& c, bool* fits = nullptr) const {
        dev::AttentionQ8Args a{};
        a.plan.seq_lens = c.seq_lens;
        a.plan.starts = c.query_starts;
        a.plan.B = c.batch_size;
        a.plan.T = c.num_tokens;
        a.plan.group = c.num_heads / c.num_kv_heads;
        a.plan.cap = c.page_size * c.max_pages;
        a.plan.shares = shares;
        a.plan.causal = c.causal;
        a.plan.group_div = dev::fast_div(a.plan.group);
        const bool fit = dev::q8_set_grains(a.plan, rows, least_shift);
        if (fits) *fits = fit;
        a.plan.least = least;
        a.block_table = c.block_table;
        a.H = c.num_heads;
        a.Hkv = c.num_kv_heads;
        a.page_size = c.page_size;
        a.max_pages = c.max_pages;
        a.page_exps = static_cast<uint64_t>(c.page_size) * c.num_kv_heads;
        a.page_bytes = a.page_exps * c.head_dim;
        a.page_div = dev::fast_div(c.page_size);
        a.c = c.scale * dev::kLog2e;
        a.slot_rows = slot_rows;
        return a;
    }
};

// A given workspace that is too small, or a captured call without one: a graph's replays need memory that is theirs.
inline FlashAttentionError workspace_refusal(const PagedCall& c, size_t bytes, hipStream_t stream) {
    return (c.workspace ? c.workspace_bytes < bytes : stream_capturing(stream))
               ? FlashAttentionError::OUT_OF_MEMORY
               : FlashAttentionError::SUCCESS;
}

// Launches attend(args) and then the merge of R-row tiles, with the partial results in the caller's
// workspace or the library's.
template <typename T, int D, int R, class Attend>
FlashAttentionError run_q8(const PagedCall& c, const Q8Grid& grid, hipStream_t stream, Attend attend) {
    using E = typename dev::Mma<T>::elem;
    bool fits;
    dev::AttentionQ8Args a = grid.args(c, &fits);
    if (!fits) return FlashAttentionError::INVALID_DIMENSION;
    StreamWorkspace ws(stream, true);
    const FlashAttentionError refused = workspace_refusal(c, grid.bytes(), stream);
    if (refused != FlashAttentionError::SUCCESS) return refused;
    void* base = c.workspace;
    if (base == nullptr) {
        const FlashAttentionError err = ws.alloc(grid.bytes());
        if (err != FlashAttentionError::SUCCESS) return err;
        base = ws.get();
    }
    a.acc = static_cast<float*>(base);
    a.ml = reinterpret_cast<float2*>(a.acc + grid.slots() * D);
    attend(a);
    const FlashAttentionError err = from_hip(hipGetLastError());
    if (err != FlashAttentionError::SUCCESS) return err;
    auto merge = [&](auto kernel, dim3 groups, int threads) {
        launch_kernel(profile_kernel<T, D>("combine_q8"), kernel, groups,
                      dim3(static_cast<unsigned>(threads)), 0, stream, static_cast<E*>(c.O), c.L, a);
    };
    if (grid.by_share()) {
        merge(dev::merge_q8_kernel<T, D, R>,
              dim3(static_cast<unsigned>(grid.shares + std::min(c.batch_size, 64)),
                   static_cast<unsigned>(c.num_kv_heads),
                   static_cast<unsigned>((grid.slot_rows + dev::kMergeRows - 1) / dev::kMergeRows)),
              256);
    } else {
        // Few rows have many parts each and want more loads in flight: 32 rows of 256 parts 11.1 us with 256
        // threads a row, 7.8 with 1024 (of 32 parts 4.2 and 5.9); 2048 rows of 5 parts 7.7 with 256, 4.7 with 64.
        // Every workgroup finds its token's place first: with many tokens it takes several rounds of heads.
        auto rows = [&](auto kernel, int at_once, int threads) {
            const int rounds = (c.num_heads + at_once - 1) / at_once;
            const int most = std::max(1, 8 * compute_units() / c.num_tokens);
            merge(kernel,
                  dim3(static_cast<unsigned>(c.num_tokens),
                       static_cast<unsigned>(std::min(rounds, most))),
                  threads);
        };
        const long long all = static_cast<long long>(c.num_tokens) * c.num_heads;
        if (all <= 256 && a.plan.cap >= 2048)
            rows(dev::combine_q8_kernel<T, D, R, 1024 / (D / 4), 1024>, 1, 1024);
        else if (all <= 1024)
            rows(dev::combine_q8_kernel<T, D, R, 256 / (D / 4), 256>, 1, 256);
        else
            rows(dev::combine_q8_kernel<T, D, R, 256 / D, 256>, 4, 256);
    }
    return from_hip(hipGetLastError());
}

// prompt_q8.hip, for many rows a sequence, of 16 bits.
template <typename T>
Q8Grid prompt_q8_grid(const PagedCall& call);
template <typename T>
FlashAttentionError launch_prompt_q8(const PagedQ8Call& call, hipStream_t stream);

}  // namespace detail
}  // namespace cuflash
