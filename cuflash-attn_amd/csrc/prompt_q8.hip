// Attention of many 16-bit rows over an 8-bit paged cache for gfx950 (MI355X): the prompts of
// flash_attention_forward_paged_q8 (cuflash/paged_cache_q8.h).
//
// A workgroup of eight waves has 256 rows, the query heads of one key/value head over neighbouring tokens,
// 32 a wave, and a share of the keys (paged_q8_plan.hpp), 64 in a step that all of them take. In the forward
// kernels' transposed tiles: S^T = K Q^T, a lane pair per row, the softmax in the score registers,
// O^T += V^T P^T. Bound by MFMA and the softmax beside it, so codes are turned into 16-bit numbers once a
// workgroup, on their way into LDS: every thread has an eighth of a key's and of a value's codes of a step,
// in registers, one step ahead. (From the 8-bit codes in LDS every wave would convert all of them: 2 of 3
// instructions of the softmax beside it.)
//
// The two waves of a SIMD take turns on the matrix and the vector unit: waves 4 to 7 start half a step
// late, and a barrier after each half holds them there:
//   half 2 j:      waves 0-3  softmax of S_j                                  waves 4-7  products of step j
//   half 2 j + 1:  waves 0-3  O += V_j^T P_j, S_{j+1} = K_{j+1} Q^T           waves 4-7  softmax of S_j
// Products j read V_j and K_{j+1}, in the halves 2 j + 1 and 2 j + 2. Beside them, where its vector unit has
// time, a wave turns its share of the keys and values of step j + 2 (behind the softmax, in the other half, this
// took 3% longer), puts it into LDS and asks for the next.
// K_{j+2} takes the place of K_j, last read in half 2 j, and V_{j+2} that of V_{j-1}, too: two buffers for K and
// three for V.
// Measured: one prompt of 16384 tokens, bf16 over e4m3, 32 heads over 8, head_dim 128: 2133 us with its merge in a
// long loop, 1031 TFLOP/s (a large matrix product 1307), 2074 to 2186 by itself in a trace of 20 launches; the
// products alone take 1603, the softmax alone 917. Seven prompts of 285 to 2001 tokens, over int8, head_dim 64: 137 us
// with their merge in a loop, 153 by themselves in the trace, whose clock is lower; vector unit busy 54% of the time,
// MFMA 23%.

#include "attention_q8.hpp"
#include "tile_groups.hpp"

namespace cuflash {
namespace dev {

constexpr int kPromptWaves = 8;
constexpr int kPromptRows = 32 * kPromptWaves;

// Which thread puts which codes where. A wave has 8 keys, 8 lanes a key with D / 8 codes each; the
// lanes that write together, eight with 16 bytes or sixteen with 8, fall on all banks.
template <int D>
struct PromptTile : TileGroups<D> {
    using Lay = TileGroups<D>;
    static constexpr int kBytes32 = 32 / Lay::kRows * Lay::kBytes;  // 32 keys
    static constexpr int kBytes = 2 * kBytes32;                     // a step's
    static constexpr int kCodes = D / 8;                            // a thread's, of a key
    __device__ static int key(int lane) {
        return D == 128 ? ((lane >> 1) & 3) | ((lane >> 3) & 4)
               : D == 64 ? (lane >> 2) & 7 : lane >> 3;
    }
    __device__ static int part(int lane) {
        return D == 128 ? (lane & 1) | ((lane >> 2) & 6)
               : D == 64 ? (lane & 3) | ((lane >> 3) & 4) : lane & 7;
    }
    // Byte of element e (a multiple of 4) of key r of a step.
    __device__ static int at(int r, int e) {
        const int c = e >> 3, g = r / Lay::kRows, in = r % Lay::kRows;
        const int low = (e & 7) * 2;
        if constexpr (D == 128)
            return g * Lay::kBytes + 16 * (16 * (c >> 2) + 4 * in + (c & 3)) + low;
        else
            return g * Lay::kBytes + 16 * (32 * (c >> 2) + 4 * in + ((c & 3) ^ (2 * (in >> 2)))) +
                   low;
    }
};

template <typename T, int D, QuantCode C>
__global__ void __launch_bounds__((64 * kPromptWaves), (D == 32 ? 4 : 2))
    prompt_q8_kernel(const uint16_t* __restrict__ Q, const uint8_t* __restrict__ K,
                     const uint8_t* __restrict__ V, const uint8_t* __restrict__ Kx,
                     const uint8_t* __restrict__ Vx, uint16_t* __restrict__ O,
                     float* __restrict__ L, AttentionQ8Args a) {
    using Tile = PromptTile<D>;
    using Frag = typename Elem<T>::frag;
    constexpr int R = kPromptRows;
    constexpr int kStep = 64;
    constexpr int kBytes = Tile::kBytes;
    constexpr int KS = D / 16;
    constexpr int NDT = D / 32;
    constexpr int kMma = 4 * NDT;  // MFMAs of either product per step
    constexpr int kWords = Tile::kCodes / 4;
    constexpr int P = 2 * D + 16;  // pitch of a staged row of O
    constexpr int kStage = kPromptRows * P;
    __shared__ __attribute__((aligned(1024))) unsigned char
        smem[5 * kBytes > kStage ? 5 * kBytes : kStage];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31;
    const int g2 = lane >> 5;
    const int late = wave >> 2;  // 1: half a step behind
    // The items of a key/value head stay on one XCD where the heads can be dealt out evenly.
    int hk, share;
    head_rank_order(blockIdx.x, a.Hkv, hk, share);
    const uint32_t pitch = static_cast<uint32_t>(a.Hkv) * D;

    // This thread's codes of a step.
    const int my_key = 8 * wave + Tile::key(lane);
    const int my_part = Tile::part(lane) * Tile::kCodes;
    const uint8_t* const k_src = K + static_cast<size_t>(hk) * D + my_part;
    const uint8_t* const v_src = V + static_cast<size_t>(hk) * D + my_part;
    const uint8_t* const kx_src = Kx + static_cast<size_t>(hk) * a.page_size;
    const uint8_t* const vx_src = Vx + static_cast<size_t>(hk) * a.page_size;
    const int put_at = Tile::at(my_key, my_part);
    struct Codes {
        uint32_t w[kWords];
        uint32_t x;
    };
    auto get = [](Codes& to, const uint8_t* codes, const uint8_t* exps, size_t row, size_t ex) {
        if constexpr (kWords == 4) {
            const u32x4 w = ld16(codes + row);
#pragma unroll
            for (int i = 0; i < 4; ++i) to.w[i] = w[i];
        } else if constexpr (kWords == 2) {
            const u32x2 w = *reinterpret_cast<const u32x2*>(codes + row);
            to.w[0] = w[0];
            to.w[1] = w[1];
        } else {
            to.w[0] = *reinterpret_cast<const uint32_t*>(codes + row);
        }
        to.x = exps[ex];
    };
    struct Turned {
        uint32_t w[2 * kWords];
    };
    auto turn = [](const Codes& from) {
        const float by = Q8<C>::factor(from.x);
        Turned to;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            to.w[2 * i] = Q8<C>::template expand<T, 0>(from.w[i], by);
            to.w[2 * i + 1] = Q8<C>::template expand<T, 1>(from.w[i], by);
        }
        return to;
    };
    auto put = [&](const Turned& x, int buffer) {
        unsigned char* to = smem + buffer + put_at;
        if constexpr (kWords == 1) {
            st8(to, u32x2{x.w[0], x.w[1]});
        } else {
#pragma unroll
            for (int i = 0; i < kWords; i += 2)
                st16(to + 8 * i, u32x4{x.w[2 * i], x.w[2 * i + 1], x.w[2 * i + 2], x.w[2 * i + 3]});
        }
    };
    const int k_base[2] = {Tile::row_base(lane, 0), Tile::row_base(lane, 1)};
    const int v_base = Tile::tr_off(lane);
    const float cs = fmaxf(a.c, kFltMin);  // scale 0: -inf * 0 would make the masked scores NaN
    auto barrier = [] {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };

    const int step_pages = a.page_div(kStep);
    const int step_rows = kStep - step_pages * a.page_size;
    Q8Walk<R, GpuWave> walk(a.plan, share);
    Q8Segment s;
    while (walk.next(a.plan, s)) {
        const int* table = a.block_table + static_cast<size_t>(s.b) * a.max_pages;
        const int row = s.r0 + wave * 32 + l32;
        const bool on = row < s.rows;
        const int token = a.plan.group_div(on ? row : 0);
        const int orow = on ? (s.seq.t0 + token) * a.H + hk * a.plan.group +
                                  (row - token * a.plan.group)
                            : -1;
        Frag q[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            u32x4 v = {0u, 0u, 0u, 0u};
            if (on) v = ld16(Q + static_cast<size_t>(orow) * D + 16 * ks + 8 * g2);
            q[ks] = as_frag<T>(v);
        }
        // This lane's keys, and the least and the greatest end of the wave's rows.
        const int kend = on ? min(s.kend, q8_limit(a.plan, s.seq, token)) : s.kend;
        int least = kend, most = on ? kend : 0;
#pragma unroll
        for (int w = 16; w >= 1; w >>= 1) {
            least = min(least, __shfl_xor(least, w, 64));
            most = max(most, __shfl_xor(most, w, 64));
        }
        const int mask_from = __builtin_amdgcn_readfirstlane(least);
        const int wave_end = __builtin_amdgcn_readfirstlane(most);
        const int n = (s.kend - s.kbeg + kStep - 1) / kStep;  // at least 1
        // Steps in which this wave has keys to see.
        const int nw = wave_end > s.kbeg ? min(n, (wave_end - s.kbeg + kStep - 1) / kStep) : 0;

        // The place of this thread's key of the step to ask for, by walking from step to step (a division and its
        // 64-bit products are an eighth of a step at head_dim 64); the table is read a step ahead. Behind the end it
        // stands at the last key.
        const int last = s.kend - 1;
        const int last_index = a.page_div(last), last_row = last - last_index * a.page_size;
        int key = s.kbeg + my_key;
        int index = a.page_div(min(key, last));
        int in_page = min(key, last) - index * a.page_size;
        int entry = table[index];
        struct Step {
            Codes k, v;
        };
        auto ask = [&](Step& to) {
            const uint64_t row = static_cast<uint64_t>(static_cast<uint32_t>(entry)) *
                                     static_cast<uint32_t>(a.page_bytes) +
                                 static_cast<uint32_t>(in_page) * pitch;
            const uint64_t ex = static_cast<uint64_t>(static_cast<uint32_t>(entry)) *
                                    static_cast<uint32_t>(a.page_exps) +
                                static_cast<uint32_t>(in_page);
            get(to.k, k_src, kx_src, row, ex);
            get(to.v, v_src, vx_src, row, ex);
            key += kStep;
            in_page += step_rows;
            const bool over = in_page >= a.page_size;
            in_page -= over ? a.page_size : 0;
            index += step_pages + (over ? 1 : 0);
            const bool behind = key > last;
            in_page = behind ? last_row : in_page;
            index = behind ? last_index : index;
            entry = table[index];
        };
        // Values behind the end may be anything: 0, as 0 times an infinity or a NaN would be seen.
        auto cut = [&](int j, Step& x) {
            if (s.kbeg + kStep * j + my_key >= s.kend) {
#pragma unroll
                for (int w = 0; w < kWords; ++w) x.v.w[w] = 0;
                x.v.x = 127;
            }
        };

        f32x16 o[NDT];
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) o[dt] = f32x16{};
        f32x16 sc[2];
        sc[0] = sc[1] = f32x16{};
        Frag p[4];
        float m = -INFINITY, l = 0.0f;

        auto v_frag = [&](const unsigned char* vt, int i) {
            const unsigned char* at =
                vt + v_base + (i / NDT) * Tile::kTrRows16 + Tile::dtile_off(i % NDT);
            return tr_frag_at<T>(at, at + Tile::kTrHigh);
        };
        auto k_frag = [&](const unsigned char* kt, int i) {
            return as_frag<T>(
                ld16(kt + k_base[(i % KS) & 1] + (i / KS) * Tile::kBytes32 + Tile::k_off(i % KS)));
        };
        constexpr int kAhead = 4;  // MFMAs ahead of which an operand is read
        auto scores = [&](const unsigned char* kt) {
            Frag f[kMma];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) f[i] = k_frag(kt, i);
#pragma unroll
            for (int i = 0; i < kMma; ++i) {
                if (i + kAhead < kMma) f[i + kAhead] = k_frag(kt, i + kAhead);
                sc[i / KS] = Elem<T>::mma(f[i], q[i % KS], sc[i / KS]);
            }
        };
        // O += V^T P, then the next scores, in one chain. (Behind the last step these come from an old
        // tile and are not used.)
        auto products = [&](int v_from, int k_from) {
            const unsigned char* vt = smem + v_from;
            const unsigned char* kt = smem + k_from;
            Frag f[2 * kMma];
            auto frag_of = [&](int i) { return i < kMma ? v_frag(vt, i) : k_frag(kt, i - kMma); };
#pragma unroll
            for (int i = 0; i < kAhead; ++i) f[i] = frag_of(i);
#pragma unroll
            for (int i = 0; i < 2 * kMma; ++i) {
                if (i + kAhead < 2 * kMma) f[i + kAhead] = frag_of(i + kAhead);
                if (i < kMma) {
                    o[i % NDT] = Elem<T>::mma(f[i], p[i / NDT], o[i % NDT]);
                } else {
                    const int k = i - kMma;
                    if (k == 0) sc[0] = sc[1] = f32x16{};
                    sc[k / KS] = Elem<T>::mma(f[i], q[k % KS], sc[k / KS]);
                }
            }
        };
        // The softmax of S_j: masks, the lazily raised maximum, P_j rounded to T, the row sum in fp32.
        auto softmax = [&](int j) {
            const int key0 = s.kbeg + j * kStep;
            if (key0 + kStep > mask_from) {
                const int lim = kend - key0 - 4 * g2;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        sc[t][r] = 32 * t + 8 * (r >> 2) + (r & 3) < lim ? sc[t][r] : -INFINITY;
                }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int r = 0; r < 16; r += 2)
                    mx = __builtin_elementwise_maximum(
                        __builtin_elementwise_maximum(mx, sc[t][r]), sc[t][r + 1]);
            }
            const float m_new = fmaxf(m, pair_max(mx) * cs);
            const bool grow = m_new > m + kLazyRescale;
            if (__ballot(grow) != 0) {
                const float alpha = grow ? fast_exp2(m_new == -INFINITY ? 0.0f : m - m_new) : 1.0f;
                m = grow ? m_new : m;
                l *= alpha;
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) o[dt] *= alpha;
            }
            const float m_use = (m == -INFINITY) ? 0.0f : m;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f32x16& x = sc[i >> 1];
                const int r0 = 8 * (i & 1);
#pragma unroll
                for (int r = r0; r < r0 + 8; ++r) x[r] = fast_exp2(fmaf(x[r], cs, -m_use));
#pragma unroll
                for (int r = r0; r < r0 + 8; r += 2) sum += x[r] + x[r + 1];
                p[i] = pack_frag<T>(x[r0], x[r0 + 1], x[r0 + 2], x[r0 + 3], x[r0 + 4], x[r0 + 5],
                                    x[r0 + 6], x[r0 + 7]);
            }
            l += sum;
        };

        Step next;
        {
            Step first;
            ask(first);
            ask(next);
            cut(0, first);
            put(turn(first.k), 0);
            put(turn(first.v), 2 * kBytes);
            cut(1, next);
            put(turn(next.k), kBytes);
            put(turn(next.v), 3 * kBytes);
            ask(next);
        }
        barrier();
        scores(smem);
        if (late) barrier();
        int v_from = 2 * kBytes, v_to = 4 * kBytes;  // buffers of V_j and V_{j+2}
        for (int j = 0; j < n; ++j) {
            if (j < nw) softmax(j);
            barrier();
            cut(j + 2, next);
            const Turned k_next = turn(next.k), v_next = turn(next.v);
            if (j < nw) {
                __builtin_amdgcn_s_setprio(1);
                products(v_from, ((j + 1) & 1) * kBytes);
                __builtin_amdgcn_s_setprio(0);
            }
            put(k_next, (j & 1) * kBytes);
            put(v_next, v_to);
            ask(next);
            barrier();
            v_from = v_from == 4 * kBytes ? 2 * kBytes : v_from + kBytes;
            v_to = v_to == 4 * kBytes ? 2 * kBytes : v_to + kBytes;
        }
        if (!late) barrier();  // as many as the others

        // The outputs or partial results of the wave's rows.
        l = pair_sum(l);
        if (s.slot >= 0) {
            if (on) {
                const size_t slot = q8_slot_row(a, share, s.slot, hk, wave * 32 + l32);
                float* dst = a.acc + slot * D + 4 * g2;
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        f32x4 w;
#pragma unroll
                        for (int u = 0; u < 4; ++u) w[u] = o[dt][4 * i + u];
                        st16(dst + 32 * dt + 8 * i, __builtin_bit_cast(u32x4, w));
                    }
                }
                if (g2 == 0) a.ml[slot] = make_float2(m, l);
            }
        } else {
            // O rows through LDS, so that a store writes whole rows: 16 bytes a lane.
            constexpr int kChunks = D / 8;  // per row
            unsigned char* stage = smem + wave * 32 * P;
            const bool none = l == 0.0f;  // no key, or every score -inf: O = 0, L = -inf
            const float inv = none ? 0.0f : 1.0f / l;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) x[u] = none ? 0.0f : o[dt][4 * i + u] * inv;
                    st8(stage + l32 * P + (32 * dt + 8 * i + 4 * g2) * 2,
                        u32x2{Elem<T>::pack2(x[0], x[1]), Elem<T>::pack2(x[2], x[3])});
                }
            }
#pragma unroll
            for (int i = 0; i < 32 * kChunks / 64; ++i) {
                const int r = (64 * i + lane) / kChunks;
                const int cc = (64 * i + lane) % kChunks;
                const int to = __shfl(orow, r, 64);
                const u32x4 v = ld16(stage + r * P + cc * 16);
                if (to >= 0) st16(O + static_cast<size_t>(to) * D + cc * 8, v);
            }
            if (g2 == 0 && on) L[orow] = none ? -INFINITY : (m + fast_log2(l)) * kLn2;
        }
        barrier();  // before the next segment's tiles
    }
}

}  // namespace dev

namespace detail {
namespace {

template <int D>
Q8Grid grid_of(const PagedCall& c) {
    // Workgroups that run at once, as far as their partial results fit the library's workspace of a stream.
    const int groups = compute_units() * (D == 32 ? 2 : 1);
    const long long slot = static_cast<long long>(c.num_kv_heads) * dev::kPromptRows *
                           (D * sizeof(float) + sizeof(float2));
    const long long fit = (static_cast<long long>(kStreamCacheBytes) / slot + 1) / 2;
    return Q8Grid(c, dev::kPromptRows,
                  static_cast<int>(std::min<long long>(groups / c.num_kv_heads, fit)), 1,
                  4);
}

template <typename T, int D, QuantCode C>
FlashAttentionError run_prompt(const PagedQ8Call& q8, hipStream_t stream) {
    const PagedCall& c = q8.call;
    const Q8Grid grid = grid_of<D>(c);
    return run_q8<T, D, dev::kPromptRows>(c, grid, stream, [&](const dev::AttentionQ8Args& a) {
        launch_kernel(profile_kernel<T, D>("prompt_q8"), dev::prompt_q8_kernel<T, D, C>,
                      dim3(static_cast<unsigned>(grid.shares * c.num_kv_heads)),
                      dim3(64 * dev::kPromptWaves), 0, stream, static_cast<const uint16_t*>(c.Q),
                      static_cast<const uint8_t*>(c.K_cache),
                      static_cast<const uint8_t*>(c.V_cache), q8.K_exp, q8.V_exp,
                      static_cast<uint16_t*>(c.O), c.L, a);
    });
}

template <typename T, QuantCode C>
FlashAttentionError run_dim(const PagedQ8Call& c, hipStream_t stream) {
    switch (c.call.head_dim) {
        case 32:
            return run_prompt<T, 32, C>(c, stream);
        case 64:
            return run_prompt<T, 64, C>(c, stream);
        case 128:
            return run_prompt<T, 128, C>(c, stream);
    }
    return FlashAttentionError::UNSUPPORTED_HEAD_DIM;
}

}  // namespace

template <typename T>
Q8Grid prompt_q8_grid(const PagedCall& c) {
    return c.head_dim == 32 ? grid_of<32>(c) : c.head_dim == 64 ? grid_of<64>(c) : grid_of<128>(c);
}
template <typename T>
FlashAttentionError launch_prompt_q8(const PagedQ8Call& c, hipStream_t stream) {
    return c.code == QuantCode::E4M3 ? run_dim<T, QuantCode::E4M3>(c, stream)
                                     : run_dim<T, QuantCode::INT8>(c, stream);
}
#define CUFLASH_PROMPT_Q8(T)                                \
    template Q8Grid prompt_q8_grid<T>(const PagedCall&); \
    template FlashAttentionError launch_prompt_q8<T>(const PagedQ8Call&, hipStream_t);
CUFLASH_PROMPT_Q8(__half)
CUFLASH_PROMPT_Q8(__hip_bfloat16)
#undef CUFLASH_PROMPT_Q8

}  // namespace detail
}  // namespace cuflash
