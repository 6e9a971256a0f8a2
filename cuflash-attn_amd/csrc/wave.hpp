#pragma once

// Lane permutations and sums over the lanes of a wave.

#include "common.hpp"

namespace cuflash {
namespace dev {

// DPP lane permutations (row = 16 lanes).
constexpr int kDppXor1 = 0xB1;        // quad_perm [1,0,3,2]
constexpr int kDppXor2 = 0x4E;        // quad_perm [2,3,0,1]
constexpr int kDppHalfMirror = 0x141;  // lane i <-> 7 - i within each 8 lanes
constexpr int kDppMirror = 0x140;      // lane i <-> 15 - i within each row
constexpr int kDppRowShr = 0x110;      // + n: lane i takes lane i - n of its row
constexpr int kDppRowBcast15 = 0x142;  // the last lane of a row to the next row
constexpr int kDppRowBcast31 = 0x143;  // lane 31 to rows 2 and 3

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}

// The 64 lanes of a wave for the plans of paged_split.hpp and paged_plan.hpp; sums and single lanes
// are wave-uniform.
struct GpuWave {
    using Int = int;
    template <class F>
    __device__ static Int each(F f) {
        return f(static_cast<int>(threadIdx.x & 63));
    }
    template <class F>
    __device__ static Int map(Int v, F f) {
        return f(v);
    }
    template <class F>
    __device__ static Int map2(Int v, Int w, F f) {
        return f(v, w);
    }
    template <class F>
    __device__ static Int map3(Int v, Int w, F f) {
        return f(static_cast<int>(threadIdx.x & 63), v, w);
    }
    __device__ static Int add(Int a, Int b) { return a + b; }
    // f(lane, v, w, sums) forms N numbers of each lane, from 0.
    template <int N, class F>
    __device__ static void fill(Int (&out)[N], Int v, Int w, F f) {
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = 0;
        f(static_cast<int>(threadIdx.x & 63), v, w, out);
    }
    // Inclusive sum over the lanes.
    __device__ static Int scan(Int v) {
        v += __builtin_amdgcn_update_dpp(0, v, kDppRowShr + 1, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, kDppRowShr + 2, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, kDppRowShr + 4, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, kDppRowShr + 8, 0xF, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, kDppRowBcast15, 0xA, 0xF, false);
        v += __builtin_amdgcn_update_dpp(0, v, kDppRowBcast31, 0xC, 0xF, false);
        return v;
    }
    // The largest of numbers from 0 on.
    __device__ static int most(Int v) {
        v = max(v, __builtin_amdgcn_update_dpp(0, v, kDppRowShr + 1, 0xF, 0xF, false));
        v = max(v, __builtin_amdgcn_update_dpp(0, v, kDppRowShr + 2, 0xF, 0xF, false));
        v = max(v, __builtin_amdgcn_update_dpp(0, v, kDppRowShr + 4, 0xF, 0xF, false));
        v = max(v, __builtin_amdgcn_update_dpp(0, v, kDppRowShr + 8, 0xF, 0xF, false));
        v = max(v, __builtin_amdgcn_update_dpp(0, v, kDppRowBcast15, 0xA, 0xF, false));
        v = max(v, __builtin_amdgcn_update_dpp(0, v, kDppRowBcast31, 0xC, 0xF, false));
        return lane(v, 63);
    }
    __device__ static int lane(Int v, int i) { return __builtin_amdgcn_readlane(v, i); }
    // The first lane where f is not 0, or -1.
    template <class F>
    __device__ static int first(Int v, F f) {
        return __ffsll(static_cast<unsigned long long>(__ballot(f(v)))) - 1;
    }
};

// Sequence of packed token t: the number of sequences that end at or before it (`starts`, B + 1
// values, do not decrease), B where no sequence has it. All lanes of the wave take part.
__device__ __forceinline__ int sequence_of(const int* starts, int B, int t) {
    const int lane = threadIdx.x & 63;
    int b = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        const int n = __popcll(__ballot(b0 + lane < B && starts[min(b0 + lane, B - 1) + 1] <= t));
        b += n;
        if (n < 64) break;
    }
    return b < B && t < starts[b] ? B : b;
}

}  // namespace dev
}  // namespace cuflash
