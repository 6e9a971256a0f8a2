#pragma once

// The numbers of an 8-bit cache (cuflash/paged_cache_q8.h): a code of one byte times the power of two
// 2^(x - 127) of a byte x that the codes of one key (or value) of a key/value head share.
//
// Such a product has at most 8 significant bits, so it is exact in bf16 and float and, in fp16's range,
// in fp16: the matrix products take keys and values as the cache holds them. e4m3 pairs become 16-bit
// pairs, scaled, in one instruction (v_cvt_scalef32_pk_{bf16,f16}_fp8; checked on gfx950 for every code and
// every x: exact, subnormal results included, x = 0 is 2^-127 and x = 255 NaN). int8 goes through float:
// one conversion and one product an element, and one instruction for each pair to pack.

#include <type_traits>

#include "common.hpp"
#include "cuflash/paged_cache_q8.h"

namespace cuflash {
namespace dev {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// The 16-bit type in which the matrix products take the cache's numbers: the queries' own, bf16 for float.
template <typename T>
struct Q8Operand {
    using type = T;
};
template <>
struct Q8Operand<float> {
    using type = __hip_bfloat16;
};

template <QuantCode C>
struct Q8;

template <>
struct Q8<QuantCode::E4M3> {
    static constexpr float kTop = 448.0f;
    static constexpr uint32_t kNone = 0x7f7f7f7fu;  // the codes of a row without a value: NaN
    // What expand() multiplies with, from x: the number that the conversion takes its exponent from.
    static __device__ __forceinline__ float factor(uint32_t x) { return __uint_as_float(x << 23); }
    // Codes 2 i and 2 i + 1 of `codes` as two 16-bit numbers.
    template <typename M, int i>
    static __device__ __forceinline__ uint32_t expand(uint32_t codes, float f) {
        if constexpr (std::is_same<M, __half>::value)
            return __builtin_bit_cast(uint32_t,
                                      __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, f, i != 0));
        else
            return __builtin_bit_cast(uint32_t,
                                      __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, f, i != 0));
    }
    // All four; the conversion scales anyway.
    template <typename M, bool kScaled>
    static __device__ __forceinline__ u32x2 four(uint32_t codes, float f) {
        static_assert(kScaled, "e4m3 codes are scaled as they are converted");
        return u32x2{expand<M, 0>(codes, f), expand<M, 1>(codes, f)};
    }
    // Codes 2 i and 2 i + 1 of two rows, scaled: the first ones as one pair, the second ones as another.
    template <typename M, int i>
    static __device__ __forceinline__ u32x2 turned(uint32_t a, float fa, uint32_t b, float fb) {
        const uint32_t x = expand<M, i>(a, fa), y = expand<M, i>(b, fb);
        return u32x2{__builtin_amdgcn_perm(y, x, 0x05040100u), __builtin_amdgcn_perm(y, x, 0x07060302u)};
    }
    template <int i>
    static __device__ __forceinline__ f32x2 expand_f32(uint32_t codes, float f) {
        return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, f, i != 0);
    }
    // Four numbers, within the codes' range, to codes: nearest, ties to even.
    static __device__ __forceinline__ uint32_t pack4(const float* y) {
        int v = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], v, true));
    }
};

template <>
struct Q8<QuantCode::INT8> {
    static constexpr float kTop = 127.0f;
    static constexpr uint32_t kNone = 0u;
    // 2^(x - 127), 2^-127 and NaN as the e4m3 conversion has them: it turns the code of 1 into them.
    static __device__ __forceinline__ float factor(uint32_t x) {
        return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(0x38u, __uint_as_float(x << 23), false)[0];
    }
    template <int i>
    static __device__ __forceinline__ float plain(uint32_t codes) {
        return static_cast<float>(static_cast<int8_t>(codes >> (8 * i)));
    }
    template <int i>
    static __device__ __forceinline__ float one(uint32_t codes, float f) {
        return plain<i>(codes) * f;
    }
    // Two numbers that M has (in fp16 rounded, where it has not).
    template <typename M>
    static __device__ __forceinline__ uint32_t pair(float a, float b) {
        if constexpr (std::is_same<M, __half>::value) {
            return Elem<__half>::pack2(a, b);
        } else {
            // The upper halves: what is cut off is 0.
            return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
        }
    }
    template <typename M, int i>
    static __device__ __forceinline__ uint32_t expand(uint32_t codes, float f) {
        return pair<M>(one<2 * i>(codes, f), one<2 * i + 1>(codes, f));
    }
    // All four, scaled or as they are.
    template <typename M, bool kScaled>
    static __device__ __forceinline__ u32x2 four(uint32_t codes, float f) {
        if constexpr (!kScaled && std::is_same<M, __half>::value) {
            // code + 128 as the low byte of an fp16 number from 1024 on, whose steps are 1.
            const f16x2 minus = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
            codes ^= 0x80808080u;
            auto two = [&](uint32_t select) {
                const uint32_t x = __builtin_amdgcn_perm(0x64646464u, codes, select);
                return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, x) + minus);
            };
            return u32x2{two(0x04010400u), two(0x04030402u)};
        } else if constexpr (!kScaled) {
            return u32x2{pair<M>(plain<0>(codes), plain<1>(codes)),
                         pair<M>(plain<2>(codes), plain<3>(codes))};
        } else {
            return u32x2{expand<M, 0>(codes, f), expand<M, 1>(codes, f)};
        }
    }
    template <typename M, int i>
    static __device__ __forceinline__ u32x2 turned(uint32_t a, float fa, uint32_t b, float fb) {
        return u32x2{pair<M>(one<2 * i>(a, fa), one<2 * i>(b, fb)),
                     pair<M>(one<2 * i + 1>(a, fa), one<2 * i + 1>(b, fb))};
    }
    template <int i>
    static __device__ __forceinline__ f32x2 expand_f32(uint32_t codes, float f) {
        return f32x2{one<2 * i>(codes, f), one<2 * i + 1>(codes, f)};
    }
    static __device__ __forceinline__ uint32_t pack4(const float* y) {
        uint32_t v = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v |= (static_cast<uint32_t>(static_cast<int>(rintf(y[i]))) & 0xffu) << (8 * i);
        return v;
    }
};

}  // namespace dev
}  // namespace cuflash
