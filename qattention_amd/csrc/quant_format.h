// quant_format.h -- K/V rows held in 4 or 8 bits: blocks of 32 elements along
// the head dim share a scale.
//
//   element   4 bits: e2m1 (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives), the
//             block's even elements in the low halves of its bytes; 8 bits: e4m3
//             (largest 448)
//   scale     one byte c for 2^(c - 127); 255: the block is no number
//
// These are the formats that gfx950's scaled conversions read and write: two
// elements and their scale per instruction, at the rate of a float operation
// (1.8 ns per wave and SIMD, fma 1.8, exp2 3.6).  Elements times a power of two
// are exact in fp16 and bf16 (inside their range), so a row that is widened for
// a product is exactly what the cache holds, and no scale has to be multiplied
// into scores or weights afterwards.
//
// Writing: with A the block's largest magnitude and 2^T the top power of the
// format (T = 2, 8), the scale is the smallest power of two s with A <= 1.75
// 2^T s; elements are x / s, rounded to nearest, ties to the even code.  e4m3's
// largest is 1.75 2^8, so nothing is cut off; e2m1's is 1.5 2^2, and what lies in
// (6, 7] becomes 6, off by no more than the half step of 1 between its largest
// elements.  s is at least 2^-126 and at most what keeps every element in the
// rows' own range (2^(15 - T) for fp16, 2^(127 - T) for bf16: a largest element
// past 1.75 times the type's top power is cut off there).
#pragma once

#include "qattn_device.h"

namespace qattn {

constexpr int kQuantBlock = 32;  // elements of a scale

template <int BITS>
constexpr int kTopExp = BITS == 4 ? 2 : 8;

// Largest scale code of rows of T.
template <typename T, int BITS>
constexpr int kLastCode = 127 + (T::kCode == F16::kCode ? 15 : 127) - kTopExp<BITS>;

// The scale of a code, as the conversions take it (they use its exponent bits:
// code 0 is 2^-127, 255 makes every element NaN; checked for all codes).
__device__ __forceinline__ float scale_of(uint32_t code) { return __builtin_bit_cast(float, code << 23); }

// 8 elements, BITS / 4 words at w, as T.
template <typename T, int BITS>
__device__ __forceinline__ Vec16 widen8(const uint32_t* w, float s) {
    Vec16 r;
    if constexpr (BITS == 4) {
        if constexpr (T::kCode == F16::kCode) {
            r.w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], s, 0));
            r.w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], s, 1));
            r.w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], s, 2));
            r.w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], s, 3));
        } else {
            r.w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 0));
            r.w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 1));
            r.w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 2));
            r.w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 3));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (T::kCode == F16::kCode) {
                r.w[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], s, false));
                r.w[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], s, true));
            } else {
                r.w[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], s, false));
                r.w[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], s, true));
            }
        }
    }
    return r;
}

// A quad of lanes holds a block, 8 elements of T each: the lane's BITS / 4 words
// of elements, and the block's scale code (in every lane).
template <typename T, int BITS>
__device__ __forceinline__ uint32_t narrow8(const Vec16& x, uint32_t* w) {
    typedef uint16_t us2 __attribute__((ext_vector_type(2)));
    constexpr uint32_t kInf = T::kCode == F16::kCode ? 0x7c00u : 0x7f80u;
    // magnitudes order as integers do, infinities and NaN above all others
    auto mag = [](uint32_t v) { return __builtin_bit_cast(us2, v & 0x7fff7fffu); };
    const us2 m2 = __builtin_elementwise_max(__builtin_elementwise_max(mag(x.w[0]), mag(x.w[1])),
                                             __builtin_elementwise_max(mag(x.w[2]), mag(x.w[3])));
    uint32_t m = max((uint32_t)m2[0], (uint32_t)m2[1]);
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, true));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, true));
    uint32_t bits = m << 16;
    if constexpr (T::kCode == F16::kCode)
        bits = __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(_Float16, (uint16_t)m));
    const int want = (int)((bits + 0x1fffffu) >> 23) - kTopExp<BITS>;
    const int code = min(max(want, 1), kLastCode<T, BITS>);
    const float s = scale_of((uint32_t)code);
    if constexpr (BITS == 4) {
        uint32_t q = 0;  // (past 6 the conversion ends at 6)
        if constexpr (T::kCode == F16::kCode) {
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(h2_t, x.w[0]), s, 0);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(h2_t, x.w[1]), s, 1);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(h2_t, x.w[2]), s, 2);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(h2_t, x.w[3]), s, 3);
        } else {
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(b2_t, x.w[0]), s, 0);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(b2_t, x.w[1]), s, 1);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(b2_t, x.w[2]), s, 2);
            q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(b2_t, x.w[3]), s, 3);
        }
        w[0] = q;
    } else {
        typedef short s2_t __attribute__((ext_vector_type(2)));
        Vec16 y = x;
        if (__builtin_expect(want > code, 0)) {
            // the scale ends before the block does: elements end at 448 here (the
            // conversion makes NaN of those past 464)
            const float top = 448.f * s;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                y.w[i] = MfmaOps<T>::pack2(__builtin_amdgcn_fmed3f(MfmaOps<T>::lo(x.w[i]), -top, top),
                                           __builtin_amdgcn_fmed3f(MfmaOps<T>::hi(x.w[i]), -top, top));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            s2_t q = {0, 0};
            if constexpr (T::kCode == F16::kCode) {
                q = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(q, __builtin_bit_cast(h2_t, y.w[2 * i]), s, false);
                q = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(q, __builtin_bit_cast(h2_t, y.w[2 * i + 1]), s, true);
            } else {
                q = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(q, __builtin_bit_cast(b2_t, y.w[2 * i]), s, false);
                q = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(q, __builtin_bit_cast(b2_t, y.w[2 * i + 1]), s, true);
            }
            w[i] = __builtin_bit_cast(uint32_t, q);
        }
    }
    if (m >= kInf) {
#pragma unroll
        for (int i = 0; i < BITS / 4; ++i) w[i] = 0;
        return 255;
    }
    return (uint32_t)code;
}

}  // namespace qattn
