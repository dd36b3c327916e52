// Segments of 4-bit floating numbers with an fp32 scale (qt_cache.h has the definition): encoding them, and multiplying them on the
// matrix cores with operands whose bits are all kept.
//
// The eight numbers are exact in bf16, so a product with a bf16 operand is exact in the matrix instructions' fp32 sums; an fp32
// operand goes through as three bf16 pieces of eight bits each, which add up to it.  The scale multiplies the sum of a segment.
#pragma once

#include "qt_common.h"
#include "qt_divide.h"

namespace qt {
#if defined(__HIPCC__)

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float fp4_f32x4 __attribute__((ext_vector_type(4)));

// Numbers of N (4 or 8) elements of a segment whose largest magnitude has the bits `top` (NaN above infinity, so that a segment
// with a NaN gets a NaN for its scale and reads as NaN): scale and quotients by correctly rounded division (qt_divide.h;
// quotients below 2^-40, which it may round otherwise, are code 0), nearest number (ties to the even code, beyond 6 to 6) by the
// conversion instruction.
template <int N>
__device__ __forceinline__ uint32_t encode_fp4(const float *x, uint32_t top, float &scale) {
    scale = __uint_as_float(top) / 6.0f;
    const uint32_t bits = __float_as_uint(scale);
    float y[N];
    if (bits >= kFastDivLo && bits <= kFastDivHi) {
        const float r = exact_reciprocal(scale);
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = quotient(x[e], scale, r);
    } else {
        // (zeroes times a scale that is not finite are NaN)
        const bool zero = bits == 0 || top >= 0x7f800000u;
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = zero ? 0.0f : x[e] / scale;
    }
    uint32_t word = 0;
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[0], y[1], 1.0f, 0);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[2], y[3], 1.0f, 1);
    if constexpr (N == 8) {
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[4], y[5], 1.0f, 2);
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[6], y[7], 1.0f, 3);
    }
    return word;
}

// Eight numbers as a matrix operand.
__device__ __forceinline__ bf16x8 fp4_to_bf16(uint32_t word) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, 1.0f, 1),
                 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, 1.0f, 3);
    return (bf16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Eight consecutive elements from an address that is aligned to an element only (the hardware takes such loads).
struct __attribute__((packed, aligned(2))) Unaligned16 { qt_u32x4 v; };
struct __attribute__((packed, aligned(4))) Unaligned16of4 { qt_u32x4 v; };

// An operand of eight elements as it lies in memory, and as the bf16 pieces that the matrix instructions multiply: one, or three whose
// sum is the fp32 number (each piece cuts off eight bits, so every difference is exact; a number that is not finite is its first piece; bf16 ends at 2^-133,
// and what an fp32 number has behind that is lost).
template <bool BF16>
struct Eight {
    static constexpr int kPieces = BF16 ? 1 : 3;
    uint32_t raw[BF16 ? 4 : 8];

    __device__ __forceinline__ void zero() {
#pragma unroll
        for (uint32_t &r : raw) r = 0;
    }
    // elements at .. at + 7 of a row
    __device__ __forceinline__ void load(const void *row, int at) {
        if constexpr (BF16) {
            const qt_u32x4 v = ((const Unaligned16 *)((const uint16_t *)row + at))->v;
#pragma unroll
            for (int e = 0; e < 4; ++e) raw[e] = v[e];
        } else {
            const qt_u32x4 v = ((const Unaligned16of4 *)((const float *)row + at))->v, w = ((const Unaligned16of4 *)((const float *)row + at + 4))->v;
#pragma unroll
            for (int e = 0; e < 4; ++e) raw[e] = v[e], raw[4 + e] = w[e];
        }
    }
    // those from `valid` on as zeros
    __device__ __forceinline__ void load(const void *row, int at, int valid) {
        if (at + 8 <= valid) {
            load(row, at);
        } else if (at >= valid) {
            zero();
        } else {
#pragma unroll
            for (int e = 0; e < (BF16 ? 4 : 8); ++e) {
                if constexpr (BF16) {
                    const uint16_t *p = (const uint16_t *)row + at;
                    raw[e] = (at + 2 * e < valid ? p[2 * e] : 0u) | ((at + 2 * e + 1 < valid ? p[2 * e + 1] : 0u) << 16);
                } else {
                    raw[e] = at + e < valid ? ((const uint32_t *)row)[at + e] : 0u;
                }
            }
        }
    }
    // what lane 4 (l % 16) + l / 16 has loaded: a wave's loads of sixteen rows touch each row's line once if four lanes side by side have a row, the
    // matrix instructions want lanes l, l + 16, l + 32, l + 48 to have it
    __device__ __forceinline__ void exchange() {
        const int lane = threadIdx.x & 63, from = 4 * (4 * (lane & 15) + (lane >> 4));
#pragma unroll
        for (uint32_t &r : raw) r = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)r);
    }
    // piece 0 holds the first bits
    __device__ __forceinline__ void pieces(bf16x8 *out) const {
        if constexpr (BF16) {
            out[0] = __builtin_bit_cast(bf16x8, (qt_u32x4){raw[0], raw[1], raw[2], raw[3]});
        } else {
            uint32_t part[3][8];
            float last = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float rest = __uint_as_float(raw[e]) - __uint_as_float(raw[e] & 0xffff0000u);
                part[0][e] = raw[e], part[1][e] = __float_as_uint(rest);
                const float tail = rest - __uint_as_float(part[1][e] & 0xffff0000u);
                part[2][e] = __float_as_uint(tail);
                last = e ? last + tail : tail;
            }
            if (__builtin_expect(__builtin_isunordered(last, last), 0)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if ((raw[e] & 0x7f800000u) != 0x7f800000u) continue;
                    if (raw[e] & 0x7fffffu) part[0][e] |= 0x400000u;            // (NaN whose bits are all in the part cut off)
                    part[1][e] = part[2][e] = 0;
                }
            }
            qt_u32x4 p[3];
#pragma unroll
            for (int n = 0; n < 3; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) p[n][e] = __builtin_amdgcn_perm(part[n][2 * e + 1], part[n][2 * e], 0x07060302u);     // (upper halves of both)
#pragma unroll
            for (int n = 0; n < 3; ++n) out[n] = __builtin_bit_cast(bf16x8, p[n]);
        }
    }
};

// d + (rows of x) (numbers): lane l has row l % 16 of x and column l % 16 of the numbers, elements 8 (l / 16) .. + 7 of 32; of the result
// column l % 16, rows 4 (l / 16) .. + 3.
template <int PIECES>
__device__ __forceinline__ fp4_f32x4 multiply_pieces(const bf16x8 *x, bf16x8 numbers, fp4_f32x4 d) {
#pragma unroll
    for (int n = PIECES - 1; n >= 0; --n) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[n], numbers, d, 0, 0, 0);
    return d;
}

#endif  // __HIPCC__
}  // namespace qt
