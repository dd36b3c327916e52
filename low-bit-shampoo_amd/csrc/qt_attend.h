// What the attention kernels over a 4-bit cache (layout: qt_cache.h) share: arguments, which tokens a sequence's queries see,
// and the split of fp32 numbers into 6-bit ones, which the matrix instructions multiply with the cache's 4-bit numbers.
#pragma once

#include "qt_cache.h"

namespace qt {

struct AttendArgs {
    CacheShape shape;
    CachePlaces at;
    const uint8_t *codes[2];
    const float *scales[2];
    const void *q;
    void *out;
    long long q_token, q_head, out_token, out_head;
    int heads, group;
    float factor;           // scale * log2 e
    int window, sinks;      // window 0: no window
    int slots;              // workgroups that a call is cut for
    float *partial;         // 2 * slots pieces of (16 rows x (DP + 2)) floats
};

#if defined(__HIPCC__)
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x32 __attribute__((ext_vector_type(32)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x6 __attribute__((ext_vector_type(6)));

#define QT_LDS __attribute__((address_space(3)))
#define QT_GLOBAL __attribute__((address_space(1)))

constexpr int kFp4 = 4, kFp6 = 2;               // operand formats of the scaled matrix instructions
constexpr int kOne = 0x7f7f7f7f;                // scale bytes that stand for 2^0

// 32 numbers as 6-bit floating ones (two bits of exponent, three of mantissa, at most 7.5) times the scale's power of two, in the
// order x[0], y[0], x[1], y[1] ...; these instructions write their result while they still read, which the compiler does not know: all
// operands are kept alive behind them, so that none shares a register with the result.
__device__ __forceinline__ u32x6 to_fp6(const f32x16 &x, const f32x16 &y, float scale) {
    u32x6 out = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(x, y, scale);
    asm volatile("" : "+v"(out) : "v"(x), "v"(y), "v"(scale));
    return out;
}
__device__ __forceinline__ f32x32 from_fp6(const u32x6 &piece, float scale) {
    f32x32 out = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(piece, scale);
    asm volatile("" : "+v"(out) : "v"(piece), "v"(scale));
    return out;
}

// 32 numbers as a sum of N pieces of 6 bits.  The first piece's scale puts the largest number in [2, 4), where pieces are 1/4 apart;
// every further piece takes what is left at 2^-5 of the scale before: a rest is at most 4 in units of its scale.  What N pieces
// leave is below 2^-(4 + 5 (N - 1)) of the largest number: 2^-14 for three, 2^-24 for five.  `top`: bits of the largest
// magnitude.  scale[i]: the matrix instruction's byte for piece i; 255, its NaN, where the numbers are not finite.
template <int N>
__device__ __forceinline__ void split_fp6(f32x16 x, f32x16 y, uint32_t top, u32x6 *piece, int *scale) {
    const int exponent = (int)((top >> 23) & 0xff);
    const int first = max(exponent - 1, 5 * N);     // (numbers below 2^-100: in steps of the least scale)
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float by = __uint_as_float((uint32_t)(first - 5 * i) << 23);
        piece[i] = to_fp6(x, y, by);
        scale[i] = exponent == 255 ? 255 : first - 5 * i;
        if (i + 1 < N) {
            const f32x32 back = from_fp6(piece[i], by);
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] -= back[2 * e], y[e] -= back[2 * e + 1];
        }
    }
}

__device__ __forceinline__ i32x8 as_operand(const u32x6 &p) {
    return (i32x8){(int)p[0], (int)p[1], (int)p[2], (int)p[3], (int)p[4], (int)p[5], 0, 0};
}
__device__ __forceinline__ i32x8 as_operand(const i32x4 &p) { return (i32x8){p[0], p[1], p[2], p[3], 0, 0, 0, 0}; }

// The tokens that the new ones of a sequence see: all of it up to them, or with a window its first `sinks` and the window of the
// first of them, in tiles of 128: `sink_tiles` from token 0, then those from `first_tile` on.
struct SequenceView {
    int start, count;                   // its rows of the call
    int first_position, end;            // position of the first; tokens of the sequence that its table can hold
    int sink_tiles, first_tile, tiles;
};

__device__ __forceinline__ SequenceView view_sequence(const AttendArgs &a, int b) {
    SequenceView v;
    const int length = a.at.lengths[b];
    v.start = a.at.starts ? a.at.starts[b] : b;
    v.count = a.at.starts ? a.at.starts[b + 1] - v.start : 1;
    if (v.start < 0 || v.count < 0 || (long long)v.start + v.count > a.at.tokens) v.count = 0;      // (not a list of starts: nothing)
    v.first_position = length - v.count;
    const long long covered = (long long)a.at.table_pages << a.shape.page_shift;
    v.end = (int)min((long long)max(length, 0), min(covered, 0x7fffff00LL));
    int low = 0;
    if (a.window) low = min(v.end, max(0, max(v.first_position, 0) - (a.window - 1)));
    v.first_tile = low >> 7;
    v.sink_tiles = min((int)(((long long)min(a.sinks, low) + 127) >> 7), v.first_tile);
    v.tiles = v.sink_tiles + ((v.end + 127) >> 7) - v.first_tile;
    return v;
}
#endif  // __HIPCC__

}  // namespace qt
