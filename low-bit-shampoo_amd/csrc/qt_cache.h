// An attention cache held in 4 bits: where a token of a sequence lies, and its numbers.
//
// Keys and values are vectors of head_dim elements per token and head, cut into segments of `blocksize`; a segment is one
// fp32 scale, fl(largest magnitude / 6), and a 4-bit floating number per element (one sign bit, two of exponent, one of
// mantissa: 0, 1/2, 1, 3/2, 2, 3, 4, 6) -- the numbers that the matrix instructions of gfx950 multiply as they are, so that the
// attention never expands them.  Per page and head, page_size rows of row_bytes (16 bytes hold 32 elements, first element in the low
// nibble, the rest of a row's last 16 bytes zero) and [segments][page_size] scales: the scales of consecutive tokens lie side by side.
#pragma once

#include "qt_common.h"
#include "qt_fp4.h"
#include "qtensor_hip.h"

namespace qt {

struct CacheShape {
    int pages, page_shift, kv_heads, head_dim, segments, segment_shift, row_bytes;
};

struct CachePlaces {
    const int *table, *lengths, *starts;
    long long table_stride;
    int table_pages, batch, tokens;
};

// Checks a cache and its places; false with the error slot set.  `what` is the entry point's name.
bool cache_shape(const char *what, const qtensor_cache *cache, CacheShape &shape);
bool cache_places(const char *what, const qtensor_cache_places *from, CachePlaces &places);

// Lanes that hold a segment, each sixteen bytes of fp32 or bf16: it is no longer than the vector, rounded up to a power of two.
inline int cache_segment_lanes(const CacheShape &shape, bool bf16) {
    int segment = 1 << shape.segment_shift;
    while (segment > 64 && segment / 2 >= shape.head_dim) segment /= 2;
    return segment / (bf16 ? 8 : 4);
}

#if defined(__HIPCC__)
typedef float cache_f32x2 __attribute__((ext_vector_type(2)));

// The sequence of token `token` of a call, given that it is not before sequence b; batch if it belongs to none.
__device__ __forceinline__ int sequence_from(const CachePlaces &at, int token, int b) {
    while (b < at.batch && at.starts[b + 1] <= token) ++b;
    return b;
}

// Number of entries of starts[1 .. batch] that are at or below `token`, by the whole workgroup: the sequence of that token.
__device__ __forceinline__ int sequence_of_block(const CachePlaces &at, int token) {
    int b = 0;
    for (int first = 0; first < at.batch; first += blockDim.x) {
        const int i = first + (int)threadIdx.x;
        const int found = __syncthreads_count(i < at.batch && at.starts[i + 1] <= token);
        b += found;
        if (found < (int)blockDim.x) break;
    }
    return b;
}

// Sequence of `token` and its position there; -1 for a token that is of no sequence.
__device__ __forceinline__ int token_position(const CachePlaces &at, int token, int &b) {
    if (!at.starts) {
        b = token;
        return at.lengths[b] - 1;
    }
    b = sequence_from(at, token, b);
    if (b >= at.batch || token < at.starts[b]) return -1;
    return at.lengths[b] - (at.starts[b + 1] - token);
}

// A lane takes sixteen bytes of a vector: eight elements of bf16, four of fp32.
template <bool BF16>
constexpr int kLaneElements = BF16 ? 8 : 4;

// As they lie in memory, zeros behind the end of a vector.
template <bool BF16>
__device__ __forceinline__ uint4 load_lane(const void *base, long long at, int valid) {
    const uint8_t *p = (const uint8_t *)base + at * (BF16 ? 2 : 4);
    if (valid >= kLaneElements<BF16> && is_aligned16(p)) return load_u32x4<true>(p);
    uint32_t word[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (BF16) word[e] = (2 * e < valid ? ((const uint16_t *)p)[2 * e] : 0u) | ((2 * e + 1 < valid ? ((const uint16_t *)p)[2 * e + 1] : 0u) << 16);
        else word[e] = e < valid ? ((const uint32_t *)p)[e] : 0u;
    }
    return make_uint4(word[0], word[1], word[2], word[3]);
}
template <bool BF16>
__device__ __forceinline__ void unpack_lane(uint4 raw, float *x) {
    const uint32_t word[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (BF16) x[2 * e] = __uint_as_float(word[e] << 16), x[2 * e + 1] = __uint_as_float(word[e] & 0xffff0000u);
        else x[e] = __uint_as_float(word[e]);
    }
}
template <bool BF16, bool STREAM>
__device__ __forceinline__ void store_lane(void *base, long long at, int valid, const float *x) {
    uint8_t *p = (uint8_t *)base + at * (BF16 ? 2 : 4);
    if (valid >= kLaneElements<BF16> && is_aligned16(p)) {
        qt_u32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = BF16 ? floats_to_bf16_pair(x[2 * e], x[2 * e + 1]) : __float_as_uint(x[e]);
        if (STREAM) __builtin_nontemporal_store(y, (qt_u32x4 *)p);
        else *(qt_u32x4 *)p = y;
    } else {
#pragma unroll
        for (int e = 0; e < kLaneElements<BF16>; ++e) {
            if (e >= valid) continue;
            if (BF16) ((uint16_t *)p)[e] = float_to_bf16_bits(x[e]);
            else ((float *)p)[e] = x[e];
        }
    }
}
// Its codes: four bytes, or two.
template <bool BF16>
__device__ __forceinline__ uint32_t load_codes(const uint8_t *p) { return BF16 ? *(const uint32_t *)p : *(const uint16_t *)p; }
template <bool BF16>
__device__ __forceinline__ void store_codes(uint8_t *p, uint32_t word) {
    if (BF16) *(uint32_t *)p = word;
    else *(uint16_t *)p = (uint16_t)word;
}

// Largest of a segment's magnitudes (as bits), which 8 to 64 lanes side by side hold.
__device__ __forceinline__ uint32_t segment_max(uint32_t top, int segment_lanes) {
    top = group_max_u32<8>(top);
    if (segment_lanes >= 16) top = max(top, dpp_u32<0x140>(top));
    if (segment_lanes >= 32) top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
    if (segment_lanes >= 64) top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
    return top;
}
#endif  // __HIPCC__

}  // namespace qt
