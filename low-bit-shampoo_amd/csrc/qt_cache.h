// An attention cache held in 4 bits: where a token of a sequence lies, and its numbers.
//
// Keys and values are vectors of head_dim elements per token and head, cut into segments of `blocksize`; a segment is one
// fp32 scale, fl(largest magnitude / 6), and a 4-bit floating number per element (one sign bit, two of exponent, one of
// mantissa: 0, 1/2, 1, 3/2, 2, 3, 4, 6) -- the numbers that the matrix instructions of gfx950 multiply as they are, so that the
// attention never expands them.  Per page and head, page_size rows of row_bytes (16 bytes hold 32 elements, first element in the low
// nibble, the rest of a row's last 16 bytes zero) and [segments][page_size] scales: the scales of consecutive tokens lie side by side.
#pragma once

#include "qt_common.h"
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
#endif  // __HIPCC__

}  // namespace qt
