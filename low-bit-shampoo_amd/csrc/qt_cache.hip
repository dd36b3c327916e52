// Writing a 4-bit attention cache and reading it back (layout: qt_cache.h).
#include "qt_cache.h"
#include "qt_divide.h"

namespace qt {

bool cache_shape(const char *what, const qtensor_cache *cache, CacheShape &s) {
    if (!cache || !cache->codes[0] || !cache->codes[1] || !cache->scales[0] || !cache->scales[1]) {
        set_error(kNullPointer, "%s: null pointer in the cache", what);
        return false;
    }
    const int bs = cache->blocksize, ps = cache->page_size;
    if (bs != 64 && bs != 128 && bs != 256) { set_error(kBadBlocksize, "%s: blocksize %d is not one of 64,128,256", what, bs); return false; }
    if (ps < 16 || ps > 4096 || (ps & (ps - 1)) || cache->head_dim < 1 || cache->head_dim > 256 || cache->kv_heads < 1 || cache->kv_heads > 32767 ||
        cache->pages < 1) {
        set_error(kBadArgument, "%s: needs pages of 16 to 4096 tokens (a power of two), heads of 1 to 256 elements, 1 to 32767 heads and at least one page "
                                "(got %d, %d, %d, %d)", what, ps, cache->head_dim, cache->kv_heads, cache->pages);
        return false;
    }
    for (int i = 0; i < 2; ++i)
        if (!is_aligned(cache->codes[i], 16) || !is_aligned(cache->scales[i], 16)) {
            set_error(kBadArgument, "%s: unaligned cache", what);
            return false;
        }
    s = {cache->pages, __builtin_ctz((unsigned)ps), cache->kv_heads, cache->head_dim, (cache->head_dim + bs - 1) / bs, __builtin_ctz((unsigned)bs),
         16 * ((cache->head_dim + 31) / 32)};
    return true;
}

bool cache_places(const char *what, const qtensor_cache_places *from, CachePlaces &at) {
    if (!from || !from->table || !from->lengths) { set_error(kNullPointer, "%s: null pointer in the places", what); return false; }
    if (from->batch < 1 || from->table_pages < 1 || from->tokens < 0 || from->table_stride < 0 || (!from->starts && from->tokens != from->batch)) {
        set_error(kBadArgument, "%s: needs at least one sequence and page, and one token of each sequence where starts is null "
                                "(got %d sequences, %d pages, %d tokens)", what, from->batch, from->table_pages, from->tokens);
        return false;
    }
    at = {from->table, from->lengths, from->starts, from->table_stride, from->table_pages, from->batch, from->tokens};
    return true;
}

namespace {

constexpr int kCacheThreads = 256;

struct CacheVectors {
    void *base[2];
    long long token_stride[2], head_stride[2];
};

struct CacheCopy {
    CacheShape shape;
    CachePlaces at;
    CacheVectors vectors;
    uint8_t *codes[2];
    float *scales[2];
    int lanes, segment_lanes;       // lanes of eight elements per vector and per segment
    uint32_t items;                 // lanes of all vectors of keys, which take those of the values too
    FastDiv by_lanes, by_heads;
};

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

// Eight elements as they lie in memory (16 bytes of bf16, 32 of fp32), zeros behind the end of a vector.
template <bool BF16>
__device__ __forceinline__ void load_eight(const void *base, long long at, int valid, uint4 *raw) {
    constexpr int kWords = BF16 ? 1 : 2;
    const uint8_t *p = (const uint8_t *)base + at * (BF16 ? 2 : 4);
    if (valid >= 8 && is_aligned16(p)) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) raw[i] = load_u32x4<true>(p + 16 * i);
    } else {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            uint32_t word[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int n = 4 * i + e;
                if (BF16)
                    word[e] = (2 * n < valid ? ((const uint16_t *)p)[2 * n] : 0u) | ((2 * n + 1 < valid ? ((const uint16_t *)p)[2 * n + 1] : 0u) << 16);
                else
                    word[e] = n < valid ? ((const uint32_t *)p)[n] : 0u;
            }
            raw[i] = make_uint4(word[0], word[1], word[2], word[3]);
        }
    }
}
template <bool BF16>
__device__ __forceinline__ void unpack_eight(const uint4 *raw, float *x) {
#pragma unroll
    for (int i = 0; i < (BF16 ? 1 : 2); ++i) {
        const uint32_t word[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (BF16) x[2 * e] = __uint_as_float(word[e] << 16), x[2 * e + 1] = __uint_as_float(word[e] & 0xffff0000u);
            else x[4 * i + e] = __uint_as_float(word[e]);
        }
    }
}

template <bool BF16>
__device__ __forceinline__ void store_eight(void *base, long long at, int valid, const float *x) {
    if (BF16) {
        uint16_t *p = (uint16_t *)base + at;
        if (valid >= 8 && is_aligned16(p)) {
            *(uint4 *)p = make_uint4(floats_to_bf16_pair(x[0], x[1]), floats_to_bf16_pair(x[2], x[3]), floats_to_bf16_pair(x[4], x[5]),
                                     floats_to_bf16_pair(x[6], x[7]));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < valid) p[i] = float_to_bf16_bits(x[i]);
        }
    } else {
        float *p = (float *)base + at;
        if (valid >= 8 && is_aligned16(p)) {
            *(float4 *)p = make_float4(x[0], x[1], x[2], x[3]);
            *(float4 *)(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < valid) p[i] = x[i];
        }
    }
}

// What a lane works on: eight elements of the keys and the values of one head of one token.
struct CacheItem {
    int valid;          // elements of the vector from here on; 0: nothing
    uint32_t lane, token, head;
};
__device__ __forceinline__ CacheItem cache_item(const CacheCopy &a, uint32_t item) {
    CacheItem it;
    const bool there = item < a.items;
    const uint32_t vector = fastdiv(there ? item : 0, a.by_lanes);
    it.lane = (there ? item : 0) - vector * a.lanes;
    it.token = fastdiv(vector, a.by_heads);
    it.head = vector - it.token * a.shape.kv_heads;
    it.valid = there ? max(0, a.shape.head_dim - (int)it.lane * 8) : 0;
    return it;
}

// A lane takes eight elements of a vector; a segment is 8, 16 or 32 lanes side by side.  Largest magnitude by integer maximum of
// the magnitudes' bits (NaN above infinity, so that a segment with a NaN gets a NaN for its scale and reads as NaN),
// scale and quotients by correctly rounded division (qt_divide.h; quotients below 2^-40, which it may round otherwise, are code 0),
// nearest number (ties to the even code, beyond 6 to 6) by the conversion instruction.
template <bool BF16, int ITEMS>
__global__ __launch_bounds__(kCacheThreads) void cache_write_kernel(const CacheCopy a) {
    const uint32_t first = blockIdx.x * (kCacheThreads * ITEMS);
    CacheItem it[ITEMS];
    uint4 raw[ITEMS][2][BF16 ? 1 : 2];
#pragma unroll
    for (int n = 0; n < ITEMS; ++n) {
        it[n] = cache_item(a, first + n * kCacheThreads + threadIdx.x);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            load_eight<BF16>(a.vectors.base[i], it[n].token * a.vectors.token_stride[i] + it[n].head * a.vectors.head_stride[i] + it[n].lane * 8,
                             it[n].valid, raw[n][i]);
    }
    int b = 0;
    if (a.at.starts) b = sequence_of_block(a.at, (int)fastdiv(fastdiv(first, a.by_lanes), a.by_heads));
#pragma unroll
    for (int n = 0; n < ITEMS; ++n) {
        const int position = first + n * kCacheThreads + threadIdx.x < a.items ? token_position(a.at, (int)it[n].token, b) : -1;
        const long long row = position < 0 ? -1 : cache_row(a.shape, a.at, b, position, (int)it[n].head);
        const int segment = (int)(it[n].lane * 8) >> a.shape.segment_shift;
        const long long scale_at = cache_scale_at(a.shape, row) + ((long long)segment << a.shape.page_shift);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float x[8];
            unpack_eight<BF16>(raw[n][i], x);
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
            top = group_max_u32<8>(top);
            if (a.segment_lanes >= 16) top = max(top, dpp_u32<0x140>(top));
            if (a.segment_lanes >= 32) top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
            const float scale = __uint_as_float(top) / 6.0f;
            float y[8];
            const uint32_t bits = __float_as_uint(scale);
            if (bits >= kFastDivLo && bits <= kFastDivHi) {
                const float r = exact_reciprocal(scale);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = quotient(x[e], scale, r);
            } else {
                // (zeroes times a scale that is not finite are NaN)
                const bool zero = bits == 0 || top >= 0x7f800000u;
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = zero ? 0.0f : x[e] / scale;
            }
            uint32_t word = 0;
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[0], y[1], 1.0f, 0);
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[2], y[3], 1.0f, 1);
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[4], y[5], 1.0f, 2);
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[6], y[7], 1.0f, 3);
            if (row >= 0 && (int)it[n].lane * 4 < a.shape.row_bytes) *(uint32_t *)(a.codes[i] + row * a.shape.row_bytes + it[n].lane * 4) = word;
            if (row >= 0 && (it[n].lane & (a.segment_lanes - 1)) == 0) a.scales[i][scale_at] = scale;
        }
    }
}

// The reverse, eight elements a lane; tokens that the cache does not have come out as zeros.
template <bool BF16, int ITEMS>
__global__ __launch_bounds__(kCacheThreads) void cache_read_kernel(const CacheCopy a) {
    const uint32_t first = blockIdx.x * (kCacheThreads * ITEMS);
    int b = 0;
    if (a.at.starts) b = sequence_of_block(a.at, (int)fastdiv(fastdiv(first, a.by_lanes), a.by_heads));
    CacheItem it[ITEMS];
    bool there[ITEMS];
    uint32_t word[ITEMS][2];
    float scale[ITEMS][2];
#pragma unroll
    for (int n = 0; n < ITEMS; ++n) {
        it[n] = cache_item(a, first + n * kCacheThreads + threadIdx.x);
        const int position = it[n].valid > 0 ? token_position(a.at, (int)it[n].token, b) : -1;
        const long long row = position < 0 ? -1 : cache_row(a.shape, a.at, b, position, (int)it[n].head);
        there[n] = row >= 0;
        const long long from = there[n] ? row : 0;       // (every cache has a row 0)
        const int segment = (int)(it[n].lane * 8) >> a.shape.segment_shift;
        const long long scale_at = cache_scale_at(a.shape, from) + ((long long)(there[n] ? segment : 0) << a.shape.page_shift);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            word[n][i] = *(const uint32_t *)(a.codes[i] + from * a.shape.row_bytes + (there[n] ? it[n].lane * 4 : 0));
            scale[n][i] = a.scales[i][scale_at];
        }
    }
#pragma unroll
    for (int n = 0; n < ITEMS; ++n) {
        if (it[n].valid <= 0) continue;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float x[8];
#define QT_EACH(e)                                                                                             \
    {                                                                                                          \
        const cache_f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[n][i], 1.0f, e);                    \
        x[2 * e] = there[n] ? p.x * scale[n][i] : 0.0f, x[2 * e + 1] = there[n] ? p.y * scale[n][i] : 0.0f;     \
    }
            QT_EACH(0) QT_EACH(1) QT_EACH(2) QT_EACH(3)
#undef QT_EACH
            store_eight<BF16>(a.vectors.base[i], it[n].token * a.vectors.token_stride[i] + it[n].head * a.vectors.head_stride[i] + it[n].lane * 8,
                              it[n].valid, x);
        }
    }
}

template <bool BF16>
void launch_copy(bool write, const CacheCopy &a, hipStream_t stream) {
    // several items a thread where there are workgroups enough for every unit: their loads wait together
    const bool large = a.items >= 1u << 21;
    const int items = !large ? 1 : write ? 2 : 4;
    const dim3 grid((a.items + kCacheThreads * items - 1) / (kCacheThreads * items));
    if (write && large) hipLaunchKernelGGL((cache_write_kernel<BF16, 2>), grid, dim3(kCacheThreads), 0, stream, a);
    else if (write) hipLaunchKernelGGL((cache_write_kernel<BF16, 1>), grid, dim3(kCacheThreads), 0, stream, a);
    else if (large) hipLaunchKernelGGL((cache_read_kernel<BF16, 4>), grid, dim3(kCacheThreads), 0, stream, a);
    else hipLaunchKernelGGL((cache_read_kernel<BF16, 1>), grid, dim3(kCacheThreads), 0, stream, a);
}

void copy_cache(const char *what, bool write, const qtensor_cache *cache, const qtensor_cache_places *places, const qtensor_cache_vectors *keys,
                const qtensor_cache_vectors *values, hipStream_t stream) {
    clear_error();
    CacheCopy a;
    if (!cache_shape(what, cache, a.shape) || !cache_places(what, places, a.at)) return;
    if (!keys || !values || (a.at.tokens > 0 && (!keys->base || !values->base))) { set_error(kNullPointer, "%s: null vectors", what); return; }
    const qtensor_cache_vectors *both[2] = {keys, values};
    for (int i = 0; i < 2; ++i) {
        if (both[i]->is_bf16 != keys->is_bf16 || !is_aligned(both[i]->base, keys->is_bf16 ? 2 : 4)) {
            set_error(kBadArgument, "%s: keys and values of one type, aligned to an element", what);
            return;
        }
        a.vectors.base[i] = both[i]->base;
        a.vectors.token_stride[i] = both[i]->token_stride;
        a.vectors.head_stride[i] = both[i]->head_stride;
        a.codes[i] = cache->codes[i];
        a.scales[i] = cache->scales[i];
    }
    if (a.at.tokens == 0) return;
    // a segment is no longer than the vector, rounded up to a power of two
    int segment = cache->blocksize;
    while (segment > 64 && segment / 2 >= cache->head_dim) segment /= 2;
    a.segment_lanes = segment / 8;
    a.lanes = a.segment_lanes * a.shape.segments;
    const long long items = (long long)a.at.tokens * a.shape.kv_heads * a.lanes;
    if (items >= (1LL << 29)) { set_error(kBadArgument, "%s: %d tokens are too many for one call", what, a.at.tokens); return; }
    a.items = (uint32_t)items;
    a.by_lanes = make_fastdiv((uint32_t)a.lanes);
    a.by_heads = make_fastdiv((uint32_t)a.shape.kv_heads);
    if (keys->is_bf16) launch_copy<true>(write, a, stream);
    else launch_copy<false>(write, a, stream);
    launch_ok(what);
}

}  // namespace
}  // namespace qt

extern "C" void qtensor_hip_cache_write(const qtensor_cache *cache, const qtensor_cache_places *places, const qtensor_cache_vectors *keys,
                                        const qtensor_cache_vectors *values, void *stream) {
    qt::copy_cache("cache_write", true, cache, places, keys, values, (hipStream_t)stream);
}

extern "C" void qtensor_hip_cache_read(const qtensor_cache *cache, const qtensor_cache_places *places, const qtensor_cache_vectors *keys,
                                       const qtensor_cache_vectors *values, void *stream) {
    qt::copy_cache("cache_read", false, cache, places, keys, values, (hipStream_t)stream);
}
