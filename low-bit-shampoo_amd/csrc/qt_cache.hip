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
    uint32_t items;                 // lanes of all vectors of keys (of values as many)
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

template <bool BF16>
__device__ __forceinline__ void load_eight(const void *base, long long at, int valid, float *x) {
    if (BF16) {
        const uint16_t *p = (const uint16_t *)base + at;
        if (valid >= 8 && is_aligned16(p)) {
            const uint4 w = *(const uint4 *)p;
            const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = __uint_as_float(v[i] << 16);
                x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = i < valid ? bf16_bits_to_float(p[i]) : 0.0f;
        }
    } else {
        const float *p = (const float *)base + at;
        if (valid >= 8 && is_aligned16(p)) {
            const float4 u = *(const float4 *)p, v = *(const float4 *)(p + 4);
            x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
            x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = i < valid ? p[i] : 0.0f;
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

// A lane takes eight elements of a vector; a segment is 8, 16 or 32 lanes side by side.  Largest magnitude by integer maximum of
// the magnitudes' bits (NaN above infinity, so that a segment with a NaN gets a NaN for its scale and reads as NaN),
// scale and quotients by correctly rounded division, nearest number (ties to the even code, beyond 6 to 6) by the conversion
// instruction.
template <bool BF16>
__global__ __launch_bounds__(kCacheThreads) void cache_write_kernel(const CacheCopy a) {
    const uint32_t item = blockIdx.x * kCacheThreads + threadIdx.x;
    const int which = blockIdx.y;
    int b = 0;
    const uint32_t first_vector = fastdiv(blockIdx.x * kCacheThreads, a.by_lanes);
    if (a.at.starts) b = sequence_of_block(a.at, (int)fastdiv(first_vector, a.by_heads));
    const bool there = item < a.items;
    const uint32_t vector = fastdiv(there ? item : 0, a.by_lanes), lane = (there ? item : 0) - vector * a.lanes;
    const uint32_t token = fastdiv(vector, a.by_heads), head = vector - token * a.shape.kv_heads;
    const int position = there ? token_position(a.at, (int)token, b) : -1;
    const long long row = position < 0 ? -1 : cache_row(a.shape, a.at, b, position, (int)head);
    const int valid = row < 0 ? 0 : a.shape.head_dim - (int)lane * 8;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (valid > 0)
        load_eight<BF16>(a.vectors.base[which], token * a.vectors.token_stride[which] + head * a.vectors.head_stride[which] + lane * 8, valid, x);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    top = group_max_u32<8>(top);
    if (a.segment_lanes >= 16) top = max(top, dpp_u32<0x140>(top));
    if (a.segment_lanes >= 32) top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
    if (row < 0) return;
    const float scale = __uint_as_float(top) / 6.0f;
    const float by = scale == 0.0f ? 1.0f : scale;
    uint32_t word = 0;
    if (top != 0 && top < 0x7f800000u) {      // (zeroes times a scale that is not finite are NaN)
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, x[0] / by, x[1] / by, 1.0f, 0);
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, x[2] / by, x[3] / by, 1.0f, 1);
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, x[4] / by, x[5] / by, 1.0f, 2);
        word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, x[6] / by, x[7] / by, 1.0f, 3);
    }
    if ((int)lane * 4 < a.shape.row_bytes) *(uint32_t *)(a.codes[which] + row * a.shape.row_bytes + lane * 4) = word;
    const int segment = (int)(lane * 8) >> a.shape.segment_shift;
    if ((lane & (a.segment_lanes - 1)) == 0) a.scales[which][cache_scale_at(a.shape, row) + ((long long)segment << a.shape.page_shift)] = scale;
}

// The reverse, eight elements a lane; tokens that the cache does not have come out as zeros.
template <bool BF16>
__global__ __launch_bounds__(kCacheThreads) void cache_read_kernel(const CacheCopy a) {
    const uint32_t item = blockIdx.x * kCacheThreads + threadIdx.x;
    const int which = blockIdx.y;
    int b = 0;
    const uint32_t first_vector = fastdiv(blockIdx.x * kCacheThreads, a.by_lanes);
    if (a.at.starts) b = sequence_of_block(a.at, (int)fastdiv(first_vector, a.by_heads));
    if (item >= a.items) return;
    const uint32_t vector = fastdiv(item, a.by_lanes), lane = item - vector * a.lanes;
    const uint32_t token = fastdiv(vector, a.by_heads), head = vector - token * a.shape.kv_heads;
    const int position = token_position(a.at, (int)token, b);
    const long long row = position < 0 ? -1 : cache_row(a.shape, a.at, b, position, (int)head);
    const int valid = a.shape.head_dim - (int)lane * 8;
    if (valid <= 0) return;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (row >= 0) {
        const uint32_t word = *(const uint32_t *)(a.codes[which] + row * a.shape.row_bytes + lane * 4);
        const int segment = (int)(lane * 8) >> a.shape.segment_shift;
        const float scale = a.scales[which][cache_scale_at(a.shape, row) + ((long long)segment << a.shape.page_shift)];
        const cache_f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 0), q = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 1),
                          r = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 2), s = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, 1.0f, 3);
        x[0] = p.x * scale; x[1] = p.y * scale; x[2] = q.x * scale; x[3] = q.y * scale;
        x[4] = r.x * scale; x[5] = r.y * scale; x[6] = s.x * scale; x[7] = s.y * scale;
    }
    store_eight<BF16>(a.vectors.base[which], token * a.vectors.token_stride[which] + head * a.vectors.head_stride[which] + lane * 8, valid, x);
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
    const dim3 grid((a.items + kCacheThreads - 1) / kCacheThreads, 2);
    auto kernel = write ? (keys->is_bf16 ? cache_write_kernel<true> : cache_write_kernel<false>)
                        : (keys->is_bf16 ? cache_read_kernel<true> : cache_read_kernel<false>);
    hipLaunchKernelGGL(kernel, grid, dim3(kCacheThreads), 0, stream, a);
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
