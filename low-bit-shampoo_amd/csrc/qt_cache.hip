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
    int lanes, segment_lanes;       // lanes per vector and per segment
    int block_tokens;               // tokens of a workgroup
    FastDiv by_lanes;
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

// A thread's place: a lane's elements of the vectors of one token, whose heads it goes through.  A workgroup takes some
// sixteen tokens of a few heads: codes and scales of a head's consecutive tokens lie side by side, and where the token
// lies is looked up once for all of them.
struct CacheThread {
    int valid;                  // elements of a vector from `first` on; 0: nothing
    int first, token;
    long long line, inside;     // first row of head 0 of the token's page, and the token's row among that; line < 0: it has no page
};
template <bool BF16>
__device__ __forceinline__ CacheThread cache_thread(const CacheCopy &a) {
    CacheThread t;
    const int nth = (int)fastdiv(threadIdx.x, a.by_lanes);
    t.first = ((int)threadIdx.x - nth * a.lanes) * kLaneElements<BF16>;
    t.token = (int)blockIdx.x * a.block_tokens + nth;
    const bool there = nth < a.block_tokens && t.token < a.at.tokens;
    t.valid = there ? max(0, a.shape.head_dim - t.first) : 0;
    t.token = there ? t.token : 0;
    return t;
}
__device__ __forceinline__ void cache_look_up(const CacheCopy &a, CacheThread &t) {
    int b = 0;
    if (a.at.starts) b = sequence_of_block(a.at, (int)blockIdx.x * a.block_tokens);
    t.line = -1, t.inside = 0;
    const int position = t.valid > 0 ? token_position(a.at, t.token, b) : -1;
    const int nth = position >> a.shape.page_shift;
    if (position < 0 || nth >= a.at.table_pages) return;
    const int page = a.at.table[b * a.at.table_stride + nth];
    if ((unsigned)page >= (unsigned)a.shape.pages) return;
    t.line = ((long long)page * a.shape.kv_heads) << a.shape.page_shift;
    t.inside = position & ((1 << a.shape.page_shift) - 1);
}

// Bound by memory once there are some million elements, by the latency of two dependent loads (place, then vectors) and the launch below that:
// 9 prompts of up to 3500 tokens (8 heads of 128, bf16) 26 us, 12 of up to 8192 in fp32 144 us (written and read back 44 and 287: 3.9 and 4.0
// TB/s); the vectors are asked for
// before their place is known, so that both waits are one.  A lane takes sixteen bytes, so that a segment's maximum is a few exchanges
// between neighbours and its codes leave as one store per lane.
//
// A segment is 8, 16 or 32 lanes side by side in bf16, twice as many in fp32.  Largest magnitude by integer maximum of
// the magnitudes' bits (NaN above infinity, so that a segment with a NaN gets a NaN for its scale and reads as NaN),
// scale and quotients by correctly rounded division (qt_divide.h; quotients below 2^-40, which it may round otherwise, are code 0),
// nearest number (ties to the even code, beyond 6 to 6) by the conversion instruction.
template <bool BF16, int HEADS>
__global__ __launch_bounds__(kCacheThreads) void cache_write_kernel(const CacheCopy a) {
    CacheThread t = cache_thread<BF16>(a);
    const int first_head = blockIdx.y * HEADS;
    uint4 raw[HEADS][2];
#pragma unroll
    for (int n = 0; n < HEADS; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            raw[n][i] = load_lane<BF16>(a.vectors.base[i], t.token * a.vectors.token_stride[i] + (first_head + n) * a.vectors.head_stride[i] + t.first,
                                        first_head + n < a.shape.kv_heads ? t.valid : 0);
    cache_look_up(a, t);
    const int segment = t.first >> a.shape.segment_shift;
#pragma unroll
    for (int n = 0; n < HEADS; ++n) {
        const bool there = t.line >= 0 && first_head + n < a.shape.kv_heads;
        const long long line = t.line + ((long long)(first_head + n) << a.shape.page_shift);
        const long long scale_at = line * a.shape.segments + ((long long)segment << a.shape.page_shift) + t.inside;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            constexpr int kEach = kLaneElements<BF16>;
            float x[kEach], y[kEach];
            unpack_lane<BF16>(raw[n][i], x);
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < kEach; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
            top = group_max_u32<8>(top);
            if (a.segment_lanes >= 16) top = max(top, dpp_u32<0x140>(top));
            if (a.segment_lanes >= 32) top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
            if (a.segment_lanes >= 64) top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
            const float scale = __uint_as_float(top) / 6.0f;
            const uint32_t bits = __float_as_uint(scale);
            if (bits >= kFastDivLo && bits <= kFastDivHi) {
                const float r = exact_reciprocal(scale);
#pragma unroll
                for (int e = 0; e < kEach; ++e) y[e] = quotient(x[e], scale, r);
            } else {
                // (zeroes times a scale that is not finite are NaN)
                const bool zero = bits == 0 || top >= 0x7f800000u;
#pragma unroll
                for (int e = 0; e < kEach; ++e) y[e] = zero ? 0.0f : x[e] / scale;
            }
            uint32_t word = 0;
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[0], y[1], 1.0f, 0);
            word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[2], y[3], 1.0f, 1);
            if constexpr (BF16) {
                word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[4], y[5], 1.0f, 2);
                word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, y[6], y[7], 1.0f, 3);
            }
            if (there && t.first < 2 * a.shape.row_bytes) store_codes<BF16>(a.codes[i] + (line + t.inside) * a.shape.row_bytes + t.first / 2, word);
            if (there && (t.first & ((1 << a.shape.segment_shift) - 1)) == 0) a.scales[i][scale_at] = scale;
        }
    }
}

// The reverse, bound by the stores: 5 sequences of 9000 to 32768 tokens (8 heads of 128, bf16) 117 us, 5.4 TB/s; small ones by latency and the
// launch (5 x 777 tokens 5.8 us).  Tokens that the cache does not have come out as zeros.  Large results (of four heads a thread) go past the caches.
template <bool BF16, int HEADS>
__global__ __launch_bounds__(kCacheThreads) void cache_read_kernel(const CacheCopy a) {
    CacheThread t = cache_thread<BF16>(a);
    const int first_head = blockIdx.y * HEADS;
    cache_look_up(a, t);
    const bool there = t.line >= 0;
    const int segment = there ? t.first >> a.shape.segment_shift : 0;
    uint32_t word[HEADS][2];
    float scale[HEADS][2];
#pragma unroll
    for (int n = 0; n < HEADS; ++n) {
        // (what is not there is read from row 0, which every cache has)
        const long long line = there ? t.line + ((long long)min(first_head + n, a.shape.kv_heads - 1) << a.shape.page_shift) : 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            word[n][i] = load_codes<BF16>(a.codes[i] + (line + t.inside) * a.shape.row_bytes + (there ? t.first / 2 : 0));
            scale[n][i] = a.scales[i][line * a.shape.segments + ((long long)segment << a.shape.page_shift) + t.inside];
        }
    }
    if (t.valid <= 0) return;
#pragma unroll
    for (int n = 0; n < HEADS; ++n) {
        if (first_head + n >= a.shape.kv_heads) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float x[kLaneElements<BF16>];
#define QT_EACH(e)                                                                                     \
    {                                                                                                  \
        const cache_f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[n][i], 1.0f, e);            \
        x[2 * e] = there ? p.x * scale[n][i] : 0.0f, x[2 * e + 1] = there ? p.y * scale[n][i] : 0.0f;   \
    }
            QT_EACH(0) QT_EACH(1)
            if constexpr (BF16) { QT_EACH(2) QT_EACH(3) }
#undef QT_EACH
            store_lane<BF16, (HEADS > 1)>(a.vectors.base[i], t.token * a.vectors.token_stride[i] + (first_head + n) * a.vectors.head_stride[i] + t.first,
                                     t.valid, x);
        }
    }
}

template <bool BF16>
void launch_copy(bool write, const CacheCopy &a, hipStream_t stream) {
    // Several heads a thread where there are workgroups enough for every unit: their loads wait together.  Keys of 2^22 / 2^23 / 2^26 elements
    // in bf16: one head 7.2 / 12.7 / 82 us written, 7.6 / 11.7 / 115 read; four 7.7 / 11.5 / 66 and, results past the caches, 7.1 /
    // 8.6 / 54 (of 2^21, read: 5.6 with one, 6.9 with four).
    const long long elements = (long long)a.at.tokens * a.shape.kv_heads * a.shape.head_dim;
    const bool large = elements >= (write ? 1 << 23 : 1 << 22);
    const unsigned blocks = (unsigned)((a.at.tokens + a.block_tokens - 1) / a.block_tokens), heads = (unsigned)a.shape.kv_heads;
    const dim3 one(blocks, heads), few(blocks, (heads + 3) / 4);
    if (write && large) hipLaunchKernelGGL((cache_write_kernel<BF16, 4>), few, dim3(kCacheThreads), 0, stream, a);
    else if (write) hipLaunchKernelGGL((cache_write_kernel<BF16, 1>), one, dim3(kCacheThreads), 0, stream, a);
    else if (large) hipLaunchKernelGGL((cache_read_kernel<BF16, 4>), few, dim3(kCacheThreads), 0, stream, a);
    else hipLaunchKernelGGL((cache_read_kernel<BF16, 1>), one, dim3(kCacheThreads), 0, stream, a);
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
    a.segment_lanes = segment / (keys->is_bf16 ? 8 : 4);
    a.lanes = a.segment_lanes * a.shape.segments;
    a.block_tokens = kCacheThreads / a.lanes;
    a.by_lanes = make_fastdiv((uint32_t)a.lanes);
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
