// Attention over a 4-bit cache for sequences of many queries: prompts, or many heads that share one of the cache (qt_attend.h).
//
// A workgroup takes 128 queries (of all heads that share a head of the cache), thirty-two for each of its four waves, and goes through the
// tokens they see in tiles of 64.  Products of that many queries are bound by what the vector unit does between them, so the codes
// are expanded here, once for all 128: a thread turns 16 bytes of codes into 32 fp16 numbers times their scale in LDS, and the
// scores come out of v_mfma_f32_32x32x16_f16 as exponents, the running maximum already taken off (it is what the sums begin with).
//
// Roundings: keys and values to fp16 (two of 2^-12: the scale and the product), queries times the scale of the scores to fp16, weights to fp16
// (2^-12 each), all against 2^-9 of the result's type; sums, maxima and results in fp32.  fp16 has no range to spare, so keys and values
// are held relative to powers of two that follow the largest scales of the tiles so far (where one outgrows them the workgroup begins again);
// what does not fit beside the largest of its head is computed in fp32 (kUnfit).  Weights are 2^11 times what they are: those of 2^-25 of a query's
// largest keep their bits, those below 2^-36 are dropped.
//
// 4 prompts of 1500 to 8192 tokens, 8 heads of 128 with 4 queries each: 1190 to 1260 us, 840 to 885 TFLOP/s, where a large product of the library
// reaches 1155 in fp16.  By its counters the matrix pipes are busy 38 % of the cycles and the vector units 45 %, at 2.0 GHz; the two waves that a SIMD
// holds wait for 31 % of their time, for one another at a barrier a tile too, though the vector work of a tile is interleaved with its
// products, matrix instruction by matrix instruction.  Heads of 256 leave one wave per unit (registers): 320 TFLOP/s over a
// window of 4096.  Multiplying the 4-bit codes as they are instead, queries in 6-bit pieces, took 1357 us: three instructions for one.
#include "qt_attend.h"

namespace qt {
namespace {

constexpr int kManyTile = 64;
constexpr int kManyShift = 6;
constexpr int kManyLeast = 4;           // tiles of a piece, at least
constexpr float kWeightBits = 11.0f;    // weights are kept times 2^11 ...
constexpr float kSlack = 4.0f;          // ... and the running maximum may lag behind by 4: below 2^15 in fp16
// Keys and values whose scale has the largest exponent so far are held times 2^3; values of up to 2^9 times that still fit (6 * 2 * 2^(3 + 9) <
// 65504) before the power of two has to follow, keys of up to 2^3 times: what queries lose below fp16's normal numbers, 2^-25, is
// multiplied with keys of at most 6 * 2 * 2^(3 + 3) then, 0.006 of an exponent over 256 elements at the very most.
constexpr int kHeldBits = 3, kKeyHeadroom = 3, kValueHeadroom = 9;
// Scales down to 2^-16 of that keep all their bits (1/2 * 2^(3 - 16) is fp16's least normal number).  Smaller values are not left to it, nor are smaller
// keys beside queries of more than 2^6, whose products with the 2^-25 that such keys lose could reach 2^-11.
constexpr int kSpan = 16;
constexpr float kLargeQuery = 64.0f;
constexpr float kLargest = 65504.0f;    // of fp16

enum Event {
    kOutgrown = 1,          // an exponent has outgrown what is held
    kOddValue = 2,          // a scale of a value is not finite
    kHole = 4,              // a token's page is not there
    kUnfit = 8,             // fp16 does not hold a query or a value: the workgroup's part is computed in fp32 (attend_in_fp32)
    kQueryIsLarge = 16, kKeyIsSmall = 32        // nor both together
};
__device__ __forceinline__ bool is_unfit(int met) { return (met & kUnfit) || (met & (kQueryIsLarge | kKeyIsSmall)) == (kQueryIsLarge | kKeyIsSmall); }

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

// Of the tokens 8 (i / 4) + i % 4 of a lane (i < 16; bit i), those up to x.
__device__ __forceinline__ uint32_t tokens_up_to(int x) {
    const int bits = 4 * (x >> 3) + min(x & 7, 3) + 1;
    return x < 0 ? 0u : x >= 27 ? 0xffffu : (1u << (bits & 31)) - 1u;
}

// Place of 16-byte chunk `chunk` of row `row` of expanded codes in LDS.  Chunks of one place of sixteen rows (reads of keys), four chunks of each
// of four rows (a quarter of what a wave writes at a time), and the 64 bytes of each of four rows that half a transposed read takes are
// all on different banks.
template <int DP>
__device__ __forceinline__ int held_place(int row, int chunk) {
    if (DP == 64) return chunk ^ (((row >> 1) & 3) | ((((row >> 1) ^ (row >> 3)) & 1) << 2));
    const int a = row & 3, j = (row >> 2) & 3;
    return chunk ^ ((a << 2) | (a ^ j)) ^ (DP == 256 ? ((chunk >> 4) & 1) << 1 : 0);
}

// Which of a lane's tokens of a tile have a page (bit 16 t + i: token 32 t + 8 (i / 4) + 4 half + i % 4).
__device__ __forceinline__ uint32_t pages_there(const AttendArgs &a, const int *table, int end, int base) {
    uint32_t see = 0;
#pragma unroll 1
    for (int group = 0; group < kManyTile / 16; ++group) {
        const int token = base + 16 * group;
        if (token >= end) break;
        // eight of a lane's tokens lie in every group of sixteen, and past the end no query sees any
        if ((unsigned)table[token >> a.shape.page_shift] < (unsigned)a.shape.pages) see |= 0xffu << (8 * group);
    }
    return see;
}
// A bit for every 64 elements of values in whose scale there is a NaN or an infinity, over the tokens `first` to `end` that a query at
// `position` sees.
__device__ __forceinline__ uint32_t values_not_finite(const AttendArgs &a, const int *table, int first, int end, int position, int head) {
    uint32_t found = 0;
#pragma unroll 1
    for (int token = first; token < min(end, position + 1); ++token) {
        if (a.window && position - token >= a.window && token >= a.sinks) continue;
        const int page = table[token >> a.shape.page_shift];
        if ((unsigned)page >= (unsigned)a.shape.pages) continue;
        const long long line = ((long long)page * a.shape.kv_heads + head) << a.shape.page_shift;
#pragma unroll 1
        for (int u = 0; u < 4; ++u) {
            const int segment = (64 * u) >> a.shape.segment_shift;
            if (segment >= a.shape.segments) break;
            const float by = a.scales[1][line * a.shape.segments + ((long long)segment << a.shape.page_shift) + (token & ((1 << a.shape.page_shift) - 1))];
            if (!(by - by == 0.0f)) found |= 1u << u;
        }
    }
    return found;
}

// Scores of an infinite query are infinities of either sign or NaN, and the formula's weights NaN; minus infinities alone would pass for tokens that
// are not seen.
__device__ __forceinline__ float nan_if_infinite(float x) { return __builtin_fmaf(x, 0.0f, x); }

// A workgroup's part of the work: a piece of the tokens that 128 queries see.
struct ManyPart {
    AttendWork w;
    SequenceView v;                     // of these queries
    int all_rows, first_row;
    int tile_from, tile_to;
};
__device__ __forceinline__ bool find_part(const AttendArgs &a, uint32_t index, ManyPart &p) {
    if (!find_work<kRowsOfMany, kManyShift, true>(a, index, p.w, p.v)) return false;
    p.all_rows = p.v.count * a.group;
    p.first_row = first_row_of<kRowsOfMany>(p.all_rows, p.w.row_tile);
    const int last = p.v.first_position + min(p.first_row + kRowsOfMany - 1, p.all_rows - 1) / a.group;
    p.v.end = max(0, min(p.v.end, last + 1));
    view_tokens<kManyShift>(a, p.v, p.v.first_position + p.first_row / a.group, p.v.end);
    const int per_piece = (p.v.tiles + p.w.pieces - 1) / p.w.pieces;
    p.tile_from = min(p.w.piece * per_piece, p.v.tiles), p.tile_to = min(p.tile_from + per_piece, p.v.tiles);
    return true;
}

// What a workgroup does whose numbers fp16 does not hold: its queries one by one, a wave for each, in fp32 from the cache as it is.  Scores
// with a token per lane, results with DP / 64 elements per lane.  160 to 200 times slower (a prompt of 4096 tokens, 8 heads with 4 queries each, of 64 /
// 128 / 256 elements: 23, 36 and 113 ms, otherwise 0.14, 0.19 and 0.56), for inputs that are rare: largest elements of queries and keys that multiply
// to more than 2^21, values 2^16 below the largest of their head.  A function of its own that finds its work once more, so
// that nothing of this takes registers in the loop before it (inlined: 1.2 % of whole prompts).
template <int DP>
__device__ __attribute__((noinline)) void attend_in_fp32(const AttendArgs QT_CONSTANT *arguments, uint32_t index) {
    const AttendArgs &a = *(const AttendArgs *)arguments;
    ManyPart p;
    if (!find_part(a, __builtin_amdgcn_readfirstlane(index), p)) return;
    const AttendWork &w = p.w;
    const SequenceView &v = p.v;
    const int first_row = p.first_row;
    constexpr int kEach = DP / 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, d = lane * kEach, page_mask = (1 << a.shape.page_shift) - 1;
    const int *table = a.at.table + (long long)w.b * a.at.table_stride;
#pragma unroll 1
    for (int nth = 32 * wave; nth < min(32 * wave + 32, p.all_rows - first_row); ++nth) {
        const int row = first_row + nth, token = v.start + row / a.group, head = w.head * a.group + row % a.group;
        const int position = v.first_position + row / a.group;
        const uint16_t *query = (const uint16_t *)a.q + token * a.q_token + head * a.q_head;
        float best = -__builtin_inff(), sum = 0.0f, y[kEach] = {}, q[kEach];
#pragma unroll
        for (int e = 0; e < kEach; ++e) q[e] = d + e < a.shape.head_dim ? __uint_as_float((uint32_t)query[d + e] << 16) : 0.0f;
#pragma unroll 1
        for (int k = p.tile_from; k < p.tile_to; ++k) {
            const int base = (k < v.sink_tiles ? k : v.first_tile + k - v.sink_tiles) * kManyTile, mine = base + lane;
            const int page = mine < v.end ? table[mine >> a.shape.page_shift] : -1;
            const bool see = (unsigned)page < (unsigned)a.shape.pages && mine <= position && (!a.window || position - mine < a.window || mine < a.sinks);
            const long long line = ((long long)(see ? page : 0) * a.shape.kv_heads + w.head) << a.shape.page_shift;
            float score = 0.0f;
#pragma unroll 1
            for (int from = 0; from < a.shape.head_dim; from += 32) {
                const uint4 codes = *(const uint4 *)(a.codes[0] + (line + (mine & page_mask)) * a.shape.row_bytes + from / 2);
                const float by = a.scales[0][line * a.shape.segments + ((long long)(from >> a.shape.segment_shift) << a.shape.page_shift) + (mine & page_mask)];
                const uint32_t word[4] = {codes.x, codes.y, codes.z, codes.w};
                const int lanes = from / kEach;         // who has these elements of the query
                auto add = [&](cache_f32x2 two, int e) __attribute__((always_inline)) {
                    const float one = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(q[e % kEach]), lanes + e / kEach));
                    const float next = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(q[(e + 1) % kEach]), lanes + (e + 1) / kEach));
                    score = __builtin_fmaf(one, two.x * by, score), score = __builtin_fmaf(next, two.y * by, score);
                };
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    add(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[i], 1.0f, 0), 8 * i), add(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[i], 1.0f, 1), 8 * i + 2);
                    add(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[i], 1.0f, 2), 8 * i + 4), add(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[i], 1.0f, 3), 8 * i + 6);
                }
            }
            score = see ? score * a.factor : -__builtin_inff();
            float top = fmaxf(best, score);
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
            const float zero = top == -__builtin_inff() ? 0.0f : top, fade = __builtin_amdgcn_exp2f(best - zero);
            const float weight = see ? __builtin_amdgcn_exp2f(score - zero) : 0.0f;
            float all = weight;
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) all += __shfl_xor(all, off, 64);
            sum = __builtin_fmaf(sum, fade, all), best = top;
#pragma unroll
            for (int e = 0; e < kEach; ++e) y[e] *= fade;
            const unsigned long long seen = __ballot(see);
            const int segment = min(d, a.shape.head_dim - 1) >> a.shape.segment_shift, byte = min(d, 2 * a.shape.row_bytes - kEach) / 2;
#pragma unroll 8
            for (int from = 0; from < kManyTile; ++from) {
                const bool here = (seen >> from) & 1;
                const int inside = (base + from) & page_mask;
                const float by = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), from));
                const long long at = ((long long)(here ? (int)__builtin_amdgcn_readlane(page, from) : 0) * a.shape.kv_heads + w.head) << a.shape.page_shift;
                const float scale = a.scales[1][at * a.shape.segments + ((long long)segment << a.shape.page_shift) + inside];
                const uint8_t *codes = a.codes[1] + (at + inside) * a.shape.row_bytes + byte;
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    const cache_f32x2 two = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[e / 2], 1.0f, 0);
                    const float more = __builtin_fmaf(by, ((d + e) & 1 ? two.y : two.x) * scale, y[e]);
                    y[e] = here ? more : y[e];
                }
            }
        }
        float *part = a.partial + ((long long)(w.slot + w.piece) * kRowsOfMany + nth) * (DP + 2);
        if (w.pieces > 1 && lane == 0) part[0] = best, part[1] = sum;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            if (w.pieces > 1) part[2 + d + e] = y[e];
            else if (d + e < a.shape.head_dim)
                store_result<true>(a, token * a.out_token + head * a.out_head + d + e, sum == 0.0f ? 0.0f : y[e] / sum);
        }
    }
}

template <int DP>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void attend_many_kernel(const AttendArgs a) {
    constexpr int kSteps = DP / 16, kDTiles = DP / 32, kChunks = DP / 32, kRow = DP * 2;
    constexpr int kEach = DP == 256 ? 2 : 1;            // chunks of keys and of values a thread stages (heads of 64: of one of the two)
    constexpr int kKinds = DP == 64 ? 1 : 2;
    __shared__ __attribute__((aligned(16))) uint8_t s_keys[2][kManyTile * kRow];
    __shared__ __attribute__((aligned(16))) uint8_t s_values[2][kManyTile * kRow];
    __shared__ int s_exponent[2];                       // largest exponents of a scale of keys and values so far
    __shared__ int s_event[3];                          // of three tiles in turn, what has been met (Event)

    ManyPart p;
    if (!find_part(a, blockIdx.x, p)) return;
    const AttendWork &w = p.w;
    const SequenceView &v = p.v;
    const int all_rows = p.all_rows, first_row = p.first_row, tile_from = p.tile_from, tile_to = p.tile_to;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, column = lane & 31, half = lane >> 5;
    const int my_row = min(first_row + 32 * wave + column, all_rows - 1);
    const bool mine = first_row + 32 * wave + column < all_rows;
    const int my_token = v.start + my_row / a.group, my_head = w.head * a.group + my_row % a.group;
    const int position = v.first_position + my_row / a.group;
    const int behind = a.window ? max(max(position, 0) - a.window, -1) : -1;         // last token behind the window
    // positions of this wave's queries and of all of the workgroup's; a query may stand behind all tokens that the table has pages for
    const int seen_from = a.window ? max(0, max(0, v.first_position + first_row / a.group) - (a.window - 1)) : 0;        // (by any, sinks aside)
    const int lowest = v.first_position + min(first_row + 32 * wave, all_rows - 1) / a.group;
    const int highest = v.first_position + min(first_row + 32 * wave + 31, all_rows - 1) / a.group;
    const int *table = a.at.table + (long long)w.b * a.at.table_stride;
    const int page_mask = (1 << a.shape.page_shift) - 1, chunks = a.shape.row_bytes >> 4;
    auto tile_at = [&](int k) __attribute__((always_inline)) { return (k < v.sink_tiles ? k : v.first_tile + k - v.sink_tiles) * kManyTile; };

    // What this thread stages of a tile: chunk `my_chunk` of the tokens stage_row(i).  A wave's tokens lie in one group of sixteen, so in one
    // page (heads of 64: in two; the first two waves stage keys, the others values).
    const int my_chunk = lane & (kChunks - 1);
    auto stage_row = [&](int i) __attribute__((always_inline)) { return DP == 64 ? 32 * (wave & 1) + (lane >> 1) : DP == 128 ? 16 * wave + (lane >> 2) : 32 * i + 8 * wave + (lane >> 3); };
    constexpr int kPages = DP == 64 ? 2 : kEach;
    const int chunk_byte = 16 * min(my_chunk, chunks - 1), segment = min((32 * my_chunk) >> a.shape.segment_shift, a.shape.segments - 1) << a.shape.page_shift;
    int page[kPages];
    auto load_pages = [&](int k) __attribute__((always_inline)) {
        const int base = tile_at(k);
#pragma unroll
        for (int i = 0; i < kPages; ++i) {
            const int token = base + (DP == 64 ? 32 * (wave & 1) + 16 * i : DP == 128 ? 16 * wave : 32 * i + 8 * wave);
            page[i] = table[min(token, v.end - 1) >> a.shape.page_shift];
        }
    };
    i32x4 chunk[kKinds][kEach];
    float scale[kKinds][kEach];
    bool there[kEach], hole[kEach];
    auto load_tile = [&](int k) __attribute__((always_inline)) {
        const int base = tile_at(k);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int token = base + stage_row(i);
            int p = __builtin_amdgcn_readfirstlane(page[i]);
            if (DP == 64) p = lane < 32 ? p : __builtin_amdgcn_readfirstlane(page[kPages - 1]);
            there[i] = (unsigned)p < (unsigned)a.shape.pages && token < v.end && (token >= seen_from || token < a.sinks);
            hole[i] = (unsigned)p >= (unsigned)a.shape.pages && token < v.end;
            const long long line = ((long long)((unsigned)p < (unsigned)a.shape.pages ? p : 0) * a.shape.kv_heads + w.head) << a.shape.page_shift;
            const long long code_at = line * a.shape.row_bytes, scale_at = line * a.shape.segments;
            const uint32_t in_page = token & page_mask;
#pragma unroll
            for (int n = 0; n < kKinds; ++n) {
                const int kind = DP == 64 ? wave >> 1 : n;
                chunk[n][i] = *(const i32x4 *)((kind == 0 ? a.codes[0] : a.codes[1]) + code_at + (in_page * (uint32_t)a.shape.row_bytes + chunk_byte));
                scale[n][i] = *((kind == 0 ? a.scales[0] : a.scales[1]) + scale_at + (in_page + segment));
            }
        }
    };

    // places in LDS: of this lane's first operands and of what it stages (held_place: other chunks and rows differ by constants)
    const int value_row = 4 * half + ((lane & 15) >> 2);
    const uint32_t key_place = column * kRow + 16 * held_place<DP>(column, half);
    const uint32_t value_place = value_row * kRow + 16 * held_place<DP>(value_row, 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) + 8 * (lane & 1);
    const uint32_t stage_place = stage_row(0) * kRow + 16 * held_place<DP>(stage_row(0), 4 * my_chunk);

    f16x8 query[kSteps];
    f32x16 result[kDTiles] = {}, below;         // below: what the sums of the scores begin with, minus the running maximum
    float best = -__builtin_inff(), sum = 0.0f;
    int met = 0;                                // events of all tiles so far
    int exponent[2] = {1, 1};                   // of the largest scales of keys and values that are held

    // This lane's eight elements of every sixteen of its query, zeros behind its end.
    const uint16_t *my_query = (const uint16_t *)a.q + my_token * a.q_token + my_head * a.q_head;
    auto load_query_chunks = [&](uint4 *raw) __attribute__((always_inline)) {
        const int last = a.shape.head_dim - 1;
        if (a.q_in_eights) {
#pragma unroll
            for (int h = 0; h < kSteps; ++h) {
                const int d = 16 * h + 8 * half;
                raw[h] = *(const uint4 *)(my_query + (d <= last ? d : 0));
                if (d > last) raw[h] = make_uint4(0, 0, 0, 0);
            }
        } else {
            int from = 8 * half;
            asm volatile("" : "+v"(from));          // (nothing of this is worked out ahead for the other way)
#pragma unroll
            for (int h = 0; h < kSteps; ++h) {
                uint32_t word[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int d = 16 * h + from + 2 * e;
                    const uint32_t x = my_query[min(d, last)], y = my_query[min(d + 1, last)];
                    word[e] = (d <= last ? x : 0u) | ((d + 1 <= last ? y : 0u) << 16);
                }
                raw[h] = make_uint4(word[0], word[1], word[2], word[3]);
            }
        }
    };
    auto take_query = [&](const uint4 *raw) __attribute__((always_inline)) {
        const int up = exponent[0] - 127 - kHeldBits;
        float top = 0.0f;
#pragma unroll
        for (int h = 0; h < kSteps; ++h) {
            const uint32_t word[4] = {raw[h].x, raw[h].y, raw[h].z, raw[h].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = __builtin_amdgcn_ldexpf(nan_if_infinite(__uint_as_float(word[e] << 16)) * a.factor, up);
                const float y = __builtin_amdgcn_ldexpf(nan_if_infinite(__uint_as_float(word[e] & 0xffff0000u)) * a.factor, up);
                top = fmaxf(top, fmaxf(fabsf(x), fabsf(y)));
                query[h][2 * e] = (_Float16)x, query[h][2 * e + 1] = (_Float16)y;
            }
        }
        if (__builtin_expect(top > kLargeQuery, 0)) atomicOr(&s_event[0], top > kLargest ? kUnfit : kQueryIsLarge);
    };

    // Expands this thread's chunks into `buffer`, a word (eight elements) of a chunk at a time: kSteps of them.  Before them: notes in
    // s_event[slot] what the workgroup has to know.
    _Float16 scaled[kKinds][kEach];
    auto stage_scales = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < kKinds; ++n)
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int kind = DP == 64 ? wave >> 1 : n;
                float by = there[i] ? scale[n][i] : 0.0f;
                const int bits = (int)((__float_as_uint(by) >> 23) & 0xff), held = kind == 0 ? exponent[0] : exponent[1];
                const int least = max(held - kSpan, 0);
                // (what is within, but for zeros, is so by one comparison)
                if (__builtin_expect(((uint32_t)(bits - least) > (uint32_t)(min(held + (kind == 0 ? kKeyHeadroom : kValueHeadroom), 254) - least)) | hole[i], 0)) {
                    if (hole[i]) {
                        atomicOr(&s_event[slot], kHole);
                    } else if (bits == 255) {
                        if (kind == 1) {
                            atomicOr(&s_event[slot], kOddValue);
                            by = 0.0f;
                        }
                    } else if (bits > held) {
                        atomicMax(&s_exponent[kind], bits);
                        atomicOr(&s_event[slot], kOutgrown);
                    } else if (by != 0.0f) {
                        atomicOr(&s_event[slot], kind == 0 ? kKeyIsSmall : kUnfit);
                    }
                }
                scaled[n][i] = (_Float16)__builtin_amdgcn_ldexpf(by, 127 + kHeldBits - held);
            }
    };
    auto stage_word = [&](int buffer, int piece) __attribute__((always_inline)) {
        const int n = piece / (4 * kEach), i = piece / 4 % kEach, e = piece % 4, kind = DP == 64 ? wave >> 1 : n;
        const f16x2 times = {scaled[n][i], scaled[n][i]};
        const uint32_t word = (uint32_t)chunk[n][i][e];
        const f16x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, 1.0f, 0) * times, x1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, 1.0f, 1) * times,
                    x2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, 1.0f, 2) * times, x3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, 1.0f, 3) * times;
        QT_LDS uint8_t *area = kind == 0 ? (QT_LDS uint8_t *)s_keys[0] : (QT_LDS uint8_t *)s_values[0];
        *(QT_LDS f16x8 *)(area + buffer * (kManyTile * kRow) + (stage_place ^ (16 * e)) + 32 * i * kRow) =
            (f16x8){x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
    };
    auto stage_all = [&](int buffer, int slot) __attribute__((always_inline)) {
        stage_scales(slot);
#pragma unroll
        for (int piece = 0; piece < kSteps; ++piece) stage_word(buffer, piece);
    };
    if (threadIdx.x < 2) s_exponent[threadIdx.x] = 1;
    // (A later tile may hold scales that have outgrown what the first ones set: the workgroup begins again then, with the exponents that it has
    // found, which is rare and keeps the loop free of everything that would have to be corrected.)
    bool again = tile_from < tile_to;
    int event = 0;
    while (again) {
    again = false;
#pragma unroll
    for (int d = 0; d < kDTiles; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) result[d][i] = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) below[i] = 0.0f;
    best = -__builtin_inff(), sum = 0.0f;
    {
        __syncthreads();
        if (threadIdx.x < 3) s_event[threadIdx.x] = 0;
        uint4 raw[kSteps];
        load_pages(tile_from);
        load_query_chunks(raw);
        load_tile(tile_from);
        load_pages(min(tile_from + 1, tile_to - 1));
        __syncthreads();
        // the first tile sets the exponents
#pragma unroll
        for (int n = 0; n < kKinds; ++n) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const uint32_t bits = there[i] ? (__float_as_uint(scale[n][i]) >> 23) & 0xff : 0u;
                if (bits < 255) top = max(top, bits);
            }
            top = group_max_u32<64>(top);
            if (lane == 0) atomicMax(&s_exponent[DP == 64 ? wave >> 1 : n], (int)top);
        }
        __syncthreads();
        exponent[0] = s_exponent[0], exponent[1] = s_exponent[1];
        take_query(raw);
        stage_all(0, 0);
        __syncthreads();
        met = event = __builtin_amdgcn_readfirstlane(s_event[0]);
    }
    if (is_unfit(met)) break;
    // The running maximum follows where a score is more than 2^4 above it (scores are relative to it and to 2^-11), in both halves of a
    // column; `done`: weights of the tile that are not in the result yet.
    f16x8 weight[4];
    auto follow = [&](float top, f32x16 &score, int done) __attribute__((always_inline)) {
        const bool first = best == -__builtin_inff();
        if (!__ballot(top > (first ? -__builtin_inff() : kWeightBits + kSlack))) return;
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float up = first ? top : fmaxf(top - kWeightBits, 0.0f);          // what the maximum rises by
        const bool rises = up != -__builtin_inff();
        const float fade = first ? 0.0f : __builtin_amdgcn_exp2f(-up), shift = rises ? (first ? up - kWeightBits : up) : 0.0f;
        if (rises) best = first ? up : best + up;
        sum *= fade;
#pragma unroll
        for (int d = 0; d < kDTiles; ++d) result[d] *= fade;
        const _Float16 fade16 = (_Float16)fade;
#pragma unroll
        for (int n = 0; n < 2; ++n)
            if (n < done) weight[n] *= fade16;
#pragma unroll
        for (int i = 0; i < 16; ++i) score[i] -= shift;
        const float under = best == -__builtin_inff() ? 0.0f : kWeightBits - best;
#pragma unroll
        for (int i = 0; i < 16; ++i) below[i] = under;
    };
    // weights of scores 2 j and 2 j + 1 of half a tile
    auto weigh = [&](const f32x16 &score, int t, int j) __attribute__((always_inline)) {
        const float p = __builtin_amdgcn_exp2f(score[2 * j]), q = __builtin_amdgcn_exp2f(score[2 * j + 1]);
        const f16x2 both = __builtin_convertvector((cache_f32x2){p, q}, f16x2), ones = {(_Float16)1.0f, (_Float16)1.0f};
        sum = __builtin_amdgcn_fdot2(both, ones, sum, false);       // of the weights as they are multiplied, in fp32
        weight[2 * t + (j >> 2)][2 * j & 7] = both[0];
        weight[2 * t + (j >> 2)][(2 * j & 7) + 1] = both[1];
    };
    auto largest = [&](const f32x16 &score) __attribute__((always_inline)) {
        float top = score[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, score[i]);
        return top;
    };

    // Half a tile's products are interleaved with vector work of the other half or of the next tile: scores of the second half with the weights
    // of the first, values of the first with the weights of the second, values of the second with expanding the next tile.  kSteps matrix instructions
    // each, and as much vector work as fits beside them.
    int slot = 0;
    for (int k = tile_from; k < tile_to; ++k) {
        const int base = tile_at(k), buffer = (k - tile_from) & 1, next_slot = slot == 2 ? 0 : slot + 1;
        const bool more = k + 1 < tile_to;
        if (threadIdx.x == 0) s_event[next_slot == 2 ? 0 : next_slot + 1] = 0;      // (the tile before's, which all have read)
        if (more) {
            load_tile(k + 1);
            load_pages(min(k + 2, tile_to - 1));
        }
        {
            const bool full = (base + kManyTile - 1 <= min(lowest, v.end - 1)) & (!a.window | (highest - base < a.window) | (base + kManyTile <= a.sinks)) & !(event & kHole);
            f32x16 score[2];
            f16x8 ahead[2][4];
            // Operands are read from LDS four matrix instructions ahead of those that take them.  A lane's places differ by constants: by exclusive
            // ors where chunks do, by offsets where rows do (each kept as one register and worked out anew for every tile: kept apart, the
            // places would take more registers than there are).
            uint32_t key_at = buffer * (kManyTile * kRow) + key_place, value_at = buffer * (kManyTile * kRow) + value_place;
            asm volatile("" : "+v"(key_at), "+v"(value_at));
            auto read_keys = [&](int t, int first, f16x8 *to) __attribute__((always_inline)) {
#pragma unroll
                for (int h = first; h < first + 4; ++h)
                    to[h - first] = *(const QT_LDS f16x8 *)((const QT_LDS uint8_t *)s_keys[0] + (key_at ^ (32 * h ^ (h >= 8 ? 32 : 0))) + 32 * t * kRow);
            };
            auto read_values = [&](int t, int first, f16x8 *to) __attribute__((always_inline)) {
#pragma unroll
                for (int f = first; f < first + 4; ++f)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int n = 2 * t + f / kDTiles, d = f % kDTiles;
                        const uint32_t at = (value_at ^ (64 * d ^ (d >= 4 ? 32 : 0) ^ (DP == 64 ? 64 * e : 32 * e))) + (16 * n + 8 * e) * kRow;
                        const i16x4 part = __builtin_amdgcn_ds_read_tr16_b64_v4i16((QT_LDS i16x4 *)((QT_LDS uint8_t *)s_values[0] + at));
                        const f16x4 four = __builtin_bit_cast(f16x4, part);
#pragma unroll
                        for (int x = 0; x < 4; ++x) to[f - first][4 * e + x] = four[x];
                    }
            };
            uint32_t see = 0xffffffffu;
            if (!full) {
                const int x = min(position, v.end - 1) - base - 4 * half;
                see = tokens_up_to(x) | (tokens_up_to(x - 32) << 16);
                if (a.window) {
                    const int y = behind - base - 4 * half, z = a.sinks - 1 - base - 4 * half;
                    see &= ~(tokens_up_to(y) | (tokens_up_to(y - 32) << 16)) | (tokens_up_to(z) | (tokens_up_to(z - 32) << 16));
                }
                if (event & kHole) see &= pages_there(a, table, v.end, base);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_setprio(1);
                if (t == 0) read_keys(0, 0, ahead[0]);
#pragma unroll
                for (int m = 0; m < kSteps; ++m) {
                    if (m % 4 == 0) {
                        if (m + 4 < kSteps) read_keys(t, m + 4, ahead[(m >> 2 & 1) ^ 1]);
                        else if (t == 0) read_keys(1, 0, ahead[(m >> 2 & 1) ^ 1]);
                        else read_values(0, 0, ahead[(m >> 2 & 1) ^ 1]);
                    }
                    score[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ahead[(m >> 2) & 1][m & 3], query[m], m == 0 ? below : score[t], 0, 0, 0);
                    if (t == 1) {
#pragma unroll
                        for (int j = 8 * m / kSteps; j < 8 * (m + 1) / kSteps; ++j) weigh(score[0], 0, j);
                        __builtin_amdgcn_sched_barrier(0);
                    } else if (m % 4 == 3) {
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                if (t == 1) asm volatile("" : "+v"(weight[0]), "+v"(weight[1]), "+v"(sum));      // (made here, beside the products)
                __builtin_amdgcn_s_setprio(0);
                // (the number of groups of four is even or, for heads of 64, one: what is read ahead across the turn lies in the other four registers)
                if constexpr (kSteps == 4) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) ahead[0][e] = ahead[1][e];
                }
                if (!full) {
                    asm volatile("" : "+v"(see));           // (tested here, not ahead of the products)
#pragma unroll
                    for (int i = 0; i < 16; ++i) score[t][i] = see & (1u << (16 * t + i)) ? score[t][i] : -__builtin_inff();
                }
                follow(largest(score[t]), score[t], 2 * t);
            }
            if (more) stage_scales(next_slot);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int m = 0; m < kSteps; ++m) {
                    if (m % 4 == 0) {
                        if (m + 4 < kSteps) read_values(t, m + 4, ahead[(m >> 2 & 1) ^ 1]);
                        else if (t == 0) read_values(1, 0, ahead[(m >> 2 & 1) ^ 1]);
                    }
                    result[m % kDTiles] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ahead[(m >> 2) & 1][m & 3], weight[2 * t + m / kDTiles], result[m % kDTiles], 0, 0, 0);
                    if (t == 0) {
#pragma unroll
                        for (int j = 8 * m / kSteps; j < 8 * (m + 1) / kSteps; ++j) weigh(score[1], 1, j);
                    } else {
                        stage_word(buffer ^ 1, m);      // (without a next tile: of this one once more, which nobody reads)
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                __builtin_amdgcn_s_setprio(0);
                if constexpr (kSteps == 4) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) ahead[0][e] = ahead[1][e];
                }
            }
        }
        __syncthreads();
        if (more) event = __builtin_amdgcn_readfirstlane(s_event[next_slot]);
        met |= event;
        slot = next_slot;
        if (is_unfit(met)) break;
        if (event & kOutgrown) {
            again = true;
            break;
        }
    }
    }
    if (__builtin_expect(is_unfit(met), 0)) {
        attend_in_fp32<DP>((const AttendArgs QT_CONSTANT *)__builtin_amdgcn_kernarg_segment_ptr(), blockIdx.x);        // (`a`, the kernel's only argument)
        return;
    }
    sum += __shfl_xor(sum, 32, 64);
    if (!mine) return;
    // values that are not finite were staged as zeros: what is multiplied with one that it sees is NaN.  (Looked for here, once more over
    // all of this piece's tokens, only where there was one at all.)
    uint32_t poison = 0;
    if (__builtin_expect(met & kOddValue, 0)) {
#pragma unroll 1
        for (int k = tile_from; k < tile_to; ++k) poison |= values_not_finite(a, table, tile_at(k), min(v.end, tile_at(k) + kManyTile), position, w.head);
    }
    // four consecutive elements of a result at a time (of a piece: without the 2^11 of its weights)
    const int from_held = exponent[1] - 127 - kHeldBits;
    const float one = __builtin_amdgcn_exp2f(-kWeightBits), by = w.pieces > 1 ? one : sum == 0.0f ? 0.0f : 1.0f / sum;
    float *part = a.partial + ((long long)(w.slot + w.piece) * kRowsOfMany + 32 * wave + column) * (DP + 2);
    const long long at = (long long)my_token * a.out_token + (long long)my_head * a.out_head;
    if (w.pieces > 1 && half == 0) part[0] = best, part[1] = sum * one;
#pragma unroll
    for (int d = 0; d < kDTiles; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int element = 32 * d + 2 * i + 4 * half;
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[e] = __builtin_amdgcn_ldexpf(result[d][i + e] * by, from_held);
                if (poison >> (d / 2) & 1) y[e] = __builtin_nanf("");
            }
            if (w.pieces > 1) {
                *(float2 *)(part + 2 + element) = make_float2(y[0], y[1]);
                *(float2 *)(part + 4 + element) = make_float2(y[2], y[3]);
            } else {
                uint16_t *to = (uint16_t *)a.out + at + element;
                if (element + 4 <= a.shape.head_dim && (reinterpret_cast<uintptr_t>(to) & 7) == 0) {
                    *(uint2 *)to = make_uint2(floats_to_bf16_pair(y[0], y[1]), floats_to_bf16_pair(y[2], y[3]));
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (element + e < a.shape.head_dim) to[e] = float_to_bf16_bits(y[e]);
                }
            }
        }
}

// Joins the pieces of every row of tiles that was cut, a wave per query: what the pieces count for first, a piece per lane, then a share of
// them per group of DP / 4 lanes.  Reads each partial result once; bound by the latency of dependent loads, so the queries of a row
// of tiles are spread over as many workgroups (gridDim.y) as fill the device, each of which has to find its work first.
template <int DP>
__global__ __launch_bounds__(256) void attend_join_many_kernel(const AttendArgs a) {
    constexpr int kGroups = 256 / DP, kNext = kRowsOfMany * (DP + 2);
    AttendWork w;
    SequenceView v;
    if (!find_work<kRowsOfMany, kManyShift, false>(a, blockIdx.x, w, v) || w.pieces == 1) return;
    const int rows = v.count * a.group, first = first_row_of<kRowsOfMany>(rows, w.row_tile), each = kRowsOfMany / gridDim.y;
    const int lane = threadIdx.x & 63, group = lane / (DP / 4), d = lane % (DP / 4) * 4;
    for (int r = blockIdx.y * each + (threadIdx.x >> 6); r < (int)(blockIdx.y + 1) * each && first + r < rows; r += 4) {
        const float *part = a.partial + (long long)w.slot * kNext + r * (DP + 2);
        float top = -__builtin_inff(), total = 0.0f;
        for (int i = lane; i < w.pieces; i += 64) top = fmaxf(top, part[(long long)i * kNext]);
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
        const float zero = top == -__builtin_inff() ? 0.0f : top;
        f32x4 y = {0.f, 0.f, 0.f, 0.f};
        for (int from = 0; from < w.pieces; from += 64) {
            const int count = min(64, w.pieces - from);
            float share = 0.0f;
            if (lane < count) {
                const float *p = part + (long long)(from + lane) * kNext;
                share = __builtin_amdgcn_exp2f(p[0] - zero);
                total += p[1] * share;
            }
            for (int i = 0; i < count; i += kGroups) {
                const int piece = min(i + group, count - 1);
                const float by = __shfl(share, i + group, 64);
                const float2 *p = (const float2 *)(part + (long long)(from + piece) * kNext + 2 + d);
                const float2 low = p[0], high = p[1];
                if (i + group < count) y += (f32x4){low.x * by, low.y * by, high.x * by, high.y * by};
            }
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
#pragma unroll
        for (int off = DP / 4; off < 64; off <<= 1)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] += __shfl_xor(y[e], off, 64);
        if (group != 0) continue;
        const int row = first + r;
        const long long at = (long long)(v.start + row / a.group) * a.out_token + (long long)(w.head * a.group + row % a.group) * a.out_head;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < a.shape.head_dim) store_result<true>(a, at + d + e, total == 0.0f ? 0.0f : y[e] / total);
    }
}

template <int DP>
void launch_many(const AttendArgs &a, unsigned rows_of_tiles, bool may_cut, hipStream_t stream) {
    const dim3 grid(rows_of_tiles + (may_cut ? (unsigned)a.slots : 0u));
    hipLaunchKernelGGL(attend_many_kernel<DP>, grid, dim3(256), 0, stream, a);
    if (!may_cut) return;
    unsigned parts = 32;                // a workgroup per four queries, or fewer where there are rows of tiles enough
    while (parts > 4 && rows_of_tiles * parts > 2048) parts /= 2;
    hipLaunchKernelGGL(attend_join_many_kernel<DP>, dim3(rows_of_tiles, parts), dim3(256), 0, stream, a);
}

}  // namespace

int attend_many_slots(int dim) { return compute_units() * (dim == 256 ? 1 : 2); }

void launch_attend_many(AttendArgs a, unsigned rows_of_tiles, bool may_cut, hipStream_t stream) {
    a.least = may_cut ? kManyLeast : 1 << 28;
    const int dim = attend_dim(a.shape.head_dim);
    (dim == 64 ? launch_many<64> : dim == 128 ? launch_many<128> : launch_many<256>)(a, rows_of_tiles, may_cut, stream);
}

}  // namespace qt
