// Attention over a 4-bit cache for sequences of many queries: prompts, or many heads that share one of the cache (qt_attend.h).
//
// A workgroup takes 128 queries (of all heads that share a head of the cache), thirty-two for each of its four waves, and goes through the
// tokens they see in tiles of 64.  Scores as in the kernel for few queries, but by v_mfma_scale_f32_32x32x64: the codes of the keys are
// multiplied as they are with the queries' three 6-bit pieces, and scaled afterwards.  The weights' products are bound by the vector
// unit rather than by matrix instructions when weights are split, so here the values are expanded, once for all 128 queries: a thread turns 16
// bytes of codes into 32 fp16 numbers times their scale (two roundings of 2^-12, against 2^-9 of the result's type) in LDS, and weights
// are rounded to fp16 (2^-12).  fp16 has no range to spare: weights are 2^11 times what they are, and scales relative to a power of two that
// follows the largest scale of the tiles so far, so that a value loses bits only 2^25 below the largest.
#include "qt_attend.h"

namespace qt {
namespace {

constexpr int kManyTile = 64;
constexpr int kManyShift = 6;
constexpr int kManyLeast = 8;           // tiles of a piece, at least
constexpr float kWeightBits = 11.0f;    // weights are kept times 2^11 ...
constexpr float kSlack = 4.0f;          // ... and the running maximum may lag behind by 4: below 2^15 in fp16

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

// Of the tokens 8 (i / 4) + i % 4 of a lane (i < 16; bit i), those up to x.
__device__ __forceinline__ uint32_t tokens_up_to(int x) {
    const int bits = 4 * (x >> 3) + min(x & 7, 3) + 1;
    return x < 0 ? 0u : x >= 27 ? 0xffffu : (1u << (bits & 31)) - 1u;
}

// Sixteen scores times what the lanes of the lane's row of sixteen hold, one each.
template <bool ADD>
__device__ __forceinline__ f32x16 times_row(const f32x16 &x, float by, const f32x16 &to) {
    f32x16 y;
#define QT_EACH(i) y[i] = ADD ? __builtin_fmaf(x[i], of_row<i>(by), to[i]) : x[i] * of_row<i>(by);
    QT_EACH(0) QT_EACH(1) QT_EACH(2) QT_EACH(3) QT_EACH(4) QT_EACH(5) QT_EACH(6) QT_EACH(7)
    QT_EACH(8) QT_EACH(9) QT_EACH(10) QT_EACH(11) QT_EACH(12) QT_EACH(13) QT_EACH(14) QT_EACH(15)
#undef QT_EACH
    return y;
}
__device__ __forceinline__ uint32_t rows_not_finite(float by) {
    uint32_t y = 0;
#define QT_EACH(i) y |= (uint32_t)((__float_as_uint(of_row<i>(by)) & 0x7f800000u) == 0x7f800000u) << i;
    QT_EACH(0) QT_EACH(1) QT_EACH(2) QT_EACH(3) QT_EACH(4) QT_EACH(5) QT_EACH(6) QT_EACH(7)
    QT_EACH(8) QT_EACH(9) QT_EACH(10) QT_EACH(11) QT_EACH(12) QT_EACH(13) QT_EACH(14) QT_EACH(15)
#undef QT_EACH
    return y;
}

// Bytes of row `row` of expanded values in LDS are moved by this (exclusive or), so that the eight rows of 64 bytes that a transposed
// read takes lie in different banks two by two.
template <int DP>
__device__ __forceinline__ int value_swap(int row) { return (DP == 64 ? (row >> 1) & 1 : row & 3) << 6; }

template <int DP, int UNITS>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void attend_many_kernel(const AttendArgs a) {
    constexpr int kPieces = 3, kSteps = DP / 64, kDTiles = DP / 32, kChunks = DP / 32;
    constexpr int kKeyBytes = kManyTile * DP / 2, kRowBytes = DP / 2, kValueRow = DP * 2;
    constexpr int kEach = kManyTile * kChunks > 256 ? kManyTile * kChunks / 256 : 1;        // 16-byte chunks of a tile's codes per thread
    __shared__ __attribute__((aligned(16))) uint8_t s_keys[2][kKeyBytes];
    __shared__ __attribute__((aligned(16))) uint8_t s_values[2][kManyTile * kValueRow];

    AttendWork w;
    if (!find_work<kRowsOfMany, kManyShift, true>(a, blockIdx.x, w)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, column = lane & 31, half = lane >> 5;
    SequenceView v = view_sequence<kManyShift>(a, w.b);
    const int all_rows = v.count * a.group;
    const int first_row = first_row_of<kRowsOfMany>(all_rows, w.row_tile);
    const int my_row = min(first_row + 32 * wave + column, all_rows - 1);
    const bool mine = first_row + 32 * wave + column < all_rows;
    const int my_token = v.start + my_row / a.group, my_head = w.head * a.group + my_row % a.group;
    const int position = v.first_position + my_row / a.group;
    const int behind = a.window && position >= 0 ? position - a.window : -0x7fffffff;
    // positions of this wave's queries and of all of the workgroup's
    const int lowest = v.first_position + min(first_row + 32 * wave, all_rows - 1) / a.group;
    const int highest = first_row + 32 * wave < all_rows ? v.first_position + min(first_row + 32 * wave + 31, all_rows - 1) / a.group : -1;
    {
        const int last = v.first_position + min(first_row + kRowsOfMany - 1, all_rows - 1) / a.group;
        v.end = max(0, min(v.end, last + 1));
        view_tokens<kManyShift>(a, v, v.first_position + first_row / a.group, v.end);
    }
    const int per_piece = (v.tiles + w.pieces - 1) / w.pieces;
    const int tile_from = min(w.piece * per_piece, v.tiles), tile_to = min(tile_from + per_piece, v.tiles);

    const int *table = a.at.table + (long long)w.b * a.at.table_stride;
    const int page_mask = (1 << a.shape.page_shift) - 1, chunks = a.shape.row_bytes >> 4;
    auto tile_at = [&](int k) { return (k < v.sink_tiles ? k : v.first_tile + k - v.sink_tiles) * kManyTile; };

    // what this thread stages of a tile: chunk id % kChunks of token id / kChunks
    const int own_token = 8 * ((lane & 15) >> 2) + 4 * half + (lane & 3);       // ... and whose scales its row of lanes needs: this + 32 i
    i32x4 key_chunk[kEach], value_chunk[kEach];
    float chunk_scale[kEach], key_scale[UNITS][2], value_scale[UNITS][2];
    unsigned long long valid[2];
    int page[kEach + 2];
    auto load_pages = [&](int k) {
        const int base = tile_at(k);
#pragma unroll
        for (int i = 0; i < kEach + 2; ++i) {
            const int token = base + (i < kEach ? (threadIdx.x + 256 * i) / kChunks % kManyTile : own_token + 32 * (i - kEach));
            page[i] = table[min(token, v.end - 1) >> a.shape.page_shift];
        }
    };
    auto load_tile = [&](int k) {
        const int base = tile_at(k);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int id = threadIdx.x + 256 * i, inside = id / kChunks % kManyTile, token = base + inside;
            const bool there = (unsigned)page[i] < (unsigned)a.shape.pages && token < v.end;
            const long long line = ((long long)(there ? page[i] : 0) * a.shape.kv_heads + w.head) << a.shape.page_shift;
            const int chunk = min(id % kChunks, chunks - 1), in_page = token & page_mask;
            const long long at = (line + in_page) * a.shape.row_bytes + 16 * chunk;
            key_chunk[i] = *(const i32x4 *)(a.codes[0] + at);
            value_chunk[i] = *(const i32x4 *)(a.codes[1] + at);
            const int segment = min((32 * chunk) >> a.shape.segment_shift, a.shape.segments - 1);
            chunk_scale[i] = a.scales[1][line * a.shape.segments + ((long long)segment << a.shape.page_shift) + in_page];
            if (!there) page[i] = -1;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int token = base + own_token + 32 * i;
            const bool there = (unsigned)page[kEach + i] < (unsigned)a.shape.pages && token < v.end;
            valid[i] = __ballot(there);
            const long long line = ((long long)(there ? page[kEach + i] : 0) * a.shape.kv_heads + w.head) << a.shape.page_shift;
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                const int segment = min((u * 64) >> a.shape.segment_shift, a.shape.segments - 1);
                const long long at = line * a.shape.segments + ((long long)segment << a.shape.page_shift) + (token & page_mask);
                key_scale[u][i] = a.scales[0][at];
                value_scale[u][i] = a.scales[1][at];
            }
        }
    };

    u32x6 query[kSteps][kPieces];
    int query_scale[kSteps][kPieces];
    f32x16 result[kDTiles];
#pragma unroll
    for (int d = 0; d < kDTiles; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) result[d][i] = 0.0f;
    float best = -__builtin_inff(), sum = 0.0f, poison[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) poison[u] = 0.0f;
    int exponent = 1;                       // of the largest scale of a value so far: values are kept times 2^(138 - exponent)

    // scales of the tile that is worked on; writes of the next tile's codes
    float by_key[UNITS][2], by_value[UNITS][2];
    unsigned long long here[2];
    bool odd = false;                       // a scale of its values is not finite
    auto stage = [&](int buffer) {
        uint32_t top = 0;
        bool bad = false;
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bool there = (valid[i] >> lane) & 1;
                by_key[u][i] = there ? key_scale[u][i] * a.factor : 0.0f;
                by_value[u][i] = there ? value_scale[u][i] : 0.0f;
                const uint32_t bits = __float_as_uint(by_value[u][i]) & 0x7fffffffu;
                bad |= bits >= 0x7f800000u;
                if (bits < 0x7f800000u) top = max(top, bits);
            }
        here[0] = valid[0], here[1] = valid[1];
        odd = __ballot(bad) != 0;
        top = group_max_u32<64>(top);
        const int larger = max(exponent, (int)(top >> 23));
        if (larger != exponent) {
            const float fade = __builtin_amdgcn_ldexpf(1.0f, exponent - larger);
#pragma unroll
            for (int d = 0; d < kDTiles; ++d) result[d] *= fade;
            exponent = larger;
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int id = threadIdx.x + 256 * i, row = id / kChunks, chunk = id % kChunks;
            if (kManyTile * kChunks < 256 && row >= kManyTile) break;
            *(i32x4 *)(s_keys[buffer] + row * kRowBytes + 16 * (chunk ^ swap_of<DP>(row))) = key_chunk[i];
            const float scale = page[i] < 0 || (__float_as_uint(chunk_scale[i]) & 0x7fffffffu) >= 0x7f800000u ? 0.0f : chunk_scale[i];
            const _Float16 scaled = (_Float16)__builtin_amdgcn_ldexpf(scale, 138 - exponent);
            const f16x2 by = {scaled, scaled};
            uint8_t *to = s_values[buffer] + row * kValueRow + ((64 * chunk) ^ value_swap<DP>(row));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t word = (uint32_t)value_chunk[i][e];
                const f16x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, 1.0f, 0) * by, x1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, 1.0f, 1) * by,
                            x2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, 1.0f, 2) * by, x3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, 1.0f, 3) * by;
                *(f16x8 *)(to + 16 * e) = (f16x8){x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
            }
        }
    };

    if (tile_from < tile_to) {
        uint4 raw[kSteps][4];
        load_pages(tile_from);
#pragma unroll
        for (int h = 0; h < kSteps; ++h) load_query<true>(a, my_token * a.q_token + my_head * a.q_head, 64 * h + 32 * half, mine, raw[h]);
        load_tile(tile_from);
#pragma unroll
        for (int h = 0; h < kSteps; ++h) {
            f32x16 even, odd_places;
            unpack_query<true>(raw[h], even, odd_places);
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) top = max(top, max(__float_as_uint(even[i]) & 0x7fffffffu, __float_as_uint(odd_places[i]) & 0x7fffffffu));
            split_fp6<kPieces>(even, odd_places, top, query[h], query_scale[h]);
        }
        stage(0);
        load_pages(min(tile_from + 1, tile_to - 1));
        __syncthreads();
    }
    for (int k = tile_from; k < tile_to; ++k) {
        const int base = tile_at(k), buffer = (k - tile_from) & 1;
        const bool more = k + 1 < tile_to;
        if (more) load_tile(k + 1);
        // (a wave whose queries see nothing of the tile only stages the next one)
        if (base <= highest && (!a.window || base + kManyTile - 1 > lowest - a.window || base < a.sinks)) {
            f32x16 score[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                f32x16 c;
#pragma unroll
                for (int h = 0; h < kSteps; ++h) {
                    const int row = 32 * t + column;
                    const i32x4 keys = *(const i32x4 *)(s_keys[buffer] + row * kRowBytes + 16 * ((2 * h + half) ^ swap_of<DP>(row)));
#pragma unroll
                    for (int i = kPieces - 1; i >= 0; --i) {
                        const f32x16 none = {};
                        c = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(as_operand(keys), as_operand(query[h][i]),
                                                                            i == kPieces - 1 && (h == 0 || UNITS > 1) ? none : c, kFp4, kFp6, 0, kOne, 0,
                                                                            query_scale[h][i]);
                    }
                    if constexpr (UNITS > 1) score[t] = h == 0 ? times_row<false>(c, by_key[h][t], c) : times_row<true>(c, by_key[h][t], score[t]);
                }
                if constexpr (UNITS == 1) score[t] = times_row<false>(c, by_key[0][t], c);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) asm volatile("" : "+v"(score[t]));      // (here, in one block with what they are made of)
            __builtin_amdgcn_sched_barrier(0);
            const bool whole = !(~here[0] | ~here[1]);
            const bool full = base + kManyTile - 1 <= lowest && (!a.window || highest - base < a.window || base + kManyTile <= a.sinks) && whole;
            uint32_t see = 0xffffffffu;
            if (!full) {
                const int x = position - base - 4 * half;
                see = tokens_up_to(x) | (tokens_up_to(x - 32) << 16);
                if (a.window) {
                    const int y = behind - base - 4 * half, z = a.sinks - 1 - base - 4 * half;
                    see &= ~(tokens_up_to(y) | (tokens_up_to(y - 32) << 16)) | (tokens_up_to(z) | (tokens_up_to(z - 32) << 16));
                }
                if (!whole) see &= ((uint32_t)(here[0] >> (32 * half)) & 0xffffu) | ((uint32_t)(here[1] >> (32 * half)) << 16);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) score[t][i] = see & (1u << (16 * t + i)) ? score[t][i] : -__builtin_inff();
            }
            if (__builtin_expect(odd, 0)) {
#pragma unroll
                for (int u = 0; u < UNITS; ++u)
                    if (see & (rows_not_finite(by_value[u][0]) | (rows_not_finite(by_value[u][1]) << 16))) poison[u] = __builtin_nanf("");
            }
            float top = -__builtin_inff();
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, score[t][i]);
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            if (__ballot(top > best + kSlack)) {
                // (-inf + 4 is -inf: the first token that is seen sets the maximum)
                const float next = fmaxf(best, top);
                const float fade = next == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(best - next);
                sum *= fade;
#pragma unroll
                for (int d = 0; d < kDTiles; ++d) result[d] *= fade;
                best = next;
            }
            const float zero = best == -__builtin_inff() ? 0.0f : best - kWeightBits;
            f16x8 weight[4];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const float p = __builtin_amdgcn_exp2f(score[t][i] - zero), q = __builtin_amdgcn_exp2f(score[t][i + 1] - zero);
                    const f16x2 both = __builtin_convertvector((cache_f32x2){p, q}, f16x2), ones = {(_Float16)1.0f, (_Float16)1.0f};
                    sum = __builtin_amdgcn_fdot2(both, ones, sum, false);       // of the weights as they are multiplied, in fp32
                    weight[2 * t + (i >> 3)][i & 7] = both[0];
                    weight[2 * t + (i >> 3)][(i & 7) + 1] = both[1];
                }
#pragma unroll
            for (int d = 0; d < kDTiles; ++d)
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    f16x8 rows;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int token = 16 * n + 8 * e + 4 * half + ((lane & 15) >> 2), byte = 64 * d + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
                        const i16x4 part = __builtin_amdgcn_ds_read_tr16_b64_v4i16((QT_LDS i16x4 *)(s_values[buffer] + token * kValueRow + (byte ^ value_swap<DP>(token))));
                        const f16x4 four = __builtin_bit_cast(f16x4, part);
                        rows[4 * e] = four[0], rows[4 * e + 1] = four[1], rows[4 * e + 2] = four[2], rows[4 * e + 3] = four[3];
                    }
                    result[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(rows, weight[n], result[d], 0, 0, 0);
                }
        }
        if (more) {
            stage(buffer ^ 1);
            load_pages(min(k + 2, tile_to - 1));
        }
        __syncthreads();
    }
    sum += __shfl_xor(sum, 32, 64);
#pragma unroll
    for (int u = 0; u < UNITS; ++u) poison[u] += __shfl_xor(poison[u], 32, 64);
    if (!mine) return;
    // four consecutive elements of a result at a time
    const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
    float *part = a.partial + ((long long)(w.slot + w.piece) * kRowsOfMany + 32 * wave + column) * (DP + 2);
    const long long at = (long long)my_token * a.out_token + (long long)my_head * a.out_head;
    if (w.pieces > 1 && half == 0) part[0] = best, part[1] = sum;
#pragma unroll
    for (int d = 0; d < kDTiles; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int element = 32 * d + 2 * i + 4 * half;
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                y[e] = __builtin_amdgcn_ldexpf(w.pieces > 1 ? result[d][i + e] : result[d][i + e] * by, exponent - 138) + poison[UNITS == 1 ? 0 : d / 2];
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

template <int DP>
void launch_many(const AttendArgs &a, unsigned rows_of_tiles, bool may_cut, hipStream_t stream) {
    const dim3 grid(rows_of_tiles + (may_cut ? (unsigned)a.slots : 0u));
    if (DP == 64 || a.shape.segments == 1) hipLaunchKernelGGL((attend_many_kernel<DP, 1>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((attend_many_kernel<DP, DP / 64>), grid, dim3(256), 0, stream, a);
    if (may_cut)
        hipLaunchKernelGGL((attend_join_kernel<kRowsOfMany, kManyShift, DP, true>), dim3(rows_of_tiles, kRowsOfMany), dim3(256), 0, stream, a);
}

}  // namespace

int attend_many_slots(int dim) { return compute_units() * (dim == 256 ? 1 : 2); }

void launch_attend_many(AttendArgs a, unsigned rows_of_tiles, bool may_cut, hipStream_t stream) {
    a.least = may_cut ? kManyLeast : 1 << 28;
    const int dim = attend_dim(a.shape.head_dim);
    (dim == 64 ? launch_many<64> : dim == 128 ? launch_many<128> : launch_many<256>)(a, rows_of_tiles, may_cut, stream);
}

}  // namespace qt
