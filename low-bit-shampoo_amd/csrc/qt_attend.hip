// Attention over a cache held in 4 bits (layout: qt_cache.h): out_i = sum_j p_ij v_j, p_ij = softmax_j(scale q_i . k_j) over the
// tokens j that query i sees: j <= i and, with a window, i - j < window or j < sinks.
//
// The cache is never expanded: its 4-bit numbers are operands of the scaled matrix instructions as they lie in memory.  Queries and
// weights are split into pieces of 6 bits (qt_attend.h) and multiplied piece by piece; the fp32 scales of keys multiply scores, those of
// values the weights before they are split.
#include "qt_attend.h"

#include <type_traits>

namespace qt {
namespace {

constexpr int kTile = 128;              // tokens a wave takes at a time: one step of k of a matrix instruction with the weights
constexpr int kRows = 16;               // queries (of all heads that share a head of the cache) in a tile of rows
// Queries of a sequence that are still few: two rows of tiles.  (32 sequences of 4000 tokens and 4 heads of the cache, 32 / 64 / 96 queries
// each: 47 / 63 / 91 us here, 74 / 66 / 69 by the kernel for many.)
constexpr int kFewRows = 32;
// Pairs of a query and a token (of a head of the cache) up to which all of a call is taken to be few: 8 sequences of 2000 tokens, 4 heads and
// 32 queries each (2 * 10^6) 16 us, 22 with the kernel for many launched beside it; 1 of 16000 with 64 (4 * 10^6) 12 and 35; 32 of 500 with
// 256 (16 * 10^6) 39 and 26.
constexpr double kFewWork = 8388608.0;
constexpr int kLeastTiles = 4;          // tiles of a piece: one for each wave (4 sequences of 2500 tokens 13.2 us; in pieces of 8 15.8)
// A call whose sequences have no more tiles than that is not cut: three rounds of the waves take less time than two and a launch that joins
// pieces (32 sequences of 1500 tokens 14.7 us, 16.8 if they are cut; of 1700 17.9 and 16.7).
constexpr int kWholeTiles = 12;

// Of the tokens 16 t + i of a lane (t < 8, i < 4; bit 4 t + i), those up to x.
__device__ __forceinline__ uint32_t tokens_up_to(int x) {
    const int bits = 4 * (x >> 4) + min(x & 15, 3) + 1;
    return x < 0 ? 0u : x >= 115 ? 0xffffffffu : (1u << (bits & 31)) - 1u;
}

// x times what lanes 4 t ... 4 t + 3 of the lane's row of sixteen hold.
__device__ __forceinline__ f32x4 times_row(f32x4 x, float by, int t) {
    switch (t) {
    case 0: return (f32x4){x[0] * of_row<0>(by), x[1] * of_row<1>(by), x[2] * of_row<2>(by), x[3] * of_row<3>(by)};
    case 1: return (f32x4){x[0] * of_row<4>(by), x[1] * of_row<5>(by), x[2] * of_row<6>(by), x[3] * of_row<7>(by)};
    case 2: return (f32x4){x[0] * of_row<8>(by), x[1] * of_row<9>(by), x[2] * of_row<10>(by), x[3] * of_row<11>(by)};
    default: return (f32x4){x[0] * of_row<12>(by), x[1] * of_row<13>(by), x[2] * of_row<14>(by), x[3] * of_row<15>(by)};
    }
}

constexpr int kWaitLds = 0xc07f;        // s_waitcnt lgkmcnt(0), nothing else

constexpr int few_waves(int dim, int units, bool bf16) { return dim == 256 || (units > 1 && !bf16) ? 1 : 2; }

// Zeros for rows of the call that are of no sequence (a step captured with room for more tokens than there are), from the `nth` of them on every `each`th.
template <bool BF16>
__device__ __forceinline__ void clear_rows_of_none(const AttendArgs &a, int nth, int each) {
    int end = 0;                            // of the last sequence whose rows are all there
    for (int b = threadIdx.x & 63; b < a.at.batch; b += 64) {
        const int from = a.at.starts[b], to = a.at.starts[b + 1];
        if (from >= 0 && from <= to && to <= a.at.tokens) end = max(end, to);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) end = max(end, __shfl_xor(end, off, 64));
    for (int row = end + nth; row < a.at.tokens; row += each)
        for (int e = threadIdx.x; e < a.group * a.shape.kv_heads * a.shape.head_dim; e += 256)
            store_result<BF16>(a, row * a.out_token + e / a.shape.head_dim * a.out_head + e % a.shape.head_dim, 0.0f);
}

// Few queries per sequence: generation.  A workgroup takes one piece of a row of tiles, its four waves every fourth tile of it.
//
// Scores are computed transposed, K Q^T by v_mfma_scale_f32_16x16x128: a lane holds those of query lane % 16 and the tokens 16 t + 4 (lane
// / 16) + i (t < 8, i < 4) -- 32 of the 128 tokens of a tile, which is just what it has to hold of the weights for O^T = V^T P^T, so weights
// never leave their lane.  Keys go from memory straight to registers (16 lanes' rows of 64 bytes side by side); values pass through an area
// of LDS that belongs to the wave, to be read transposed (ds_read_b64_tr_b4: sixteen tokens of one element a lane) in the order of
// tokens that the weights have.
//
// The running maximum and sum of the softmax are kept per wave and joined at the end, so the cache is read once.  Bound by memory where
// sequences are long (2 of up to 131072 tokens, 8 heads of 128 in one segment, 8 queries each: 52.6 us, 4.85 TB/s with the join), otherwise
// by latency: about 5 us of finding work and asking for the first tile, 2.5 to 3.6 us a tile, and 5 us of a second launch where pieces are
// joined (32 sequences of up to 8000 tokens, 4 queries per head, segments of 64: 44 us, 3.4 TB/s).  By its counters such a tile is some 970 vector
// instructions, 3900 cycles of the vector unit (the split of the weights, conversions of 32 numbers that take 73 cycles each, is 730 of
// them), beside 1170 of the matrix pipe, which takes sixteen queries where four are; waves wait for a third of their time.  Splitting by value scale, not expanding the values, keeps the products exact in
// the cache's numbers; four waves to a piece share nothing but the join, so no barrier stands in the loop.  DP: head_dim
// rounded up to 64, 128 or 256; UNITS: 1, or DP / 64 where a vector has several scales (each 64 elements then have scores and weights of
// their own).
template <int DP, int UNITS, bool BF16>
__global__ __launch_bounds__(256, few_waves(DP, UNITS, BF16)) void attend_few_kernel(const AttendArgs a) {
    constexpr int kPieces = BF16 ? 3 : 5, kQueryPieces = 5;         // of weights, and of queries (of bf16 queries the last two only where they matter)
    // One or two rows of tiles read a long sequence: past the L2 (two of 131072 tokens 58.8 -> 52.9 us).  More of them come in calls that are little work,
    // which read it again and take the same time either way (2048 tokens by 4096 queries, one head of 128: 28.7 us).  Queries in 32 bits come in any
    // number and read it again for every sixteen (4 x 2048 of them 1669 us, 1719 past the L2).
    constexpr bool kOnce = BF16;
    constexpr int kHalves = DP == 256 ? 2 : 1;              // 16-byte chunks of a row that a lane holds
    constexpr int kLoads = DP == 64 ? 4 : 8;                // loads of sixteen tokens by all lanes (thirty-two for rows of 32 bytes)
    constexpr int kRowBytes = DP / 2;                       // of a token's values in LDS; the 16-byte chunks of a row stand in an order of
                                                            // its own (swap), so that transposed reads fall on all banks
    constexpr int kValueLoads = kTile * kRowBytes / 1024;
    constexpr int kDTiles = DP / 16;
    constexpr int kArea = kTile * kRowBytes > kRows * (DP + 4) * 4 ? kTile * kRowBytes : kRows * (DP + 4) * 4;      // a wave's results take the place of its values
    __shared__ __attribute__((aligned(16))) uint8_t s_area[4][kArea];
    __shared__ float s_best[4][kRows], s_sum[4][kRows];

    AttendWork w;
    SequenceView v;
    if (!find_work<kRows, 7, true>(a, blockIdx.x, w, v)) {
        if (a.at.starts && w.pieces == 0) clear_rows_of_none<BF16>(a, w.piece, (int)gridDim.x - ((int)blockIdx.x - w.piece));
        return;
    }
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, column = lane & 15, g = lane >> 4;
    const int rows = min(kRows, v.count * a.group - w.row_tile * kRows);
    const int first_row = first_row_of<kRows>(0, w.row_tile);
    uint8_t *s_values = s_area[wave];

    // the query of this lane's column
    const int my_row = first_row + min(column, rows - 1);
    const int my_token = v.start + my_row / a.group, my_head = w.head * a.group + my_row % a.group;
    const int position = v.first_position + my_row / a.group;
    const int behind = a.window ? max(max(position, 0) - a.window, -1) : -1;         // last token behind the window
    const int lowest = v.first_position + first_row / a.group, highest = v.first_position + (first_row + rows - 1) / a.group;

    const int tile_from = min(w.piece * w.per_piece, v.tiles), tile_to = min(tile_from + w.per_piece, v.tiles);
    const int *table = a.at.table + (long long)w.b * a.at.table_stride;
    const int page_mask = (1 << a.shape.page_shift) - 1, chunks = a.shape.row_bytes >> 4;

    auto tile_at = [&](int k) { return (k < v.sink_tiles ? k : v.first_tile + k - v.sink_tiles) * kTile; };
    // The token whose page and scales this lane looks up, and 64 further on: those that its row of 16 lanes has scores of, one each, so that
    // they reach the others of the row as operands of its multiplications (row_newbcast)
    const int own_token = 16 * (column >> 2) + 4 * g + (column & 3);
    auto load_pages = [&](int k, int *page) {
        const int base = tile_at(k) + own_token;
#pragma unroll
        for (int i = 0; i < 2; ++i) page[i] = table[min(base + 64 * i, v.end - 1) >> a.shape.page_shift];
    };
    i32x4 keys[kHalves][kLoads];
    uint32_t inside[kHalves];           // this lane's 16 bytes among sixteen rows; behind the end of a row the last chunk again (queries are
                                        // zero there, and results are not stored)
#pragma unroll
    for (int h = 0; h < kHalves; ++h) inside[h] = column * a.shape.row_bytes + 16 * min(DP == 64 ? g & 1 : g + 4 * h, chunks - 1);
    float key_scale[UNITS][2], value_scale[UNITS][2];
    unsigned long long valid[2];
    uint32_t value_inside[DP == 256 ? 2 : 1];       // what the same lane loads of the values: chunk (lane's place) ^ swap of its row
#pragma unroll
    for (int i = 0; i < (DP == 256 ? 2 : 1); ++i) {
        constexpr int kChunks = DP / 32;
        const int row = DP == 64 ? (lane >> 1) & 15 : DP == 128 ? lane >> 2 : 8 * i + (lane >> 3);
        value_inside[i] = row * a.shape.row_bytes + 16 * min((lane & (kChunks - 1)) ^ swap_of<DP>(row), chunks - 1);
    }
    // sixteen tokens from 16 t of a tile on: where their rows begin
    auto line_of = [&](const int *safe, int base, int t) {
        const int p = __builtin_amdgcn_readlane(safe[t >> 2], 4 * (t & 3));
        return ((((long long)p * a.shape.kv_heads + w.head) << a.shape.page_shift) + ((base + 16 * t) & page_mask)) * a.shape.row_bytes;
    };
    int safe[2];
    auto load_tile = [&](int k, const int *page) {
        const int base = tile_at(k);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bool there = (unsigned)page[i] < (unsigned)a.shape.pages && base + 64 * i + own_token < v.end;
            safe[i] = there ? page[i] : 0;
            valid[i] = __ballot(there);
            const long long line = ((long long)safe[i] * a.shape.kv_heads + w.head) << a.shape.page_shift;
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                const int segment = min((u * 64) >> a.shape.segment_shift, a.shape.segments - 1);
                const long long at = line * a.shape.segments + ((long long)segment << a.shape.page_shift) + ((base + 64 * i + own_token) & page_mask);
                key_scale[u][i] = a.scales[0][at];
                value_scale[u][i] = a.scales[1][at];
            }
        }
        // (one base per sixteen tokens in scalar registers, the lane's place among them in one vector register for all loads)
#pragma unroll
        for (int t = 0; t < kLoads; ++t) {
            const long long at = DP == 64 ? (lane < 32 ? line_of(safe, base, 2 * t) : line_of(safe, base, 2 * t + 1)) : line_of(safe, base, t);
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                const i32x4 *from = (const i32x4 *)(a.codes[0] + at + inside[h]);
                keys[h][t] = kOnce ? __builtin_nontemporal_load(from) : *from;
            }
        }
    };
    // values of a tile whose pages `safe` has, from memory to LDS: lane i of a load fills bytes 16 i of a kilobyte
    auto load_values = [&](int k, const int *safe) {
        const int base = tile_at(k);
#pragma unroll
        for (int t = 0; t < kValueLoads; ++t) {
            const uint8_t *from;
            if (DP == 64) from = a.codes[1] + (lane < 32 ? line_of(safe, base, 2 * t) : line_of(safe, base, 2 * t + 1)) + value_inside[0];
            else if (DP == 128) from = a.codes[1] + line_of(safe, base, t) + value_inside[0];
            else from = a.codes[1] + line_of(safe, base, t >> 1) + value_inside[t & 1];
            __builtin_amdgcn_global_load_lds((const QT_GLOBAL void *)from, (QT_LDS void *)(s_values + 1024 * t), 16, 0, kOnce ? 2 : 0);
        }
    };

    f32x4 result[kDTiles];
#pragma unroll
    for (int d = 0; d < kDTiles; ++d) result[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float best = -__builtin_inff(), sum = 0.0f;
    u32x6 query[kHalves][kQueryPieces];
    int query_scale[kHalves][kQueryPieces];
    float matters = 0.0f;               // scale of a key (times that of the scores) above which what kPieces pieces leave of the queries matters
    int page[2];
    // one tile; `more`: the wave has another one, which is asked for on the way (without a branch: waits count loads)
    auto step = [&](int k, auto more) {
        const int base = tile_at(k);
        const unsigned long long here[2] = {valid[0], valid[1]};
        // (a scale that is not finite makes every score NaN: the sums are zero only to 2^-127 of another token's where a load holds two)
        // what no page holds has scale 0; a weight of zero times a scale that is not finite is not zero: only then such weights are looked for
        float by_key[UNITS][2], by_value[UNITS][2], odd_scale = 0.0f;
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bool there = (here[i] >> lane) & 1;
                by_key[u][i] = there ? __builtin_fmaf(key_scale[u][i], 0.0f, key_scale[u][i] * a.factor) : 0.0f;
                by_value[u][i] = there ? value_scale[u][i] : 0.0f;
                odd_scale += 0.0f * by_value[u][i];
            }
        const bool odd = __ballot(odd_scale != 0.0f) != 0;
        bool rest = false;
        if constexpr (kQueryPieces > kPieces) {
#pragma unroll
            for (int u = 0; u < UNITS; ++u) rest |= fmaxf(fabsf(by_key[u][0]), fabsf(by_key[u][1])) > matters;
            rest = __ballot(rest) != 0;
        }

        // scores
        f32x4 score[8];
        // (pieces from `to` - 1 down to `from`)
        auto products = [&](int t, int from, int to) __attribute__((always_inline)) {
            f32x4 all;
            if constexpr (UNITS == 1) {
                f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < kHalves; ++h)
#pragma unroll
                    for (int i = to - 1; i >= from; --i) {
                        // (rows of 32 bytes: a load holds two times sixteen tokens, of which the scale of 2^-127 takes one away)
                        const int by = DP == 64 ? ((lane >> 5) == (t & 1) ? query_scale[h][i] : 0) : query_scale[h][i];
                        c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(as_operand(keys[h][DP == 64 ? t >> 1 : t]), as_operand(query[h][i]), c, kFp4, kFp6,
                                                                             0, kOne, 0, by);
                    }
                all = times_row(c, by_key[0][t >> 2], t & 3);
            } else {
#pragma unroll
                for (int u = 0; u < UNITS; ++u) {
                    f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = to - 1; i >= from; --i) {
                        const int by = (lane >> 5) == (u & 1) ? query_scale[u >> 1][i] : 0;
                        c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(as_operand(keys[u >> 1][t]), as_operand(query[u >> 1][i]), c, kFp4, kFp6, 0, kOne,
                                                                             0, by);
                    }
                    c = times_row(c, by_key[u][t >> 2], t & 3);
                    all = u == 0 ? c : all + c;
                }
            }
            return all;
        };
#pragma unroll
        for (int t = 0; t < 8; ++t) score[t] = products(t, 0, kPieces);
        if constexpr (kQueryPieces > kPieces) {
            if (rest) {
#pragma unroll
                for (int t = 0; t < 8; ++t) score[t] += products(t, kPieces, kQueryPieces);
            }
        }
#pragma unroll
        for (int t = 0; t < 8; ++t) asm volatile("" : "+v"(score[t]));      // (done here: the keys' registers are free)
        __builtin_amdgcn_sched_barrier(0);

        // which of the lane's tokens its query sees: bit 4 t + i of `see` (tokens past the end are past every position)
        const bool whole = !(~here[0] | ~here[1]);
        const bool full = base + kTile - 1 <= lowest && (!a.window || highest - base < a.window || base + kTile <= a.sinks) && whole;
        uint32_t see = 0xffffffffu;
        if (!full) {
            see = tokens_up_to(position - base - 4 * g);
            if (a.window) see &= ~tokens_up_to(behind - base - 4 * g) | tokens_up_to(a.sinks - 1 - base - 4 * g);
            if (!whole) {
                see &= ((uint32_t)(here[0] >> (16 * g)) & 0xffffu) | ((uint32_t)(here[1] >> (16 * g)) << 16);
            }
#pragma unroll
            for (int t = 0; t < 8; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) score[t][i] = see & (1u << (4 * t + i)) ? score[t][i] : -__builtin_inff();
        }
        float top = best;
#pragma unroll
        for (int t = 0; t < 8; ++t) top = fmaxf(fmaxf(fmaxf(top, score[t][0]), fmaxf(score[t][1], score[t][2])), score[t][3]);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float zero = top == -__builtin_inff() ? 0.0f : top;
        if (__ballot(top != best)) {
            const float fade = __builtin_amdgcn_exp2f(best - zero);
            sum *= fade;
#pragma unroll
            for (int d = 0; d < kDTiles; ++d) result[d] *= fade;
            best = top;
        }
        f32x4 weight[8];
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                weight[t][i] = __builtin_amdgcn_exp2f(score[t][i] - zero);
                sum += weight[t][i];
            }

        __builtin_amdgcn_sched_barrier(0);
        // their values: weights times scales in pieces, element by element of the values' rows
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            f32x16 early, late;
            uint32_t most = 0;
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const f32x4 scaled = times_row(weight[t], by_value[u][t >> 2], t & 3);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = scaled[i];
                    most = max(most, __float_as_uint(x));
                    if (t < 4) early[4 * t + i] = x;
                    else late[4 * (t - 4) + i] = x;
                }
                if (t == 3) __builtin_amdgcn_sched_barrier(0);
            }
            if (__builtin_expect(odd, 0)) {
                most = 0;
#pragma unroll
                for (int n = 0; n < 16; ++n) {
                    early[n] = see & (1u << n) ? early[n] : 0.0f;
                    late[n] = see & (1u << (16 + n)) ? late[n] : 0.0f;
                    most = max(most, max(__float_as_uint(early[n]), __float_as_uint(late[n])));
                }
            }
            u32x6 piece[kPieces];
            int by[kPieces];
            split_fp6<kPieces>(early, late, most, piece, by);
            __builtin_amdgcn_sched_barrier(0);
            constexpr int kMine = kDTiles / UNITS;
            i32x4 rows_of_v[kMine];
#pragma unroll
            for (int d = 0; d < kMine; ++d)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    // position 16 h + j of the weights is register (16 h + j) / 2 of the first or (odd) the second sixteen
                    const int dt = u * kMine + d, n = 8 * h + (column >> 1), token = 16 * (n >> 2) + 4 * g + (n & 3) + 64 * (column & 1);
                    const i32x2 part = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
                        (QT_LDS i32x2 *)(s_values + token * kRowBytes + 16 * ((dt >> 1) ^ swap_of<DP>(token)) + 8 * (dt & 1)));
                    rows_of_v[d][2 * h] = part[0], rows_of_v[d][2 * h + 1] = part[1];
                }
            if constexpr (decltype(more)::value) {
                if (u == UNITS - 1) {
                    // the next tile, as soon as nothing of this one is read any more: keys into registers that were free while the
                    // weights were split, values to LDS, where the reads above have to be through
                    __builtin_amdgcn_sched_barrier(0);
                    __builtin_amdgcn_s_waitcnt(kWaitLds);
                    wave_lds_sync();
                    load_tile(k + 4, page);
                    load_values(k + 4, safe);
                    load_pages(min(k + 8, tile_to - 1), page);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
#pragma unroll
            for (int i = kPieces - 1; i >= 0; --i)
#pragma unroll
                for (int d = 0; d < kMine; ++d)
                    result[u * kMine + d] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(as_operand(rows_of_v[d]), as_operand(piece[i]), result[u * kMine + d],
                                                                                             kFp4, kFp6, 0, kOne, 0, by[i]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // pages, queries and the first tile are asked for before any of them is waited for
    int k = tile_from + wave;
    uint4 raw[kHalves][BF16 ? 4 : 8];
    if (k < tile_to) load_pages(k, page);
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
        load_query<BF16>(a, my_token * a.q_token + my_head * a.q_head, 32 * (DP == 64 ? g & 1 : g + 4 * h), column < rows, raw[h]);
    if (k < tile_to) {
        load_tile(k, page);
        load_values(k, safe);
        load_pages(min(k + 4, tile_to - 1), page);
        uint32_t largest = 0;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            f32x16 even, odd;
            unpack_query<BF16>(raw[h], even, odd);
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) top = max(top, max(__float_as_uint(even[i]) & 0x7fffffffu, __float_as_uint(odd[i]) & 0x7fffffffu));
            split_fp6<kQueryPieces>(even, odd, top, query[h], query_scale[h]);
            largest = max(largest, top);
        }
        if constexpr (kQueryPieces > kPieces) {
            // An element of a query is off by 2^-14 of the largest of them at most, with even odds anywhere below; a score by this over sqrt(3) times
            // sqrt(DP) elements of keys, which are some two times their scale.  Up to 2^-9 of an exponent of 2 are left.
            constexpr float kLeft = 0.001953125f * 1.7320508f / 2.0f / (DP == 64 ? 8.0f : DP == 128 ? 11.3137085f : 16.0f);
            const int exponent = (int)(group_max_u32<64>(largest) >> 23);
            matters = __builtin_amdgcn_ldexpf(kLeft, 127 + 14 - exponent);
        }
        for (; k + 4 < tile_to; k += 4) step(k, std::true_type());
        step(k, std::false_type());
    }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);

    // the four waves' results, joined
    if (lane < kRows) s_best[wave][lane] = best, s_sum[wave][lane] = sum;
    float *s_result = (float *)s_area[wave];
#pragma unroll
    for (int d = 0; d < kDTiles; ++d) *(f32x4 *)(s_result + column * (DP + 4) + 16 * d + 4 * g) = result[d];
    __syncthreads();
    for (int e = threadIdx.x; e < rows * DP; e += 256) {
        const int r = e / DP, d = e % DP;
        float top = s_best[0][r];
#pragma unroll
        for (int i = 1; i < 4; ++i) top = fmaxf(top, s_best[i][r]);
        const float zero = top == -__builtin_inff() ? 0.0f : top;
        float total = 0.0f, y = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float fade = __builtin_amdgcn_exp2f(s_best[i][r] - zero);
            total += s_sum[i][r] * fade;
            y += ((const float *)s_area[i])[r * (DP + 4) + d] * fade;
        }
        if (w.pieces > 1) {
            float *part = a.partial + (long long)(w.slot + w.piece) * kRows * (DP + 2) + r * (DP + 2);
            part[2 + d] = y;
            if (d == 0) part[0] = top, part[1] = total;
        } else if (d < a.shape.head_dim) {
            const int row = first_row + r;
            store_result<BF16>(a, (long long)(v.start + row / a.group) * a.out_token + (long long)(w.head * a.group + row % a.group) * a.out_head + d,
                               total == 0.0f ? 0.0f : y / total);
        }
    }
}

// Joins the pieces of every row of tiles that was cut, a workgroup for each of its rows: what the pieces count for first, then a
// share of them per group of DP / 4 threads.  Sums in a fixed order.  Bound by latency (about 5 us with its launch, of any number of pieces up
// to some hundred).  The last piece of a row to arrive could join them all in this order and save the launch; that takes a counter per row that is
// zero when a call begins and that no call on another stream shares, which scratch of the call is not.
template <int DP, bool BF16>
__global__ __launch_bounds__(256) void attend_join_kernel(const AttendArgs a) {
    constexpr int kGroups = 1024 / DP;
    __shared__ float s_share[256];
    __shared__ float s_reduce[4], s_total[4];
    __shared__ f32x4 s_part[256];
    AttendWork w;
    SequenceView v;
    if (!find_work<kRows, 7, false>(a, blockIdx.x, w, v) || w.pieces == 1) return;
    const int rows = v.count * a.group, row = first_row_of<kRows>(rows, w.row_tile) + blockIdx.y;
    if (row >= rows) return;
    constexpr int kNext = kRows * (DP + 2);
    const float *part = a.partial + (long long)w.slot * kNext + blockIdx.y * (DP + 2);
    const int wave = threadIdx.x >> 6;
    float top = -__builtin_inff();
    for (int i = threadIdx.x; i < w.pieces; i += 256) top = fmaxf(top, part[(long long)i * kNext]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
    if ((threadIdx.x & 63) == 0) s_reduce[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_reduce[0], s_reduce[1]), fmaxf(s_reduce[2], s_reduce[3]));
    const float zero = top == -__builtin_inff() ? 0.0f : top;
    const int group = threadIdx.x / (DP / 4), d = threadIdx.x % (DP / 4) * 4;
    float total = 0.0f;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    for (int first = 0; first < w.pieces; first += 256) {
        const int i = first + (int)threadIdx.x, count = min(256, w.pieces - first);
        __syncthreads();
        float share = 0.0f;
        if (i < w.pieces) {
            share = __builtin_amdgcn_exp2f(part[(long long)i * kNext] - zero);
            total += part[(long long)i * kNext + 1] * share;
        }
        s_share[threadIdx.x] = share;
        __syncthreads();
#pragma unroll 4
        for (int j = group; j < count; j += kGroups) {
            const float2 *p = (const float2 *)(part + (long long)(first + j) * kNext + 2 + d);
            const float2 u = p[0], v2 = p[1];
            const float by = s_share[j];
            y += (f32x4){u.x * by, u.y * by, v2.x * by, v2.y * by};
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
    if ((threadIdx.x & 63) == 0) s_total[wave] = total;
    s_part[threadIdx.x] = y;
    __syncthreads();
    total = (s_total[0] + s_total[1]) + (s_total[2] + s_total[3]);
    if (group != 0) return;
#pragma unroll
    for (int i = 1; i < kGroups; ++i) y += s_part[threadIdx.x + i * (DP / 4)];
    const long long at = (long long)(v.start + row / a.group) * a.out_token + (long long)(w.head * a.group + row % a.group) * a.out_head;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (d + e < a.shape.head_dim) store_result<BF16>(a, at + d + e, total == 0.0f ? 0.0f : y[e] / total);
}

// Workgroups that the device holds of the kernel for few.
int few_slots(int dim, int segments, bool bf16) { return compute_units() * few_waves(dim, dim == 64 || segments == 1 ? 1 : dim / 64, bf16); }

template <int DP, bool BF16>
void launch_few(const AttendArgs &a, unsigned rows_of_tiles, bool may_cut, hipStream_t stream) {
    // (with starts some workgroups more than there can be work for: they see to the rows of no sequence)
    const dim3 grid(rows_of_tiles + (may_cut ? (unsigned)a.slots : 0u) + (a.at.starts ? (unsigned)(a.at.tokens < 1024 ? (a.at.tokens + 15) / 16 : 64) : 0u));
    if (DP == 64 || a.shape.segments == 1) hipLaunchKernelGGL((attend_few_kernel<DP, 1, BF16>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((attend_few_kernel<DP, DP / 64, BF16>), grid, dim3(256), 0, stream, a);
    if (may_cut)
        hipLaunchKernelGGL((attend_join_kernel<DP, BF16>), dim3(rows_of_tiles, a.at.starts ? kRows : min(kRows, a.group)), dim3(256), 0, stream, a);
}

long long workspace_of(const CacheShape &shape, int group, bool bf16, bool ragged) {
    const int dim = attend_dim(shape.head_dim);
    const long long few = (long long)attend_places(few_slots(dim, shape.segments, bf16)) * kRows;
    const long long many = bf16 && (ragged || group > kFewRows) ? (long long)attend_places(attend_many_slots(dim)) * kRowsOfMany : 0;
    return (few > many ? few : many) * (dim + 2) * (long long)sizeof(float);
}

}  // namespace
}  // namespace qt

extern "C" long long qtensor_hip_cache_attend_workspace(const qtensor_cache *cache, int heads, int is_bf16, int has_starts) {
    using namespace qt;
    clear_error();
    CacheShape shape;
    if (!cache_shape("cache_attend_workspace", cache, shape)) return 0;
    return workspace_of(shape, heads / shape.kv_heads, is_bf16 != 0, has_starts != 0);
}

extern "C" void qtensor_hip_cache_attend(const qtensor_cache *cache, const qtensor_cache_places *places, const qtensor_cache_vectors *q,
                                         const qtensor_cache_vectors *out, int heads, float scale, int window, int sinks, void *workspace,
                                         long long workspace_bytes, void *stream_v) {
    using namespace qt;
    clear_error();
    AttendArgs a;
    if (!cache_shape("cache_attend", cache, a.shape) || !cache_places("cache_attend", places, a.at)) return;
    if (!q || !out || (a.at.tokens > 0 && (!q->base || !out->base))) { set_error(kNullPointer, "cache_attend: null queries or result"); return; }
    if (heads < 1 || heads > 32767 || heads % a.shape.kv_heads || window < 0 || sinks < 0 || !(scale - scale == 0.0f) || q->is_bf16 != out->is_bf16) {
        set_error(kBadArgument, "cache_attend: needs query heads that are a multiple of the cache's, a finite scale, window and sinks of at least 0 and a "
                                "result of the queries' type (got %d heads of %d, scale %g, window %d, sinks %d)", heads, a.shape.kv_heads, scale, window, sinks);
        return;
    }
    if (!is_aligned(q->base, q->is_bf16 ? 2 : 4) || !is_aligned(out->base, q->is_bf16 ? 2 : 4)) {
        set_error(kBadArgument, "cache_attend: queries or result not aligned to an element");
        return;
    }
    if (a.at.tokens == 0) return;
    for (int i = 0; i < 2; ++i) a.codes[i] = cache->codes[i], a.scales[i] = cache->scales[i];
    a.q = q->base, a.q_token = q->token_stride, a.q_head = q->head_stride;
    a.out = out->base, a.out_token = out->token_stride, a.out_head = out->head_stride;
    a.group = heads / a.shape.kv_heads;
    a.q_in_eights = q->is_bf16 && is_aligned(q->base, 16) && q->token_stride % 8 == 0 && q->head_stride % 8 == 0 && a.shape.head_dim % 8 == 0;
    a.factor = scale * 1.4426950408889634f;
    a.window = window, a.sinks = sinks;
    a.partial = (float *)workspace;
    const bool bf16 = q->is_bf16 != 0, ragged = a.at.starts != nullptr;
    const int dim = attend_dim(a.shape.head_dim);
    const long long rows = (long long)a.at.tokens * a.group, batch = a.at.batch;
    if (rows >= (1LL << 31) || (rows / kRows + batch) * a.shape.kv_heads >= (1LL << 30)) {
        set_error(kBadArgument, "cache_attend: %d tokens are too many for one call", a.at.tokens);
        return;
    }
    if (!workspace || !is_aligned(workspace, 16) || workspace_bytes < workspace_of(a.shape, a.group, bf16, ragged)) {
        set_error(kBadArgument, "cache_attend: the workspace is smaller than qtensor_hip_cache_attend_workspace says");
        return;
    }
    const hipStream_t stream = (hipStream_t)stream_v;
    const long long held = (long long)a.at.table_pages << a.shape.page_shift;        // most tokens of a sequence
    // Queries in 32 bits are all the kernel for few's, which has pieces enough for them; and all of a call that is too little work for a second
    // pair of launches (kFewWork).
    const bool few_alone = !bf16 || (double)rows * a.shape.kv_heads * (double)held <= kFewWork;
    a.few_rows = few_alone ? 0x7fffffff : kFewRows;
    if (!few_alone && (ragged ? rows : (long long)a.group) > kFewRows) {
        const long long rows_of_tiles = a.shape.kv_heads * (ragged ? rows / kRowsOfMany + batch : batch * ((a.group + kRowsOfMany - 1) / kRowsOfMany));
        AttendArgs many = a;
        many.slots = attend_many_slots(dim);
        // (not cut where whole rows of tiles keep every unit busy: 4 sequences of 4000 tokens, 4 heads, 4000 queries of each, 147 us, 151 with the
        // launch that joins; nor short ones: 32 of 700 tokens with 256 queries 31 us, cut 51)
        launch_attend_many(many, (unsigned)rows_of_tiles, held > 1024 && rows_of_tiles < many.slots, stream);
    }
    if (few_alone || ragged || a.group <= kFewRows) {
        // rows of tiles: at most one more per sequence than full ones, and no more per sequence than few queries have
        long long rows_of_tiles = ragged ? rows / kRows + batch : batch * ((a.group + kRows - 1) / kRows);
        if (!few_alone) rows_of_tiles = rows_of_tiles < batch * (kFewRows / kRows) ? rows_of_tiles : batch * (kFewRows / kRows);
        long long tiles = (held + kTile - 1) / kTile;
        if (window) {
            const long long seen = ((long long)window + (ragged ? kFewRows : 1) + kTile - 2) / kTile + 1 + ((long long)sinks + kTile - 1) / kTile;
            if ((!few_alone || !ragged) && seen < tiles) tiles = seen;
        }
        const bool may_cut = tiles > kWholeTiles;
        a.slots = few_slots(dim, a.shape.segments, bf16);
        a.least = may_cut ? kLeastTiles : 1 << 28;
        const unsigned n = (unsigned)(rows_of_tiles * a.shape.kv_heads);
        auto launch = dim == 64 ? (bf16 ? launch_few<64, true> : launch_few<64, false>)
                    : dim == 128 ? (bf16 ? launch_few<128, true> : launch_few<128, false>)
                                 : (bf16 ? launch_few<256, true> : launch_few<256, false>);
        launch(a, n, may_cut, stream);
    }
    launch_ok("cache_attend");
}
