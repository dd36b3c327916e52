// Weights that the tokens of a 4-bit attention cache are given, summed for each head of the cache: what decides which tokens are kept.
//
// For every new token i and query head g of a cache's head h, w(i, g, t) = 2^(s(t) - m) / l over the tokens t that i sees, s = scale log2(e) q k, m the
// largest and l the sum of 2^(s - m); totals[b][h][t] += sum over i and g of w.  As t is summed over first and i afterwards, the scores are
// worked out twice: once a row (i, g) at a time for m and l, once a token at a time for the sums, instead of being kept (a score is 4
// bytes, as much as a key's 8 elements); but where each sequence has one token they are, if there is room.  Every sum has one order: results do not change from call to call.
//
// Scores come from the matrix cores with all bits: keys' numbers are exact in bf16, fp32 queries go through in three pieces (qt_fp4.h).
#include "qt_cache.h"

#define QT_CONSTANT __attribute__((address_space(4)))

namespace qt {
namespace {

constexpr int kWeighThreads = 256, kWeighWaves = 4;
constexpr int kMostParts = 64;         // of a row's tokens
constexpr int kLeastTiles = 16;        // of a part
constexpr long long kMostTokens = 0x7fffff00;       // of a sequence

struct WeighArgs {
    CacheShape shape;
    CachePlaces at;
    const uint8_t *codes;
    const float *scales;
    long long code_page, scale_page;    // bytes and scales of a page
    const void *q;
    long long q_token, q_head;
    int group;
    float factor;                       // scale * log2 e
    int window, sinks;                  // window 0: no window
    float *totals;
    long long total_sequence, total_head;
    float2 *partial;                    // [head][row][parts]: (m, l) of each part of a row's tokens, rows of all sequences in order
    float2 *statistics;                 // [head][row]: (m, 1 / l); (0, 0) where nothing is seen
    float *scores;                      // [sequence][head][group][score_stride]: of the only token of a sequence, or null
    long long score_stride;
    int parts;                          // at most
    long long wanted;                   // workgroups that the rows' work is cut for
    FastDiv by_group, by_tiles;         // and by tiles of rows of a token
    float *sums;                        // [row part][sequence][head][sums_stride]: of the rows of a token cut into row_parts, if these are more than one
    long long sums_stride;
    int row_parts;
};

// Rows (i, g) of a sequence and what they see.
struct WeighSequence {
    int start, count, first_position, end;

    __device__ __forceinline__ int position(const WeighArgs &a, int row) const { return first_position + (int)fastdiv((uint32_t)row, a.by_group); }
};
// Where a row's statistics lie.
__device__ __forceinline__ long long row_entry(const WeighArgs &a, const WeighSequence &v, int head, int row) {
    return ((long long)head * a.at.tokens + v.start) * a.group + row;
}
template <bool UNIFORM>
__device__ __forceinline__ int load_int(const int *p) {
    return UNIFORM ? *(const QT_CONSTANT int *)p : *p;
}
// UNIFORM: b is the same for all lanes
template <bool UNIFORM>
__device__ __forceinline__ WeighSequence weigh_sequence(const WeighArgs &a, int b) {
    WeighSequence v;
    const int length = load_int<UNIFORM>(a.at.lengths + b);
    v.start = a.at.starts ? load_int<UNIFORM>(a.at.starts + b) : b;
    v.count = a.at.starts ? load_int<UNIFORM>(a.at.starts + b + 1) - v.start : 1;
    if (v.start < 0 || v.count < 0 || (long long)v.start + v.count > a.at.tokens) v.count = 0;      // (not a list of starts: nothing)
    v.first_position = length - v.count;
    const long long covered = (long long)a.at.table_pages << a.shape.page_shift;
    v.end = (int)min((long long)max(length, 0), min(covered, kMostTokens));
    return v;
}

__device__ __forceinline__ bool row_sees(const WeighArgs &a, int position, int token) {
    return token <= position && (!a.window || position - token < a.window || token < a.sinks);
}

// Sixteen rows as a matrix operand: STEPS of 32 elements.  SIDE: loaded by four lanes side by side a row, which touches a row's line once instead of four
// times, and exchanged.
template <bool BF16, int STEPS, bool SIDE>
struct WeighRows {
    bf16x8 x[STEPS][Eight<BF16>::kPieces];

    Eight<BF16> raw[STEPS];

    __device__ __forceinline__ void fetch(const WeighArgs &a, const WeighSequence &v, int head, int first_row) {
        const int lane = threadIdx.x & 63, quarter = SIDE ? lane & 3 : lane >> 4;
        const int row = min(first_row + (SIDE ? lane >> 2 : lane & 15), v.count * a.group - 1), i = (int)fastdiv((uint32_t)row, a.by_group);
        const int steps = a.shape.row_bytes >> 4;
        const uint8_t *p = (const uint8_t *)a.q + ((v.start + i) * a.q_token + (head * a.group + row - i * a.group) * a.q_head + 8 * quarter) * (BF16 ? 2 : 4);
        if (a.shape.head_dim == 32 * STEPS) {
#pragma unroll
            for (int j = 0; j < STEPS; ++j) raw[j].load(p, 32 * j);
        } else {
#pragma unroll
            for (int j = 0; j < STEPS; ++j) {
                raw[j].zero();
                if (j < steps) raw[j].load(p, 32 * j, a.shape.head_dim - 8 * quarter);
            }
        }
    }
    // (rows behind the last are the last one again: what comes of them is not used)
    __device__ __forceinline__ void arrange() {
#pragma unroll
        for (int j = 0; j < STEPS; ++j) {
            if (SIDE) raw[j].exchange();
            raw[j].pieces(x[j]);
        }
    }
};

// Four words of the lanes l, l + 16, l + 32, l + 48: word j of the qth of them and word q of the jth change places.
__device__ __forceinline__ void transpose_quarters(uint32_t *w) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const auto two = __builtin_amdgcn_permlane32_swap(w[i], w[i + 2], false, false);
        w[i] = two[0], w[i + 2] = two[1];
    }
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const auto two = __builtin_amdgcn_permlane16_swap(w[i], w[i + 1], false, false);
        w[i] = two[0], w[i + 1] = two[1];
    }
}
// Word q of lane l to all of l % 16 + 16 i, where it is that of lane l % 16 + 16 q.
__device__ __forceinline__ void spread_quarters(uint32_t w, uint32_t *each) {
    const auto halves = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    const auto low = __builtin_amdgcn_permlane16_swap(halves[0], halves[0], false, false), high = __builtin_amdgcn_permlane16_swap(halves[1], halves[1], false, false);
    each[0] = low[0], each[1] = low[1], each[2] = high[0], each[3] = high[1];
}

// Keys of N tiles of sixteen tokens: numbers as matrix operands want them, eight of each step of 32 elements a lane, and scales.  Lanes load sixteen
// bytes, a quarter of the wave a step of all tokens, and exchange words; scales likewise, a quarter 64 elements (which are in one segment of any size).
template <int STEPS, int N>
struct WeighKeys {
    static constexpr int kSegments = STEPS / 2, kFetches = N * STEPS / 4, kScales = N * kSegments / 4;
    qt_u32x4 raw[kFetches];
    float raw_scale[kScales];
    bool there[N];
    uint32_t word[N][STEPS];
    float scale[N][kSegments];

    // asks for tile `first` and those behind it, of sequence b in front of `end`; `first` a multiple of N and the same for all lanes
    __device__ __forceinline__ void fetch(const WeighArgs &a, int b, int head, int first, int end) {
        const int lane = threadIdx.x & 63, quarter = lane >> 4, token = lane & 15, steps = a.shape.row_bytes >> 4;
        // (steps and segments that the heads do not have are the first and the last one again: queries are zero there)
        const auto page_of = [&](int tile) {
            const int at = tile << 4;
            return at < end ? load_int<true>(a.at.table + b * a.at.table_stride + (at >> a.shape.page_shift)) : -1;
        };
        const auto codes_of = [&](int page, int tile) {
            return a.codes + (long long)page * a.code_page + (((long long)head << a.shape.page_shift) + ((tile << 4) & ((1 << a.shape.page_shift) - 1))) * a.shape.row_bytes;
        };
        const auto scales_of = [&](int page, int tile) {
            return a.scales + (long long)page * a.scale_page + ((long long)(head * a.shape.segments) << a.shape.page_shift) + ((tile << 4) & ((1 << a.shape.page_shift) - 1));
        };
        const auto step_of = [&](int f) {                   // what a lane loads of a tile: a step, and for short heads one of two tiles
            const int step = STEPS == 2 ? quarter & 1 : quarter + 4 * (f % (STEPS / 4));
            return (token + (STEPS == 2 ? 16 * (quarter >> 1) : 0)) * a.shape.row_bytes + (step < steps ? 16 * step : 0);
        };
        const auto segment_of = [&](int f) { return min(((4 * f + quarter) % kSegments) >> (a.shape.segment_shift - 6), a.shape.segments - 1) << a.shape.page_shift; };
        if (16 * N <= 1 << a.shape.page_shift) {
            const int page = page_of(first);
            const bool is = (unsigned)page < (unsigned)a.shape.pages;
            const uint8_t *codes = codes_of(is ? page : 0, first);
            const float *scales = scales_of(is ? page : 0, first);
#pragma unroll
            for (int n = 0; n < N; ++n) there[n] = is;
#pragma unroll
            for (int f = 0; f < kFetches; ++f) {
                const int n = STEPS == 2 ? 2 * f : f / (STEPS / 4);
                raw[f] = *(const qt_u32x4 *)(codes + (uint32_t)(step_of(f) + 16 * n * a.shape.row_bytes));
            }
#pragma unroll
            for (int f = 0; f < kScales; ++f) raw_scale[f] = scales[(uint32_t)(segment_of(f) + 16 * ((4 * f + quarter) / kSegments) + token)];
        } else {
            const uint8_t *codes[N];
            const float *scales[N];
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int page = page_of(first + n);
                there[n] = (unsigned)page < (unsigned)a.shape.pages;
                codes[n] = codes_of(there[n] ? page : 0, first + n), scales[n] = scales_of(there[n] ? page : 0, first + n);
            }
#pragma unroll
            for (int f = 0; f < kFetches; ++f) {
                if constexpr (STEPS == 2) raw[f] = *(const qt_u32x4 *)((quarter < 2 ? codes[2 * f] : codes[2 * f + 1] - 16 * a.shape.row_bytes) + step_of(f));
                else raw[f] = *(const qt_u32x4 *)(codes[f / (STEPS / 4)] + step_of(f));
            }
#pragma unroll
            for (int f = 0; f < kScales; ++f) {
                const float *p = scales[(4 * f) / kSegments];
#pragma unroll
                for (int q = 1; q < 4; ++q) p = quarter == q ? scales[(4 * f + q) / kSegments] : p;
                raw_scale[f] = p[segment_of(f) + token];
            }
        }
    }
    __device__ __forceinline__ void arrange(float factor) {
#pragma unroll
        for (int f = 0; f < kFetches; ++f) {
            uint32_t w[4] = {raw[f][0], raw[f][1], raw[f][2], raw[f][3]};
            transpose_quarters(w);
#pragma unroll
            for (int i = 0; i < 4; ++i) word[(4 * f + i) / STEPS][(4 * f + i) % STEPS] = w[i];
        }
#pragma unroll
        for (int f = 0; f < kScales; ++f) {
            uint32_t each[4];
            spread_quarters(__float_as_uint(raw_scale[f] * factor), each);
#pragma unroll
            for (int q = 0; q < 4; ++q) scale[(4 * f + q) / kSegments][(4 * f + q) % kSegments] = __uint_as_float(each[q]);
        }
    }
};

// Scores of sixteen rows (4 (lane / 16) + i) and a token (lane % 16), times log2 e: `numbers` are its keys' numbers, `scale` has the factor already.
template <bool BF16, int STEPS, bool SIDE>
__device__ __forceinline__ fp4_f32x4 weigh_scores(const WeighRows<BF16, STEPS, SIDE> &rows, const bf16x8 *numbers, const float *scale) {
    constexpr int P = Eight<BF16>::kPieces;
    fp4_f32x4 sum;
#pragma unroll
    for (int g = 0; g < STEPS / 2; ++g) {
        const fp4_f32x4 part = multiply_pieces<P>(rows.x[2 * g + 1], numbers[2 * g + 1], multiply_pieces<P>(rows.x[2 * g], numbers[2 * g], (fp4_f32x4){0.f, 0.f, 0.f, 0.f}));
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = g ? __builtin_fmaf(scale[g], part[i], sum[i]) : scale[g] * part[i];
    }
    return sum;
}

// The same from the segments' products of N tiles, for the nth.
template <int STEPS, int N>
__device__ __forceinline__ fp4_f32x4 scale_scores(const fp4_f32x4 (&part)[STEPS / 2][N], int n, const float *scale) {
    fp4_f32x4 sum;
#pragma unroll
    for (int g = 0; g < STEPS / 2; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = g ? __builtin_fmaf(scale[g], part[g][n][i], sum[i]) : scale[g] * part[g][n][i];
    return sum;
}

// Over the sixteen lanes of a row of the wave, and over its four rows, for all lanes.
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float x) { return __uint_as_float(dpp_u32<CTRL>(__float_as_uint(x))); }
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, dpp_f32<0xB1>(x)), x = fmaxf(x, dpp_f32<0x4E>(x)), x = fmaxf(x, dpp_f32<0x141>(x));
    return fmaxf(x, dpp_f32<0x140>(x));
}
__device__ __forceinline__ float row_sum(float x) {
    x += dpp_f32<0xB1>(x), x += dpp_f32<0x4E>(x), x += dpp_f32<0x141>(x);
    return x + dpp_f32<0x140>(x);
}
__device__ __forceinline__ float quarters_sum(float x) {
    const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const uint32_t both = __float_as_uint(__uint_as_float(halves[0]) + __uint_as_float(halves[1]));
    const auto rest = __builtin_amdgcn_permlane16_swap(both, both, false, false);
    return __uint_as_float(rest[0]) + __uint_as_float(rest[1]);
}
__device__ __forceinline__ float quarters_max(float x) {
    const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const uint32_t both = __float_as_uint(fmaxf(__uint_as_float(halves[0]), __uint_as_float(halves[1])));
    const auto rest = __builtin_amdgcn_permlane16_swap(both, both, false, false);
    return fmaxf(__uint_as_float(rest[0]), __uint_as_float(rest[1]));
}

// Joins (m, l) of two parts of a row.
__device__ __forceinline__ float2 join_parts(float2 x, float2 y) {
    const float m = fmaxf(x.x, y.x), by = m == -INFINITY ? 0.0f : m;
    return make_float2(m, x.y * __builtin_amdgcn_exp2f(x.x - by) + y.y * __builtin_amdgcn_exp2f(y.x - by));
}

// Whether a row's query has an infinite element: its scores are infinities of either sign or NaN, and the formula's weights NaN; minus infinities alone would pass for
// tokens that are not seen.  Looked for where a row has nothing else (infinities made NaN in front of the products cost 2 % of a call).
template <bool BF16>
__device__ __forceinline__ bool row_is_infinite(const WeighArgs &a, const WeighSequence &v, int head, int row) {
    const int i = (int)fastdiv((uint32_t)row, a.by_group);
    const uint8_t *p = (const uint8_t *)a.q + ((v.start + i) * a.q_token + (head * a.group + row - i * a.group) * a.q_head) * (BF16 ? 2 : 4);
    bool found = false;
#pragma unroll 4
    for (int d = 0; d < a.shape.head_dim; d += 8) {
        Eight<BF16> x;
        x.load(p, d, a.shape.head_dim);
#pragma unroll
        for (const uint32_t r : x.raw) found |= BF16 ? (r & 0x7fffu) == 0x7f80u || (r & 0x7fff0000u) == 0x7f800000u : (r & 0x7fffffffu) == 0x7f800000u;
    }
    return found;
}

// (m, 1 / l) of the row `first_row` + lane % 16, from its parts; (0, 0) where nothing is seen, (infinity, 0) behind the last row.
template <bool BF16>
__device__ __forceinline__ float2 row_statistics(const WeighArgs &a, const WeighSequence &v, int head, int first_row) {
    const int lane = threadIdx.x & 63, quarter = lane >> 4, row = first_row + (lane & 15);
    float m = -INFINITY, l = 0.0f;
    const float2 *p = a.partial + row_entry(a, v, head, min(row, v.count * a.group - 1)) * a.parts;
    for (int first = 0; first < a.parts; first += 16) {
        float2 each[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int at = first + 4 * n + quarter;
            each[n] = at < a.parts ? p[at] : make_float2(-INFINITY, 0.0f);
        }
        const float top = fmaxf(fmaxf(fmaxf(each[0].x, each[1].x), fmaxf(each[2].x, each[3].x)), m), by = top == -INFINITY ? 0.0f : top;
        l *= __builtin_amdgcn_exp2f(m - by);
#pragma unroll
        for (int n = 0; n < 4; ++n) l += each[n].y * __builtin_amdgcn_exp2f(each[n].x - by);
        m = top;
    }
    const float mine = m;
    m = quarters_max(m);
    m = m == -INFINITY ? 0.0f : m;
    l = quarters_sum(l * __builtin_amdgcn_exp2f(mine - m));
    if (l == 0.0f && row < v.count * a.group && row_is_infinite<BF16>(a, v, head, row)) l = NAN;
    return row < v.count * a.group ? make_float2(m, l == 0.0f ? 0.0f : 1.0f / l) : make_float2(INFINITY, 0.0f);
}

// Sums over the rows of N tiles' tokens (lane % 16): of the tile lane / 16, or with two of lane / 32.
template <int N>
__device__ __forceinline__ float sum_of_rows(const float *sum) {
    if constexpr (N == 4) {
        uint32_t w[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) w[n] = __float_as_uint(sum[n]);
        transpose_quarters(w);
        return (__uint_as_float(w[0]) + __uint_as_float(w[1])) + (__uint_as_float(w[2]) + __uint_as_float(w[3]));
    } else {
        const auto two = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum[0]), __float_as_uint(sum[1]), false, false);
        const uint32_t half = __float_as_uint(__uint_as_float(two[0]) + __uint_as_float(two[1]));
        const auto both = __builtin_amdgcn_permlane16_swap(half, half, false, false);
        return __uint_as_float(both[0]) + __uint_as_float(both[1]);
    }
}

// Tiles of sixteen tokens that rows at `nearest` to `furthest` see of a sequence with `end` tokens: `sink_tiles` from the first, then `first_tile` and
// those behind it, both whole fours.
struct WeighView { int first_tile, sink_tiles, tiles; };
__device__ __forceinline__ WeighView weigh_view(const WeighArgs &a, int nearest, int furthest, int end) {
    const int high = min(furthest + 1, end);
    const int low = a.window ? min(max(high, 0), max(0, max(nearest, 0) - (a.window - 1))) : 0;
    WeighView w;
    w.first_tile = (low >> 4) & ~3, w.sink_tiles = min((int)(((long long)min(a.sinks, low) + 63) >> 6) * 4, w.first_tile);
    w.tiles = high <= 0 ? 0 : w.sink_tiles + ((high + 15) >> 4) - w.first_tile;
    return w;
}

// The `index`th piece of work of the call: ROWS rows of a sequence, and which of how many parts of the tokens that they see, of `each` tiles.  Every part of
// all rows has as many tiles as make a.wanted of them, at least kLeastTiles and no more than a.parts for a row; a sequence's rows have equally many.
struct WeighWork { int b, first_row, part, parts, each; };
template <int ROWS>
__device__ __forceinline__ bool find_work(const WeighArgs &a, int index, WeighWork &w) {
    const int lane = threadIdx.x & 63;
    if (!a.at.starts && a.parts == 1) {
        const int b = (int)fastdiv((uint32_t)index, a.by_tiles);
        w = {b, (index - b * ((a.group + ROWS - 1) / ROWS)) * ROWS, 0, 1, 0x7fffffff};
        return b < a.at.batch;
    }
    int rows = 0, tiles = 0;                            // tiles of rows of this lane's sequence, of tokens that any of them may see
    const auto look = [&](int b) {
        rows = tiles = 0;
        if (b >= a.at.batch) return;
        const WeighSequence v = weigh_sequence<false>(a, b);
        rows = (v.count * a.group + ROWS - 1) / ROWS;
        tiles = weigh_view(a, v.first_position, v.first_position + v.count - 1, v.end).tiles;
        // (with a window fewer than the whole call's: sinks in whole fours, the window and as many places more as rows, from a whole four on)
        if (a.window) tiles = (int)min((long long)tiles, (((long long)a.sinks + 63) >> 6) * 4 + (((long long)a.window + ROWS + 63) >> 4) + 2);
    };
    int least = kLeastTiles;
    if (a.parts > 1) {
        float all = 0.0f;
        for (int first = 0; first < a.at.batch; first += 64) {
            look(first + lane);
            all += (float)rows * (float)tiles;
        }
        all = quarters_sum(row_sum(all));
        least = max(least, (int)fminf(ceilf(all * (float)a.shape.kv_heads / (float)a.wanted), 1.0e9f));
    }
    int before = 0;
    for (int first = 0; first < a.at.batch; first += 64) {
        if (a.parts == 1 || a.at.batch > 64) look(first + lane);
        const int each = (max(least, (int)((uint32_t)(tiles + a.parts - 1) / (uint32_t)a.parts)) + 3) & ~3;
        const int parts = a.parts == 1 ? 1 : max(1, (int)((uint32_t)(tiles + each - 1) / (uint32_t)each));
        int upto = rows * parts;
#pragma unroll
        for (int off = 1; off < 64; off *= 2) {
            const int other = __shfl_up(upto, off, 64);
            if (lane >= off) upto += other;
        }
        const unsigned long long at = __ballot(index < before + upto);
        if (at) {
            const int found = __builtin_ctzll(at);
            w.b = first + found;
            w.parts = __builtin_amdgcn_readlane(parts, found), w.each = a.parts == 1 ? 0x7fffffff : __builtin_amdgcn_readlane(each, found);
            const int nth = index - before - __builtin_amdgcn_readlane(upto - rows * parts, found);
            const int tile = (int)((uint32_t)nth / (uint32_t)w.parts);
            w.first_row = tile * ROWS, w.part = nth - tile * w.parts;
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// 16 T rows and a part of the tokens that they see: m and l of each, or (WEIGHTS, where a sequence has no more rows than these) the
// weights themselves, added to the totals.  A wave goes through the tokens of its part 16 N at a time, the next ones' keys on their way.
//
// A step of 32 sequences of 100 to 8000 tokens, 8 heads of 128, groups of 4, bf16: 26 us for 85 MB of keys and scores written, 3.3 TB/s; 4 us are the
// launch and the work found, 2.5 to 5 the first keys (length, page, keys: three loads that wait for each other), and a part has so few tokens that this is a third of its
// time.  The last 1 to 27 tokens of four prompts of up to 32768, two tiles of rows at a time: 29 us.  No pipe is full (vector instructions, exponentials, scales and numbers
// expanded, in 50 % of all cycles, matrix ones in 11 %): too few waves, 1.6 a SIMD on average, hide each other's loads and results, as each holds two tiles of rows and four
// of keys in registers.  Tried: scores of a step transposed, so that no lane works on rows that are not there (31 us against 28: more registers), all tiles' products in
// front (31 against 29).
template <bool BF16, int STEPS, int T, bool WEIGHTS>
__global__ __launch_bounds__(kWeighThreads, STEPS == 8 || T > 1 ? 2 : BF16 ? 4 : 3) void weigh_rows_kernel(const WeighArgs a) {
    static_assert(T == 1 || !WEIGHTS, "weights of sixteen rows");
    constexpr int N = STEPS == 8 ? 2 : 4, kRows = 16 * T;
    __shared__ float2 s_part[kWeighWaves][kRows];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quarter = lane >> 4;
    // (heads first: workgroups without work, of which the host knows no better, are the last ones)
    const int head = blockIdx.x;
    WeighWork work;
    if (!find_work<kRows>(a, (int)(blockIdx.y + gridDim.y * blockIdx.z), work)) return;
    const int b = __builtin_amdgcn_readfirstlane(work.b), first_row = __builtin_amdgcn_readfirstlane(work.first_row);
    const WeighSequence v = weigh_sequence<true>(a, b);
    const int rows = v.count * a.group;
    if (first_row >= rows) return;
    const int nearest = v.position(a, first_row), furthest = v.position(a, min(rows, first_row + kRows) - 1);
    const WeighView view = weigh_view(a, nearest, furthest, v.end);
    const int each = __builtin_amdgcn_readfirstlane(work.each), nth = __builtin_amdgcn_readfirstlane(work.part);
    const int from = (int)min((long long)view.tiles, (long long)nth * each), to = (int)min((long long)view.tiles, (long long)from + each);
    if (!WEIGHTS && nth == work.parts - 1) {
        // (parts of other sequences' rows)
        const int row = first_row + (int)threadIdx.x % kRows;
        for (int n = work.parts + (int)threadIdx.x / kRows; n < a.parts && row < rows; n += kWeighThreads / kRows)
            a.partial[row_entry(a, v, head, row) * a.parts + n] = make_float2(-INFINITY, 0.0f);
    }
    const auto put = [&](float2 part) {
        const long long entry = row_entry(a, v, head, first_row + (int)threadIdx.x);
        if (a.parts == 1 && a.statistics)
            a.statistics[entry] = make_float2(part.x == -INFINITY ? 0.0f : part.x, part.y == 0.0f ? 0.0f : 1.0f / part.y);
        else
            a.partial[entry * a.parts + nth] = part;
    };
    if (from >= to) {
        if (!WEIGHTS && threadIdx.x < kRows && first_row + (int)threadIdx.x < rows) put(make_float2(-INFINITY, 0.0f));
        return;
    }
    const auto tile_at = [&](int index) { return index < view.sink_tiles ? index : view.first_tile + index - view.sink_tiles; };
    WeighRows<BF16, STEPS, false> q[T];
#pragma unroll
    for (int r = 0; r < T; ++r) q[r].fetch(a, v, head, first_row + 16 * r);
    WeighKeys<STEPS, N> keys;
    int tile = 0;
    const int first = from + wave * N;
    if (first < to) {
        tile = tile_at(first);
        keys.fetch(a, b, head, tile, v.end);
    }
#pragma unroll
    for (int r = 0; r < T; ++r) q[r].arrange();
    float m[T][4], l[T][4];             // WEIGHTS: 1 / l
    if constexpr (WEIGHTS) {
        const float2 part = row_statistics<BF16>(a, v, head, first_row);
#pragma unroll
        for (int i = 0; i < 4; ++i) m[0][i] = __shfl(part.x, 4 * quarter + i, 64), l[0][i] = __shfl(part.y, 4 * quarter + i, 64);
    } else {
#pragma unroll
        for (int r = 0; r < T; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) m[r][i] = -INFINITY, l[r][i] = 0.0f;
    }
    for (int index = first; index < to; index += kWeighWaves * N) {
        keys.arrange(a.factor);
        const int token = tile << 4;
        bool there[N], all = token + 16 * N - 1 <= nearest && token + 16 * N <= v.end && (!a.window || furthest - token < a.window || token + 16 * N <= a.sinks);
#pragma unroll
        for (int n = 0; n < N; ++n) there[n] = keys.there[n], all = all && there[n];
        if (index + kWeighWaves * N < to) {
            tile = tile_at(index + kWeighWaves * N);
            keys.fetch(a, b, head, tile, v.end);
        }
        fp4_f32x4 s[T][N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            bf16x8 numbers[STEPS];
#pragma unroll
            for (int j = 0; j < STEPS; ++j) numbers[j] = fp4_to_bf16(keys.word[n][j]);
#pragma unroll
            for (int r = 0; r < T; ++r) s[r][n] = weigh_scores(q[r], numbers, keys.scale[n]);
        }
        if (!all) {
#pragma unroll
            for (int r = 0; r < T; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = first_row + 16 * r + 4 * quarter + i, position = row < rows ? v.position(a, row) : -1;
#pragma unroll
                    for (int n = 0; n < N; ++n) {
                        const int t = token + 16 * n + (lane & 15);
                        s[r][n][i] = there[n] && t < v.end && row_sees(a, position, t) ? s[r][n][i] : -INFINITY;
                    }
                }
        }
        if constexpr (T == 1 && !WEIGHTS) {
            if (a.scores) {
                // (a row's scores change places so that the lanes of a wave hold tokens side by side)
                float *to = a.scores + ((long long)b * a.shape.kv_heads + head) * a.group * a.score_stride + token + lane;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (i >= a.group) break;
                    uint32_t w[4];
#pragma unroll
                    for (int n = 0; n < 4; ++n) w[n] = n < N ? __float_as_uint(s[0][n][i]) : 0u;
                    transpose_quarters(w);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (4 * r + i < a.group && lane < 16 * N) to[(4 * r + i) * a.score_stride] = __uint_as_float(w[r]);
                }
            }
        }
        if constexpr (WEIGHTS) {
            float sum[N];
#pragma unroll
            for (int n = 0; n < N; ++n) {
                sum[n] = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[n] = __builtin_fmaf(__builtin_amdgcn_exp2f(s[0][n][i] - m[0][i]), l[0][i], sum[n]);
            }
            const float weight = sum_of_rows<N>(sum);
            const int mine = N == 4 ? quarter : quarter >> 1, t = token + 16 * mine + (lane & 15);
            bool is = N == 4 || (quarter & 1) == 0;
#pragma unroll
            for (int n = 0; n < N; ++n) is = is && (mine != n || there[n]);
            if (is && t < v.end && row_sees(a, furthest, t)) a.totals[b * a.total_sequence + head * a.total_head + t] += weight;
        } else {
#pragma unroll
            for (int r = 0; r < T; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float top = m[r][i];
#pragma unroll
                    for (int n = 0; n < N; ++n) top = fmaxf(top, s[r][n][i]);
                    const float by = top == -INFINITY ? 0.0f : top;
                    l[r][i] *= __builtin_amdgcn_exp2f(m[r][i] - by);
#pragma unroll
                    for (int n = 0; n < N; ++n) l[r][i] += __builtin_amdgcn_exp2f(s[r][n][i] - by);
                    m[r][i] = top;
                }
        }
    }
    if constexpr (!WEIGHTS) {
#pragma unroll
        for (int r = 0; r < T; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float top = row_max(m[r][i]), by = top == -INFINITY ? 0.0f : top;
                const float all = row_sum(l[r][i] * __builtin_amdgcn_exp2f(m[r][i] - by));
                if ((lane & 15) == 0) s_part[wave][16 * r + 4 * quarter + i] = make_float2(top, all);
            }
        __syncthreads();
        if (threadIdx.x < kRows && first_row + (int)threadIdx.x < rows) {
            float2 part = s_part[0][threadIdx.x];
#pragma unroll
            for (int w = 1; w < kWeighWaves; ++w) part = join_parts(part, s_part[w][threadIdx.x]);
            // (a token of each sequence: when the parts are joined; not for rows in front of the part: 20 over 8193 tokens 19.8 us, else 21.4)
            const int row = first_row + (int)threadIdx.x;
            if (!(BF16 && T == 1) && part.x == -INFINITY && v.position(a, row) >= tile_at(from) << 4 && row_is_infinite<BF16>(a, v, head, row)) part.y = NAN;
            put(part);
        }
    }
}

// Weights of the only token of a sequence from its scores: four tokens a thread.  Bound by latency, length to scores: 9.3 us for the step above, whose 25 MB
// are 5 us at a copy's rate; 10.5 with the statistics in front of the loads.
template <bool BF16>
__global__ __launch_bounds__(kWeighThreads) void weigh_scores_kernel(const WeighArgs a) {
    __shared__ float2 s_row[16];
    const int head = blockIdx.y, b = blockIdx.z, first = (int)blockIdx.x * 4 * kWeighThreads;
    const WeighSequence v = weigh_sequence<true>(a, b);
    const WeighView view = weigh_view(a, v.first_position, v.first_position, v.end);
    const int end = min(v.first_position + 1, v.end);
    if (first >= end) return;
    // (what is read hangs on the length alone)
    constexpr int kAhead = 4;
    const int token = first + 4 * (int)threadIdx.x;
    const bool mine = token < end && (token < 16 * view.sink_tiles || token >= 16 * view.first_tile);
    float *total = a.totals + b * a.total_sequence + head * a.total_head + token;
    const float *from = a.scores + ((long long)b * a.shape.kv_heads + head) * a.group * a.score_stride + token;
    int page = -1;
    float4 ahead[kAhead];
    qt_u32x4 before;
    if (mine) {
        page = a.at.table[b * a.at.table_stride + (token >> a.shape.page_shift)];
#pragma unroll
        for (int g = 0; g < kAhead; ++g) ahead[g] = load_f32x4<true>(from + min(g, a.group - 1) * a.score_stride);
        before = ((const Unaligned16of4 *)total)->v;
    }
    if (threadIdx.x < 64) {
        const float2 row = row_statistics<BF16>(a, v, head, 0);
        if (threadIdx.x < 16) s_row[threadIdx.x] = row;
    }
    __syncthreads();
    if ((unsigned)page >= (unsigned)a.shape.pages) return;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const auto add = [&](const float4 &s, int g) {
        const float2 row = s_row[g];
        sum[0] = __builtin_fmaf(__builtin_amdgcn_exp2f(s.x - row.x), row.y, sum[0]), sum[1] = __builtin_fmaf(__builtin_amdgcn_exp2f(s.y - row.x), row.y, sum[1]);
        sum[2] = __builtin_fmaf(__builtin_amdgcn_exp2f(s.z - row.x), row.y, sum[2]), sum[3] = __builtin_fmaf(__builtin_amdgcn_exp2f(s.w - row.x), row.y, sum[3]);
    };
#pragma unroll
    for (int g = 0; g < kAhead; ++g)
        if (g < a.group) add(ahead[g], g);
    for (int g = kAhead; g < a.group; ++g) add(load_f32x4<true>(from + g * a.score_stride), g);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (token + e < end && row_sees(a, v.first_position, token + e)) total[e] = __uint_as_float(before[e]) + sum[e];
}

// (m, 1 / l) of every row from its parts, sixteen lanes a row: of all rows that a sequence may have (what is behind the last sequence is not used).
// A launch and two loads: 4.7 us for 1440 rows in 21 parts.
__global__ __launch_bounds__(kWeighThreads) void weigh_join_kernel(const WeighArgs a, long long entries) {
    const long long entry = ((long long)blockIdx.x * kWeighThreads + threadIdx.x) >> 4;
    float2 part = make_float2(-INFINITY, 0.0f);
    for (int n = threadIdx.x & 15; n < a.parts && entry < entries; n += 16) part = join_parts(part, a.partial[entry * a.parts + n]);
    const float top = row_max(part.x), m = top == -INFINITY ? 0.0f : top;
    const float l = row_sum(part.y * __builtin_amdgcn_exp2f(part.x - m));
    if (entry < entries && (threadIdx.x & 15) == 0) a.statistics[entry] = make_float2(m, l == 0.0f ? 0.0f : 1.0f / l);
}

// Groups of 16 N tokens of all sequences that rows see, one sequence after the other, cut into parts of equal cost: a group's is its ROWS rows at a time, and
// two more for its keys.  (Groups in turn: the waves with most of the longest work took half as long again as all on average.)
struct WeighGroup { int b, first; WeighSequence v; };
template <int N, int ROWS>
struct WeighGroups {
    typedef unsigned long long Cost;
    int block;                          // of 64 sequences, one a lane:
    int groups, sinks, skip, cost;      // groups, those of sinks, what is left out behind these, cost of each
    Cost before;                        // of all groups in front of the sequence's
    Cost base;                          // of the sequences behind the block
    Cost at, end;                       // the next group's, and where this part ends
    int b, nth;

    __device__ __forceinline__ void look(const WeighArgs &a, int first) {
        const int lane = threadIdx.x & 63;
        block = first, groups = sinks = skip = cost = 0;
        if (first + lane < a.at.batch) {
            const WeighSequence v = weigh_sequence<false>(a, first + lane);
            if (v.count > 0) {
                const WeighView w = weigh_view(a, v.first_position, v.first_position + v.count - 1, v.end);
                groups = (w.tiles + N - 1) / N, sinks = w.sink_tiles / N, skip = w.first_tile / N - sinks;
                long long rows = (long long)v.count * a.group;
                if (a.window) rows = min(rows, ((long long)a.window + 16 * N) * a.group);
                cost = (int)((rows + ROWS - 1) / ROWS) + 2;
            }
        }
        const Cost mine = (Cost)groups * (Cost)cost;
        Cost upto = mine;
#pragma unroll
        for (int off = 1; off < 64; off *= 2) {
            const Cost other = __shfl_up(upto, off, 64);
            if (lane >= off) upto += other;
        }
        before = base + upto - mine;
        base += of_lane(upto, 63);
    }
    static __device__ __forceinline__ Cost of_lane(Cost x, int lane) {
        return (Cost)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
    }
    // part `part` of `parts`
    __device__ __forceinline__ void cut(const WeighArgs &a, int part, int parts) {
        base = 0;
        for (int first = 0; first < a.at.batch; first += 64) look(a, first);
        const Cost each = base / (uint32_t)parts, rest = base - each * (uint32_t)parts;
        at = each * (uint32_t)part + min((Cost)part, rest), end = at + each + ((Cost)part < rest ? 1 : 0);
        if (a.at.batch > 64) base = 0, look(a, 0);
        b = -1, nth = 0;
        if (at >= end) return;
        // the first group that begins at or behind `at`
        while (true) {
            const unsigned long long in = __ballot(at < before + (Cost)groups * (Cost)cost);
            if (in) {
                const int lane = __builtin_ctzll(in);
                const Cost first = of_lane(before, lane);
                const uint32_t price = (uint32_t)__builtin_amdgcn_readlane(cost, lane);
                b = block + lane, nth = at > first ? (int)((at - first + price - 1) / price) : 0;
                at = first + (Cost)nth * price;
                return;
            }
            // (at is in front of all groups' end, unless lengths have changed in between)
            if (block + 64 >= a.at.batch) return;
            look(a, block + 64);
        }
    }
    __device__ __forceinline__ bool next(const WeighArgs &a, WeighGroup &g) {
        if (b < 0 || at >= end) return false;
        while (nth >= __builtin_amdgcn_readlane(groups, b - block)) {
            nth = 0, ++b;
            if (b >= a.at.batch) return false;
            if (b - block >= 64) look(a, block + 64);
        }
        const int lane = b - block;
        g.b = b, g.v = weigh_sequence<true>(a, b);
        g.first = (nth + (nth < __builtin_amdgcn_readlane(sinks, lane) ? 0 : __builtin_amdgcn_readlane(skip, lane))) * 16 * N;
        ++nth, at += (uint32_t)__builtin_amdgcn_readlane(cost, lane);
        return true;
    }
};

// Tokens and the rows that see them, sixteen at a time: a wave keeps 16 N tokens' keys and goes through all rows, or (SHARED) the waves of
// a workgroup have the same tokens and take rows in turn.  Then the next tokens, whose keys and first rows are on their way by then: one round of waves has
// all tokens, a round for each four tokens' tiles took 179 us where this takes 118 (the last 100 tokens of six prompts of up to 9000, 8 heads of 128, groups of 4, bf16).
//
// Bound by having few waves, two a SIMD at most and 1.3 on average, as four tiles' expanded keys alone are 64 registers: 32 us for the four prompts above, with vector
// instructions (an exponential, a multiplication, two fused ones and a difference for each score and lane) in 37 % of all cycles, matrix ones in 8 %.  What waves wait for shows: rows' 16 bytes a lane touch sixteen lines an instruction where four lanes side by side load a
// row, else 64 (36 us, 129 for the six prompts), and products of all tiles go first (35, 122).  Tried: 32 tokens a wave and four waves a SIMD, 57 us.
template <bool BF16, int STEPS, bool SHARED>
__global__ __launch_bounds__(kWeighThreads, BF16 && STEPS == 2 ? 3 : 2) void weigh_tokens_kernel(const WeighArgs a) {
    constexpr int N = STEPS == 8 ? 2 : 4;           // tiles of sixteen tokens of a wave
    __shared__ float s_sum[2][SHARED ? kWeighWaves : 1][16 * N];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quarter = lane >> 4;
    const int head = blockIdx.x;
    constexpr int kStep = SHARED ? 16 * kWeighWaves : 16;
    constexpr bool kAhead = BF16 || STEPS < 8;         // (or registers are too few)
    int buffer = 0;
    WeighGroups<N, kStep> groups;
    if (SHARED) groups.cut(a, (int)blockIdx.y, (int)gridDim.y);
    else groups.cut(a, (int)blockIdx.y * kWeighWaves + wave, (int)gridDim.y * kWeighWaves);
    WeighGroup g;
    if (!groups.next(a, g)) return;
    WeighKeys<STEPS, N> keys;
    WeighRows<BF16, STEPS, BF16> q;            // (fp32: a prompt of 2000 tokens, 8 heads, groups of 4 202 us, side by side 213)
    qt_u32x4 next[2];
    const auto fetch_rows = [&](const WeighSequence &v, int at) {
        q.fetch(a, v, head, at);
        // (behind the last row: what lies there, or room that is kept free)
        const Unaligned16of4 *p = (const Unaligned16of4 *)(a.statistics + row_entry(a, v, head, at + 4 * quarter));
        next[0] = p[0].v, next[1] = p[1].v;
    };
    // rows that see any of the tokens: those at or behind the first, and with a window not too far behind the last
    int first_row, to;
    const auto range = [&](const WeighGroup &g) {
        const long long from = max(0LL, ((long long)g.first - g.v.first_position) * a.group);
        long long end = (long long)g.v.count * a.group;
        if (a.window && g.first >= a.sinks) end = min(end, ((long long)g.first + 16 * N - 1 + a.window - g.v.first_position) * a.group);
        first_row = from < end ? ((int)from & ~15) + (SHARED ? 16 * wave : 0) : 0, to = from < end ? (int)end : 0;
        if (SHARED && a.row_parts > 1 && to) {
            const int begin = (int)from & ~15, each = ((to - begin + kStep - 1) / kStep + a.row_parts - 1) / a.row_parts * kStep;
            first_row = (int)min((long long)to, begin + (long long)blockIdx.z * each) + 16 * wave, to = (int)min((long long)to, begin + (long long)(blockIdx.z + 1) * each);
        }
    };
    keys.fetch(a, g.b, head, g.first >> 4, g.v.end);
    range(g);
    if (first_row < to) fetch_rows(g.v, first_row);
    while (true) {
        const int rows = g.v.count * a.group, first = g.first;
        keys.arrange(a.factor);
        bf16x8 numbers[BF16 ? N : 1][STEPS];            // (fp32 queries take the registers: expanded again for every sixteen rows)
        bool all_there = first + 16 * N <= g.v.end, there[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if constexpr (BF16) {
#pragma unroll
                for (int j = 0; j < STEPS; ++j) numbers[n][j] = fp4_to_bf16(keys.word[n][j]);
            }
            all_there = all_there && keys.there[n], there[n] = keys.there[n];
        }
        const int mine = N == 4 ? quarter : quarter >> 1, t = 16 * mine + (lane & 15);
        bool writes = first + t < g.v.end && (N == 4 || (quarter & 1) == 0);
#pragma unroll
        for (int n = 0; n < N; ++n) writes = writes && (mine != n || there[n]);
        float *total = a.totals + g.b * a.total_sequence + head * a.total_head + first + t;
        const bool parted = SHARED && a.row_parts > 1;
        const float held = writes && !parted && (!SHARED || wave == 0) ? *total : 0.0f;
        WeighGroup after;
        const bool more = groups.next(a, after);
        if (kAhead && more) keys.fetch(a, after.b, head, after.first >> 4, after.v.end);
        float sum[N];
#pragma unroll
        for (int n = 0; n < N; ++n) sum[n] = 0.0f;
        const int end = to;
        int row_at = first_row;
        if (more) range(after);
        writes = writes && end > 0;
        if (kAhead && row_at >= end && more && first_row < to) fetch_rows(after.v, first_row);
        for (; row_at < end; row_at += kStep) {
            q.arrange();
            float m[4], by[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) m[i] = __uint_as_float(next[i / 2][2 * (i % 2)]), by[i] = __uint_as_float(next[i / 2][2 * (i % 2) + 1]);
            if (row_at + 16 > rows) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (row_at + 4 * quarter + i >= rows) m[i] = INFINITY, by[i] = 0.0f;
            }
            if (row_at + kStep < end) fetch_rows(g.v, row_at + kStep);
            else if (kAhead && more && first_row < to) fetch_rows(after.v, first_row);
            const bool all = all_there && first + 16 * N - 1 <= g.v.position(a, row_at) &&
                             (!a.window || g.v.position(a, min(rows, row_at + 16) - 1) - first < a.window || first + 16 * N <= a.sinks);
            fp4_f32x4 s[N];
            if constexpr (BF16) {
                // (all tiles' products first)
                fp4_f32x4 part[STEPS / 2][N];
#pragma unroll
                for (int j = 0; j < STEPS; ++j)
#pragma unroll
                    for (int n = 0; n < N; ++n) part[j / 2][n] = multiply_pieces<1>(q.x[j], numbers[n][j], j & 1 ? part[j / 2][n] : (fp4_f32x4){0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int n = 0; n < N; ++n) s[n] = scale_scores<STEPS>(part, n, keys.scale[n]);
            } else {
#pragma unroll
                for (int n = 0; n < N; ++n) {
#pragma unroll
                    for (int j = 0; j < STEPS; ++j) {
                        uint32_t word = keys.word[n][j];
                        asm volatile("" : "+v"(word));          // (not in front of the loop)
                        numbers[0][j] = fp4_to_bf16(word);
                    }
                    s[n] = weigh_scores(q, numbers[0], keys.scale[n]);
                }
            }
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][i] -= m[i];        // (m is one of these, bit for bit: a token seen alone has weight 1)
            if (all) {
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[n] = __builtin_fmaf(__builtin_amdgcn_exp2f(s[n][i]), by[i], sum[n]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = row_at + 4 * quarter + i, position = row < rows ? g.v.position(a, row) : -1;
#pragma unroll
                    for (int n = 0; n < N; ++n) {
                        const int at = first + 16 * n + (lane & 15);
                        float weight = __builtin_amdgcn_exp2f(s[n][i]) * by[i];
                        asm volatile("" : "+v"(weight));        // (and then looked at: a branch for each takes longer)
                        sum[n] += there[n] && at < g.v.end && row_sees(a, position, at) ? weight : 0.0f;
                    }
                }
            }
        }
        const float weight = sum_of_rows<N>(sum);
        if constexpr (SHARED) {
            s_sum[buffer][wave][t] = weight;
            __syncthreads();
            if (wave == 0) {
                const float all = (s_sum[buffer][0][t] + s_sum[buffer][1][t]) + (s_sum[buffer][2][t] + s_sum[buffer][3][t]);
                if (parted) a.sums[(((long long)blockIdx.z * a.at.batch + g.b) * a.shape.kv_heads + head) * a.sums_stride + first + t] = all;
                else if (writes) *total = held + all;
            }
            buffer ^= 1;
        } else {
            if (writes) *total = held + weight;
        }
        if (!more) break;
        g = after;
        if (!kAhead) {
            keys.fetch(a, g.b, head, g.first >> 4, g.v.end);
            if (first_row < to) fetch_rows(g.v, first_row);
        }
    }
}

// Adds the sums of all row parts to the totals, in order: of the tokens whose groups the kernel above goes through.
__global__ __launch_bounds__(kWeighThreads) void weigh_add_kernel(const WeighArgs a) {
    const int head = blockIdx.y, b = blockIdx.z, token = ((int)blockIdx.x * kWeighThreads + (int)threadIdx.x) * 4;
    const WeighSequence v = weigh_sequence<true>(a, b);
    if (v.count <= 0 || token >= v.end) return;
    const WeighView view = weigh_view(a, v.first_position, v.first_position + v.count - 1, v.end);
    if (view.tiles == 0 || (token >= 16 * view.sink_tiles && token < 16 * view.first_tile)) return;
    if ((unsigned)a.at.table[b * a.at.table_stride + (token >> a.shape.page_shift)] >= (unsigned)a.shape.pages) return;
    float *total = a.totals + b * a.total_sequence + head * a.total_head + token;
    const float *from = a.sums + ((long long)b * a.shape.kv_heads + head) * a.sums_stride + token;
    const long long part = (long long)a.at.batch * a.shape.kv_heads * a.sums_stride;
    float4 all = load_f32x4<true>(from);
    for (int n = 1; n < a.row_parts; ++n) {
        const float4 more = load_f32x4<true>(from + n * part);
        all.x += more.x, all.y += more.y, all.z += more.z, all.w += more.w;
    }
    const float sum[4] = {all.x, all.y, all.z, all.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (token + e < v.end) total[e] += sum[e];
}

// Tiles of rows at most, and parts of the tokens that they see: no more than leave several to a workgroup of a round, nor than there are tokens to see.
long long weigh_row_tiles(const CachePlaces &at, int group, int rows) {
    return at.starts ? (long long)at.tokens * group / rows + at.batch : (long long)at.batch * ((group + rows - 1) / rows);
}
int weigh_parts(long long workgroups, long long seen) {
    const long long least = (seen + 16 * kLeastTiles - 1) / (16 * kLeastTiles), spread = 6LL * compute_units() / (workgroups < 1 ? 1 : workgroups) + 1;
    const long long parts = least < spread ? least : spread;
    return (int)(parts < 1 ? 1 : parts < kMostParts ? parts : kMostParts);
}

template <bool BF16, int STEPS, int T>
void launch_rows(const WeighArgs &a, const dim3 &work, hipStream_t stream) {
    hipLaunchKernelGGL((weigh_rows_kernel<BF16, STEPS, T, false>), work, dim3(kWeighThreads), 0, stream, a);
}
template <bool BF16, int STEPS>
void launch_weigh(WeighArgs a, bool few, hipStream_t stream) {
    constexpr int N = STEPS == 8 ? 2 : 4, T = BF16 ? 2 : 1;
    const int rows = few ? 16 : 16 * T;
    const long long row_tiles = weigh_row_tiles(a.at, a.group, rows);
    const long long room = (long long)a.at.table_pages << a.shape.page_shift, covered = room < kMostTokens ? room : kMostTokens, seen = a.window ? (long long)a.window + a.sinks + 80 : covered;
    // Parts of rows as make one round of the workgroups that the units hold, or, where tiles of rows are so many that this would leave few, three quarters of it:
    // 16 sequences of up to 7600 tokens and 8 heads 21.4 us of 896, 24.1 of 1536; 64 of up to 7975 74.1 us of 512, 63.7 of 768; parts that go to workgroups in order of
    // their own, for lack of one of these, began in a second round at 20 us where the first took 25.
    const long long held = (BF16 ? (few ? 4 : 3) - (STEPS == 8) : STEPS == 8 ? 2 : 3) * compute_units(), tiles = row_tiles * a.shape.kv_heads;
    a.wanted = held - tiles > 3 * held / 4 ? held - tiles : 3 * held / 4;
    a.parts = weigh_parts(row_tiles * a.shape.kv_heads, covered < seen ? covered : seen);
    a.by_tiles = make_fastdiv((uint32_t)((a.group + rows - 1) / rows));
    // (parts of equal size, and one more for each tile of rows that they do not divide)
    const long long pieces = a.parts == 1 ? row_tiles : min(row_tiles * a.parts, row_tiles + a.wanted / a.shape.kv_heads + 1), most = 32768;
    const dim3 work(a.shape.kv_heads, (unsigned)min(pieces, most), (unsigned)((pieces + most - 1) / most));
    if (few) {
        a.statistics = nullptr;
        launch_rows<BF16, STEPS, 1>(a, work, stream);
        if (a.scores) {
            const dim3 grid((unsigned)((covered + 4 * kWeighThreads - 1) / (4 * kWeighThreads)), a.shape.kv_heads, a.at.batch);
            hipLaunchKernelGGL(weigh_scores_kernel<BF16>, grid, dim3(kWeighThreads), 0, stream, a);
        } else
            hipLaunchKernelGGL((weigh_rows_kernel<BF16, STEPS, 1, true>), work, dim3(kWeighThreads), 0, stream, a);
        return;
    }
    launch_rows<BF16, STEPS, T>(a, work, stream);
    const long long entries = (long long)a.at.tokens * a.group * a.shape.kv_heads;
    if (a.parts > 1) hipLaunchKernelGGL(weigh_join_kernel, dim3((unsigned)((16 * entries + kWeighThreads - 1) / kWeighThreads)), dim3(kWeighThreads), 0, stream, a, entries);
    // a round of workgroups, or fewer where there are not as many tokens; of waves with tokens of their own if every one has some then
    const long long round = (BF16 && STEPS == 2 ? 3 : 2) * compute_units(), blocks = (covered + 16 * N - 1) / (16 * N) * a.at.batch;
    const long long heads = a.shape.kv_heads, each = round / heads < 1 ? 1 : round / heads;
    const dim3 grid((unsigned)heads, (unsigned)min(min(blocks, each), 65535LL));
    if (a.row_parts > 1) {
        hipLaunchKernelGGL((weigh_tokens_kernel<BF16, STEPS, true>), dim3(grid.x, grid.y, (unsigned)a.row_parts), dim3(kWeighThreads), 0, stream, a);
        hipLaunchKernelGGL(weigh_add_kernel, dim3((unsigned)((covered + 4 * kWeighThreads - 1) / (4 * kWeighThreads)), a.shape.kv_heads, a.at.batch), dim3(kWeighThreads), 0, stream, a);
    } else if (blocks >= kWeighWaves * each) hipLaunchKernelGGL((weigh_tokens_kernel<BF16, STEPS, false>), grid, dim3(kWeighThreads), 0, stream, a);
    else hipLaunchKernelGGL((weigh_tokens_kernel<BF16, STEPS, true>), grid, dim3(kWeighThreads), 0, stream, a);
}

template <bool BF16>
void launch_weigh_type(const WeighArgs &a, bool few, hipStream_t stream) {
    if (a.shape.head_dim <= 64) launch_weigh<BF16, 2>(a, few, stream);
    else if (a.shape.head_dim <= 128) launch_weigh<BF16, 4>(a, few, stream);
    else launch_weigh<BF16, 8>(a, few, stream);
}

// Scores of a token of each sequence are kept, if they take up to 512 MB, instead of being worked out twice: 32 sequences of 100 to 8000 tokens 47 us
// without and 38 with them.
constexpr long long kMostScores = 1LL << 29;
struct WeighSizes { long long partial, scores, stride, all; int parts, row_parts; bool few; };
// Parts of the rows that see a token, where the tokens alone do not make two workgroups for each unit, of at least 256 rows on average.  A prompt of 1487 tokens, 3
// heads of 128, groups of 8, a window of 349, bf16: 47.7 us, whole 72; of 3950, one head, groups of 5 79 and 223; of 2000, 8 heads, groups of 4 103 and 128; three of 371, 2
// heads, groups of 4 28 and 35.
int weigh_row_parts(const CacheShape &shape, const CachePlaces &at, int group, long long room) {
    const int tokens = shape.head_dim > 128 ? 32 : 64;
    const long long groups = (room + tokens - 1) / tokens * at.batch * shape.kv_heads, rows = (long long)at.tokens * group / at.batch;
    const long long parts = min(2LL * compute_units() / groups, rows / 256);
    return (int)(parts < 2 ? 1 : parts < 16 ? parts : 16);
}
WeighSizes weigh_sizes(const CacheShape &shape, const CachePlaces &at, int heads) {
    WeighSizes s;
    s.few = !at.starts && heads / shape.kv_heads <= 16;         // a tile of rows for every sequence
    // (the tiles of bf16 queries, of which there are fewest, and without a window)
    s.parts = weigh_parts(weigh_row_tiles(at, heads / shape.kv_heads, 32) * shape.kv_heads, (long long)at.table_pages << shape.page_shift);
    s.partial = (((long long)at.tokens * heads * (s.parts + 1) + 16) * (long long)sizeof(float2) + 255) & ~255LL;      // (and room behind the statistics)
    s.stride = (((long long)at.table_pages << shape.page_shift) + 63) & ~63LL;
    s.scores = s.few && s.stride <= kMostScores / 4 / heads / at.batch ? s.stride * heads * at.batch * 4 : 0;
    s.row_parts = s.few ? 1 : weigh_row_parts(shape, at, heads / shape.kv_heads, (long long)at.table_pages << shape.page_shift);
    if (s.row_parts > 1) s.scores = (long long)s.row_parts * at.batch * shape.kv_heads * s.stride * 4;          // (of parts of rows in their place)
    s.all = s.partial + s.scores;
    s.all = s.all < 16 ? 16 : s.all;
    return s;
}

}  // namespace
}  // namespace qt

extern "C" long long qtensor_hip_cache_weigh_workspace(const qtensor_cache *cache, const qtensor_cache_places *places, int heads) {
    using namespace qt;
    clear_error();
    CacheShape shape;
    CachePlaces at;
    if (!cache_shape("cache_weigh", cache, shape) || !cache_places("cache_weigh", places, at)) return 0;
    if (heads < 1 || heads % shape.kv_heads) { set_error(kBadArgument, "cache_weigh: %d query heads are not a multiple of the cache's %d", heads, shape.kv_heads); return 0; }
    return weigh_sizes(shape, at, heads).all;
}

extern "C" void qtensor_hip_cache_weigh(const qtensor_cache *cache, const qtensor_cache_places *places, const qtensor_cache_vectors *q, int heads, float scale,
                                        int window, int sinks, float *totals, long long total_sequence, long long total_head, void *workspace,
                                        long long workspace_bytes, void *stream) {
    using namespace qt;
    const char *what = "cache_weigh";
    clear_error();
    WeighArgs a;
    if (!cache_shape(what, cache, a.shape) || !cache_places(what, places, a.at)) return;
    if (!q || !totals || !workspace || (a.at.tokens > 0 && !q->base)) { set_error(kNullPointer, "%s: null pointer", what); return; }
    const bool bf16 = q->is_bf16 != 0;
    if (heads < 1 || heads > 32767 || heads % a.shape.kv_heads || window < 0 || sinks < 0 || (sinks && !window) || !(scale - scale == 0.0f) || total_sequence < 0 || total_head < 0 ||
        !is_aligned(q->base, bf16 ? 2 : 4) || !is_aligned(totals, 4) || !is_aligned(workspace, 16)) {
        set_error(kBadArgument, "%s: needs query heads that are a multiple of the cache's, a finite scale, sinks only beside a window and aligned tensors", what);
        return;
    }
    const WeighSizes size = weigh_sizes(a.shape, a.at, heads);
    if (workspace_bytes < size.all) { set_error(kBadArgument, "%s: needs %lld bytes of workspace, got %lld", what, size.all, workspace_bytes); return; }
    if (a.at.tokens == 0) return;
    a.codes = cache->codes[0], a.scales = cache->scales[0];
    a.scale_page = (long long)a.shape.kv_heads << a.shape.page_shift, a.code_page = a.scale_page * a.shape.row_bytes, a.scale_page *= a.shape.segments;
    a.q = q->base, a.q_token = q->token_stride, a.q_head = q->head_stride;
    a.group = heads / a.shape.kv_heads;
    a.factor = scale * 1.4426950408889634f;
    a.window = window, a.sinks = sinks;
    a.totals = totals, a.total_sequence = total_sequence, a.total_head = total_head;
    a.partial = (float2 *)workspace;
    a.statistics = a.partial + (long long)a.at.tokens * heads * size.parts;
    float *behind = size.scores ? (float *)((uint8_t *)workspace + size.partial) : nullptr;
    a.scores = size.few ? behind : nullptr, a.score_stride = size.stride;
    a.sums = behind, a.sums_stride = size.stride, a.row_parts = size.row_parts;
    a.by_group = make_fastdiv((uint32_t)a.group);
    if ((long long)a.at.tokens * a.group >= 1 << 27 || a.group >= 1 << 15 || a.at.batch > 65535 || a.shape.kv_heads > 65535) {
        set_error(kBadArgument, "%s: too many tokens, heads or sequences (%d, %d, %d)", what, a.at.tokens, heads, a.at.batch);
        return;
    }
    if (bf16) launch_weigh_type<true>(a, size.few, (hipStream_t)stream);
    else launch_weigh_type<false>(a, size.few, (hipStream_t)stream);
    launch_ok(what);
}
