// Weights that the tokens of a 4-bit attention cache are given, summed for each head of the cache: what decides which tokens are kept.
//
// For every new token i and query head g of a cache's head h, w(i, g, t) = 2^(s(t) - m) / l over the tokens t that i sees, s = scale log2(e) q k, m the
// largest and l the sum of 2^(s - m); totals[b][h][t] += sum over i and g of w.  As t is summed over first and i afterwards, the scores are
// worked out twice: once a row (i, g) at a time for m and l, once a token at a time for the sums, instead of being kept (a score is 4
// bytes, as much as a key's 8 elements).  Every sum has one order: results do not change from call to call.
//
// Scores come from the matrix cores with all bits: keys' numbers are exact in bf16, fp32 queries go through in three pieces (qt_fp4.h).
#include "qt_cache.h"

namespace qt {
namespace {

constexpr int kWeighThreads = 256, kWeighWaves = 4;

struct WeighArgs {
    CacheShape shape;
    CachePlaces at;
    const uint8_t *codes;
    const float *scales;
    const void *q;
    long long q_token, q_head;
    int group;
    float factor;                       // scale * log2 e
    int window, sinks;                  // window 0: no window
    float *totals;
    long long total_sequence, total_head;
    float2 *partial;                    // [token][head][splits]: (m, l) of a row
    int splits;
};

// Rows (i, g) of a sequence and what they see.
struct WeighSequence {
    int start, count, first_position, end;
};
__device__ __forceinline__ WeighSequence weigh_sequence(const WeighArgs &a, int b) {
    WeighSequence v;
    const int length = a.at.lengths[b];
    v.start = a.at.starts ? a.at.starts[b] : b;
    v.count = a.at.starts ? a.at.starts[b + 1] - v.start : 1;
    if (v.start < 0 || v.count < 0 || (long long)v.start + v.count > a.at.tokens) v.count = 0;      // (not a list of starts: nothing)
    v.first_position = length - v.count;
    const long long covered = (long long)a.at.table_pages << a.shape.page_shift;
    v.end = (int)min((long long)max(length, 0), min(covered, 0x7fffff00LL));
    return v;
}

__device__ __forceinline__ bool row_sees(const WeighArgs &a, int position, int token) {
    return token <= position && (!a.window || position - token < a.window || token < a.sinks);
}

// Sixteen rows as a matrix operand: STEPS of 32 elements.
template <bool BF16, int STEPS>
struct WeighRows {
    bf16x8 x[STEPS][Eight<BF16>::kPieces];

    __device__ __forceinline__ void load(const WeighArgs &a, const WeighSequence &v, int head, int first_row, int steps) {
        const int lane = threadIdx.x & 63, row = first_row + (lane & 15), rows = v.count * a.group;
        const int i = row / a.group;
        const uint8_t *p = (const uint8_t *)a.q + ((long long)(v.start + (row < rows ? i : 0)) * a.q_token + (long long)(head * a.group + (row < rows ? row - i * a.group : 0)) * a.q_head) * (BF16 ? 2 : 4);
        Eight<BF16> raw[STEPS];
#pragma unroll
        for (int j = 0; j < STEPS; ++j) {
            raw[j].zero();
            if (j < steps) raw[j].load(p, 32 * j + 8 * (lane >> 4), row < rows ? a.shape.head_dim : 0);
        }
#pragma unroll
        for (int j = 0; j < STEPS; ++j) raw[j].pieces(x[j]);
    }
};

// Sixteen tokens' keys: numbers as they lie, and the scales of up to four segments.
template <int STEPS>
struct WeighKeys {
    uint32_t word[STEPS];
    float scale[STEPS / 2];
    bool there;

    // `tile`: of sixteen tokens of sequence b, in front of `end`
    __device__ __forceinline__ void load(const WeighArgs &a, int b, int head, int tile, int end, int steps) {
        const int lane = threadIdx.x & 63;
        const int first = tile << 4, nth = first >> a.shape.page_shift;
        int page = -1;
        if (first < end) page = a.at.table[b * a.at.table_stride + nth];
        there = (unsigned)page < (unsigned)a.shape.pages;
        const long long line = ((long long)(there ? page : 0) * a.shape.kv_heads + head) << a.shape.page_shift;
        const long long inside = (there ? first & ((1 << a.shape.page_shift) - 1) : 0) + (lane & 15);
        const uint8_t *p = a.codes + (line + inside) * a.shape.row_bytes + 4 * (lane >> 4);
#pragma unroll
        for (int j = 0; j < STEPS; ++j) word[j] = j < steps ? *(const uint32_t *)(p + 16 * j) : 0u;
        const float *s = a.scales + line * a.shape.segments + inside;
#pragma unroll
        for (int g = 0; g < STEPS / 2; ++g) scale[g] = g < a.shape.segments ? s[(long long)g << a.shape.page_shift] : 0.0f;
    }
};

// Scores of sixteen rows (4 (lane / 16) + i) and a token (lane % 16), times log2 e: `numbers` are its keys' numbers.
template <bool BF16, int STEPS>
__device__ __forceinline__ fp4_f32x4 weigh_scores(const WeighArgs &a, const WeighRows<BF16, STEPS> &rows, const bf16x8 *numbers, const float *scale) {
    constexpr int P = Eight<BF16>::kPieces;
    fp4_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    const int each = 1 << (a.shape.segment_shift - 5);          // steps of a segment
    fp4_f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
        part = multiply_pieces<P>(rows.x[j], numbers[j], part);
        if (((j + 1) & (each - 1)) == 0 || j == STEPS - 1) {
            float by = scale[0];
#pragma unroll
            for (int g = 1; g < STEPS / 2; ++g) by = (j >> (a.shape.segment_shift - 5)) == g ? scale[g] : by;
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(by, part[i], sum[i]);
            part = (fp4_f32x4){0.f, 0.f, 0.f, 0.f};
        }
    }
    return sum * a.factor;
}

// Finds the tile of sixteen rows that is the `index`th of the call: its sequence and the row that it begins with.
__device__ __forceinline__ bool find_rows(const WeighArgs &a, int index, int &b, int &first_row) {
    if (!a.at.starts) {
        const int each = (a.group + 15) >> 4;
        b = index / each, first_row = (index - b * each) << 4;
        return b < a.at.batch;
    }
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int first = 0; first < a.at.batch; first += 64) {
        int tiles = 0;
        if (first + lane < a.at.batch) {
            const WeighSequence v = weigh_sequence(a, first + lane);
            tiles = (int)(((long long)v.count * a.group + 15) >> 4);
        }
        int upto = tiles;
#pragma unroll
        for (int off = 1; off < 64; off *= 2) {
            const int other = __shfl_up(upto, off, 64);
            if (lane >= off) upto += other;
        }
        const unsigned long long at = __ballot(index < before + upto);
        if (at) {
            const int found = __builtin_ctzll(at);
            b = first + found;
            first_row = (index - before - __shfl(upto - tiles, found, 64)) << 4;
            return true;
        }
        before += __shfl(upto, 63, 64);
    }
    return false;
}

// Joins (m, l) of two parts of a row.
__device__ __forceinline__ float2 join_parts(float2 x, float2 y) {
    const float m = fmaxf(x.x, y.x), by = m == -INFINITY ? 0.0f : m;
    return make_float2(m, x.y * __builtin_amdgcn_exp2f(x.x - by) + y.y * __builtin_amdgcn_exp2f(y.x - by));
}

template <bool BF16, int STEPS>
__global__ __launch_bounds__(kWeighThreads) void weigh_rows_kernel(const WeighArgs a) {
    constexpr int kAtOnce = 4;
    __shared__ float2 s_part[kWeighWaves][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quarter = lane >> 4;
    const int head = blockIdx.y, steps = a.shape.row_bytes >> 4;
    int b, first_row;
    if (!find_rows(a, blockIdx.x, b, first_row)) return;
    const WeighSequence v = weigh_sequence(a, b);
    const int rows = v.count * a.group;
    if (first_row >= rows) return;
    WeighRows<BF16, STEPS> q;
    q.load(a, v, head, first_row, steps);
    // tiles of tokens that any of them sees
    const int nearest = v.first_position + first_row / a.group, furthest = v.first_position + min(rows - 1, first_row + 15) / a.group;
    const int high = min(furthest + 1, v.end);
    const int low = a.window ? min(max(high, 0), max(0, max(nearest, 0) - (a.window - 1))) : 0;
    const int first_tile = low >> 4, sink_tiles = min((int)(((long long)min(a.sinks, low) + 15) >> 4), first_tile);
    const int tiles = high <= 0 ? 0 : sink_tiles + ((high + 15) >> 4) - first_tile;
    const int each = (tiles + a.splits - 1) / a.splits;
    const int from = min(tiles, (int)blockIdx.z * each), to = min(tiles, from + each);
    int position[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = first_row + 4 * quarter + i;
        position[i] = row < rows ? v.first_position + row / a.group : -1;
    }
    float m[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = -INFINITY, l[i] = 0.0f;
    for (int index = from + wave * kAtOnce; index < to; index += kWeighWaves * kAtOnce) {
        WeighKeys<STEPS> keys[kAtOnce];
        int tile[kAtOnce];
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
            const int at = min(index + n, to - 1);
            tile[n] = at < sink_tiles ? at : first_tile + at - sink_tiles;
            keys[n].load(a, b, head, tile[n], v.end, steps);
        }
        fp4_f32x4 s[kAtOnce];
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
            bf16x8 numbers[STEPS];
#pragma unroll
            for (int j = 0; j < STEPS; ++j) numbers[j] = fp4_to_bf16(keys[n].word[j]);
            s[n] = weigh_scores<BF16, STEPS>(a, q, numbers, keys[n].scale);
            const int token = (tile[n] << 4) + (lane & 15);
            const bool there = keys[n].there && index + n < to && token < v.end;
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] = there && row_sees(a, position[i], token) ? s[n][i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float top = m[i];
#pragma unroll
            for (int n = 0; n < kAtOnce; ++n) top = fmaxf(top, s[n][i]);
            const float by = top == -INFINITY ? 0.0f : top;
            l[i] *= __builtin_amdgcn_exp2f(m[i] - by);
#pragma unroll
            for (int n = 0; n < kAtOnce; ++n) l[i] += __builtin_amdgcn_exp2f(s[n][i] - by);
            m[i] = top;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float2 part = make_float2(m[i], l[i]);
#pragma unroll
        for (int off = 1; off < 16; off *= 2) part = join_parts(part, make_float2(__shfl_xor(part.x, off, 64), __shfl_xor(part.y, off, 64)));
        if ((lane & 15) == 0) s_part[wave][4 * quarter + i] = part;
    }
    __syncthreads();
    const int row = first_row + (int)threadIdx.x;
    if (threadIdx.x < 16 && row < rows) {
        float2 part = s_part[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < kWeighWaves; ++w) part = join_parts(part, s_part[w][threadIdx.x]);
        const int i = row / a.group;
        a.partial[((long long)(v.start + i) * (a.shape.kv_heads * a.group) + head * a.group + (row - i * a.group)) * a.splits + blockIdx.z] = part;
    }
}

template <bool BF16, int STEPS>
__global__ __launch_bounds__(kWeighThreads) void weigh_tokens_kernel(const WeighArgs a) {
    constexpr int N = STEPS == 8 ? 2 : 4;           // tiles of sixteen tokens of a wave
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quarter = lane >> 4;
    const int head = blockIdx.y, b = blockIdx.z, steps = a.shape.row_bytes >> 4;
    const WeighSequence v = weigh_sequence(a, b);
    const int rows = v.count * a.group;
    const int first = ((int)blockIdx.x * kWeighWaves + wave) * 16 * N;
    if (first >= v.end) return;
    // rows that see any of the tokens: those at or behind the first, and with a window not too far behind the last
    const long long from = max(0LL, ((long long)first - v.first_position) * a.group);
    long long to = rows;
    if (a.window && first >= a.sinks) to = min(to, ((long long)first + 16 * N - 1 + a.window - v.first_position) * a.group);
    if (from >= to) return;
    bf16x8 numbers[N][STEPS];
    float scale[N][STEPS / 2];
    bool there[N];
    {
        WeighKeys<STEPS> keys[N];
#pragma unroll
        for (int n = 0; n < N; ++n) keys[n].load(a, b, head, (first >> 4) + n, v.end, steps);
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
            for (int j = 0; j < STEPS; ++j) numbers[n][j] = fp4_to_bf16(keys[n].word[j]);
#pragma unroll
            for (int g = 0; g < STEPS / 2; ++g) scale[n][g] = keys[n].scale[g];
            there[n] = keys[n].there && first + 16 * n + (lane & 15) < v.end;
        }
    }
    float sum[N];
#pragma unroll
    for (int n = 0; n < N; ++n) sum[n] = 0.0f;
    for (int first_row = (int)from & ~15; first_row < (int)to; first_row += 16) {
        WeighRows<BF16, STEPS> q;
        q.load(a, v, head, first_row, steps);
        // (m, 1 / l) of row lane % 16, parts of it in turn
        float2 part = make_float2(-INFINITY, 0.0f);
        {
            const int row = first_row + (lane & 15), i = row / a.group;
            if (row < rows) {
                const float2 *p = a.partial + ((long long)(v.start + i) * (a.shape.kv_heads * a.group) + head * a.group + (row - i * a.group)) * a.splits;
                for (int n = quarter; n < a.splits; n += 4) part = join_parts(part, p[n]);
            }
            part = join_parts(part, make_float2(__shfl_xor(part.x, 16, 64), __shfl_xor(part.y, 16, 64)));
            part = join_parts(part, make_float2(__shfl_xor(part.x, 32, 64), __shfl_xor(part.y, 32, 64)));
            part.x = part.x == -INFINITY ? 0.0f : part.x;
            part.y = part.y == 0.0f ? 0.0f : 1.0f / part.y;
        }
        float m[4], by[4];
        int position[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = first_row + 4 * quarter + i;
            m[i] = __shfl(part.x, 4 * quarter + i, 64), by[i] = __shfl(part.y, 4 * quarter + i, 64);
            position[i] = row < rows ? v.first_position + row / a.group : -1;
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const fp4_f32x4 s = weigh_scores<BF16, STEPS>(a, q, numbers[n], scale[n]);
            const int token = first + 16 * n + (lane & 15);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[n] += there[n] && row_sees(a, position[i], token) ? __builtin_amdgcn_exp2f(s[i] - m[i]) * by[i] : 0.0f;
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        sum[n] += __shfl_xor(sum[n], 16, 64);
        sum[n] += __shfl_xor(sum[n], 32, 64);
        const int token = first + 16 * n + (lane & 15);
        if (quarter == 0 && there[n]) a.totals[b * a.total_sequence + head * a.total_head + token] += sum[n];
    }
}

template <bool BF16, int STEPS>
void launch_weigh(const WeighArgs &a, unsigned row_tiles, hipStream_t stream) {
    constexpr int kTokens = kWeighWaves * 16 * (STEPS == 8 ? 2 : 4);
    const long long covered = (long long)a.at.table_pages << a.shape.page_shift;
    const unsigned blocks = (unsigned)((covered + kTokens - 1) / kTokens);
    hipLaunchKernelGGL((weigh_rows_kernel<BF16, STEPS>), dim3(row_tiles, a.shape.kv_heads, a.splits), dim3(kWeighThreads), 0, stream, a);
    hipLaunchKernelGGL((weigh_tokens_kernel<BF16, STEPS>), dim3(blocks, a.shape.kv_heads, a.at.batch), dim3(kWeighThreads), 0, stream, a);
}

template <bool BF16>
void launch_weigh_type(const WeighArgs &a, unsigned row_tiles, hipStream_t stream) {
    if (a.shape.head_dim <= 64) launch_weigh<BF16, 2>(a, row_tiles, stream);
    else if (a.shape.head_dim <= 128) launch_weigh<BF16, 4>(a, row_tiles, stream);
    else launch_weigh<BF16, 8>(a, row_tiles, stream);
}

// Tiles of sixteen rows at most, and parts that the tokens of each are cut into: enough workgroups for every unit, pieces of no fewer than 256 tokens.
long long weigh_row_tiles(int group, int batch, int tokens, bool starts) {
    return starts ? (long long)tokens * group / 16 + batch : (long long)batch * ((group + 15) / 16);
}
int weigh_splits(const qtensor_cache *cache, const qtensor_cache_places *at, int group) {
    const long long work = weigh_row_tiles(group, at->batch, at->tokens, at->starts != nullptr) * cache->kv_heads;
    const long long wanted = (8LL * compute_units() + work - 1) / (work < 1 ? 1 : work);
    const long long most = ((long long)at->table_pages * cache->page_size + 255) / 256;
    const long long n = wanted < most ? wanted : most;
    return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
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
    const long long size = (long long)at.tokens * heads * weigh_splits(cache, places, heads / shape.kv_heads) * (long long)sizeof(float2);
    return size < 16 ? 16 : size;
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
    const long long size = qtensor_hip_cache_weigh_workspace(cache, places, heads);
    if (workspace_bytes < size) { set_error(kBadArgument, "%s: needs %lld bytes of workspace, got %lld", what, size, workspace_bytes); return; }
    if (a.at.tokens == 0) return;
    a.codes = cache->codes[0], a.scales = cache->scales[0];
    a.q = q->base, a.q_token = q->token_stride, a.q_head = q->head_stride;
    a.group = heads / a.shape.kv_heads;
    a.factor = scale * 1.4426950408889634f;
    a.window = window, a.sinks = sinks;
    a.totals = totals, a.total_sequence = total_sequence, a.total_head = total_head;
    a.partial = (float2 *)workspace;
    a.splits = weigh_splits(cache, places, a.group);
    const long long row_tiles = weigh_row_tiles(a.group, a.at.batch, a.at.tokens, a.at.starts != nullptr);
    if ((long long)a.at.tokens * a.group > 0x7fffff00LL || a.at.batch > 65535 || a.shape.kv_heads > 65535) {
        set_error(kBadArgument, "%s: too many tokens, heads or sequences (%d, %d, %d)", what, a.at.tokens, heads, a.at.batch);
        return;
    }
    if (bf16) launch_weigh_type<true>(a, (unsigned)row_tiles, (hipStream_t)stream);
    else launch_weigh_type<false>(a, (unsigned)row_tiles, (hipStream_t)stream);
    launch_ok(what);
}
