// Rotary positions: queries and keys turned by where their tokens stand, alone (and back, for the gradients) or on the way into the
// attention cache.
//
// Pair p of a head's first `dims` elements, (x[2 p], x[2 p + 1]) or (x[p], x[p + dims / 2]), becomes (a c - b s, b c + a s) with c and s the
// fp32 numbers nearest to magnitude * cos and magnitude * sin of position * frequency[p], worked out in 64 bits: positions of a long context
// leave an fp32 angle few digits (2^-24 of 10^5 turns is 0.04 of a radian).  The products are rounded to fp32 each, then their sum, then the
// result to its type, so that what a call gives is defined bit for bit, and turning on the way into the cache is turning, then writing.
//
// Bound by memory but for the smallest calls.  A lane takes sixteen bytes of a vector, its pairs' cosines and sines stay in
// registers while it goes through the heads of its token: they are worked out once a workgroup, in LDS, for all of its heads.
#include "qt_cache.h"

namespace qt {
namespace {

constexpr int kTurnThreads = 256;
constexpr int kTurnPairs = 1024;        // of all tokens of a workgroup: half the elements that its lanes hold

struct TurnArgs {
    const double *frequencies;
    double magnitude;                   // of the sines with the sign of the direction
    double sine;
    int pairs, interleaved;
    int head_dim;
    int lanes, block_tokens, rows;      // lanes of a vector, tokens of a workgroup, heads that it takes at once
    FastDiv by_lanes, by_tokens, by_pairs;
};

// Sixteen bytes of a vector from `at` on, zeros behind `valid` elements; any alignment.
template <bool BF16>
__device__ __forceinline__ uint4 load_any(const void *row, int at, int valid) {
    constexpr int kEach = kLaneElements<BF16>;
    if (valid >= kEach) {
        qt_u32x4 v;
        if constexpr (BF16) v = ((const Unaligned16 *)((const uint16_t *)row + at))->v;
        else v = ((const Unaligned16of4 *)((const uint32_t *)row + at))->v;
        return make_uint4(v[0], v[1], v[2], v[3]);
    }
    return load_lane<BF16>((const uint8_t *)row + (long long)at * (BF16 ? 2 : 4), 0, valid);
}
template <bool BF16>
__device__ __forceinline__ float load_one(const void *row, int at) {
    return BF16 ? bf16_bits_to_float(((const uint16_t *)row)[at]) : ((const float *)row)[at];
}
template <bool BF16>
__device__ __forceinline__ void store_any(void *row, int at, int valid, const uint4 &y) {
    constexpr int kEach = kLaneElements<BF16>;
    if (valid >= kEach) {
        const qt_u32x4 v = {y.x, y.y, y.z, y.w};
        if constexpr (BF16) ((Unaligned16 *)((uint16_t *)row + at))->v = v;
        else ((Unaligned16of4 *)((uint32_t *)row + at))->v = v;
    } else {
        const uint32_t word[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            if (e >= valid) continue;
            if (BF16) ((uint16_t *)row)[at + e] = (uint16_t)(word[e / 2] >> (16 * (e & 1)));
            else ((uint32_t *)row)[at + e] = word[BF16 ? 0 : e];
        }
    }
}
template <bool BF16>
__device__ __forceinline__ uint4 pack_lane(const float *y) {
    uint32_t word[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) word[e] = BF16 ? floats_to_bf16_pair(y[2 * e], y[2 * e + 1]) : __float_as_uint(y[e]);
    return make_uint4(word[0], word[1], word[2], word[3]);
}

// How a lane's elements turn: where their partners lie, cosines, and sines with the sign of the partner's product.
enum LaneKind { kInPairs, kHalf, kMixed, kCopied };
template <bool BF16>
struct LaneTurn {
    static constexpr int kEach = kLaneElements<BF16>;
    LaneKind kind;
    int first, partner;
    float c[kEach], s[kEach];

    // `turn`: cosines and sines of the token's pairs
    __device__ __forceinline__ void set(const TurnArgs &a, const float2 *turn, int first_element) {
        first = first_element, partner = 0;
        const int dims = 2 * a.pairs;
        kind = first >= dims ? kCopied : a.interleaved ? kInPairs : (first + kEach <= a.pairs || (first >= a.pairs && first + kEach <= dims)) ? kHalf : kMixed;
        if (kind == kHalf) partner = first < a.pairs ? first + a.pairs : first - a.pairs;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int d = first + e;
            const bool low = a.interleaved ? (e & 1) == 0 : d < a.pairs;
            const float2 t = d < dims ? turn[a.interleaved ? d >> 1 : low ? d : d - a.pairs] : make_float2(1.0f, 0.0f);
            c[e] = t.x, s[e] = low ? t.y : -t.y;
        }
    }
    __device__ __forceinline__ uint4 load_partner(const void *row) const {
        return kind == kHalf ? load_any<BF16>(row, partner, kEach) : make_uint4(0, 0, 0, 0);
    }
    // what the elements (and in halves their partners) turn to; `row`: of the vector, for partners one by one
    __device__ __forceinline__ void apply(const TurnArgs &a, const uint4 &own, const uint4 &other, const void *row, float *y) const {
        float x[kEach], p[kEach];
        unpack_lane<BF16>(own, x);
        unpack_lane<BF16>(other, p);
        const int dims = 2 * a.pairs;
        if (kind == kInPairs) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) p[e] = x[e ^ 1];
        }
        if (kind == kMixed) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const int d = first + e;
                if (d < dims) p[e] = load_one<BF16>(row, d < a.pairs ? d + a.pairs : d - a.pairs);
            }
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) y[e] = first + e < dims ? x[e] * c[e] - p[e] * s[e] : x[e];
    }
};

// Cosines and sines of all pairs of the workgroup's tokens; position(n, there): of its nth token, if there is one.  AHEAD: frequencies are asked for in front of
// positions (8 x 2048 tokens turned and turned back 136.5 us, else 143.5; where places have to be found first it costs registers, prompts turned and written 129 us, else 117).
template <bool AHEAD, typename Position>
__device__ __forceinline__ void work_out_turns(const TurnArgs &a, float2 *turn, Position position) {
    for (int i = threadIdx.x; i < a.block_tokens * a.pairs; i += kTurnThreads) {
        const int nth = (int)fastdiv((uint32_t)i, a.by_pairs);
        double at, speed;
        if (AHEAD) speed = a.frequencies[i - nth * a.pairs];
        if (!position(nth, at)) continue;
        if (!AHEAD) speed = a.frequencies[i - nth * a.pairs];
        double s, c;
        sincos(at * speed, &s, &c);
        turn[i] = make_float2((float)(a.magnitude * c), (float)(a.sine * s));
    }
}

// A thread's vector among a workgroup's: heads of a token, `rows` of them at once.
struct TurnThread { int nth, row, first; };
template <bool BF16>
__device__ __forceinline__ TurnThread turn_thread(const TurnArgs &a) {
    const int vector = (int)fastdiv(threadIdx.x, a.by_lanes), row = (int)fastdiv((uint32_t)vector, a.by_tokens);
    return {vector - row * a.block_tokens, row, ((int)threadIdx.x - vector * a.lanes) * kLaneElements<BF16>};
}

struct TurnPart {
    const void *from;
    void *to;
    long long from_batch, from_token, from_head, to_batch, to_token, to_head;
    int heads;
};
struct TurnCall {
    TurnArgs turn;
    TurnPart part[2];
    int first_group;                    // workgroups in y of part 0
    const void *positions;
    long long position_batch;
    int long_positions;
    long long tokens, vectors;          // of a sequence, of all
    int heads_each;                     // heads that a thread goes through
    long long first_block;              // of the launch
};

// 8 sequences of 2048 tokens, 40 heads of 128 in bf16: 68 us, 4.9 TB/s, a copy's rate; a thread goes through four of
// them (69 us, one 133, eight 67; 2048 tokens 10.6, 18.2 and 11.4, as positions were read then).
template <bool BF16>
__global__ __launch_bounds__(kTurnThreads) void turn_kernel(const TurnCall a) {
    __shared__ float2 s_turn[kTurnPairs];
    const long long first = (a.first_block + blockIdx.x) * a.turn.block_tokens;
    work_out_turns<true>(a.turn, s_turn, [&](int nth, double &at) {
        const long long n = first + nth;
        if (n >= a.vectors) return false;
        const long long b = n / a.tokens, i = b * a.position_batch + (n - b * a.tokens);
        at = a.long_positions ? (double)((const long long *)a.positions)[i] : (double)((const int *)a.positions)[i];
        return true;
    });
    __syncthreads();
    const TurnThread t = turn_thread<BF16>(a.turn);
    const long long n = first + t.nth;
    const int valid = a.turn.head_dim - t.first;
    if (t.row >= a.turn.rows || n >= a.vectors || valid <= 0) return;
    const TurnPart &part = a.part[(int)blockIdx.y >= a.first_group];
    const int group = (int)blockIdx.y - ((int)blockIdx.y >= a.first_group ? a.first_group : 0);
    LaneTurn<BF16> lane;
    lane.set(a.turn, s_turn + t.nth * a.turn.pairs, t.first);
    const long long b = n / a.tokens, token = n - b * a.tokens;
    const uint8_t *from = (const uint8_t *)part.from + (b * part.from_batch + token * part.from_token) * (BF16 ? 2 : 4);
    uint8_t *to = (uint8_t *)part.to + (b * part.to_batch + token * part.to_token) * (BF16 ? 2 : 4);
    const int last = min(part.heads, (group + 1) * a.turn.rows * a.heads_each);
    for (int h = group * a.turn.rows * a.heads_each + t.row; h < last; h += a.turn.rows) {
        const uint8_t *row = from + h * part.from_head * (BF16 ? 2 : 4);
        const uint4 own = load_any<BF16>(row, t.first, valid), other = lane.load_partner(row);
        float y[kLaneElements<BF16>];
        lane.apply(a.turn, own, other, row, y);
        store_any<BF16>(to + h * part.to_head * (BF16 ? 2 : 4), t.first, valid, pack_lane<BF16>(y));
    }
}

// On the way into the cache: workgroups of the cache's heads, then of the queries, each with tokens and heads of its own number.
struct TurnWrite {
    TurnArgs keys, queries;
    int key_blocks, query_blocks;       // workgroups that the tokens are cut for, of each
    long long key_groups;               // all of the cache's heads
    int keys_each, queries_each;        // heads that a thread goes through
    CacheShape shape;
    CachePlaces at;
    const void *q, *vectors[2];
    void *out;
    long long q_token, q_head, out_token, out_head, token_stride[2], head_stride[2];
    int heads;
    const void *positions;              // or their places in the sequences
    int long_positions;
    uint8_t *codes[2];
    float *scales[2];
    int segment_lanes;
};

// Bound by memory, with the places' look-up, cosines and sines in front of the first loads: the more heads a workgroup goes through, the less of
// that, and tokens side by side in a head of the cache are written together.  9 prompts of up to 3500 tokens, 32 query heads, 8 of 128 in the cache, bf16:
// 102 us for 397 MB, 3.9 TB/s, 9 us of them for cosines and sines in 64 bits (against the instructions for 32); turned, then written by two calls 114
// (1 token of 32 sequences 5.8 and 9.2).  Tried: the first heads' loads in front of the places (registers: 125 us), keys' and queries' workgroups in turn (106),
// more waves (105 to 194: registers), 16 tokens of the keys (105).
template <bool BF16, bool LARGE>
__global__ __launch_bounds__(kTurnThreads, 4) void turn_write_kernel(const TurnWrite a) {
    constexpr int kEach = kLaneElements<BF16>, kAtOnce = LARGE ? 4 : 1, kHeads = LARGE ? 2 : 1;
    __shared__ float2 s_turn[kTurnPairs];
    __shared__ int s_sequence[kTurnThreads], s_place[kTurnThreads];
    const bool is_keys = (long long)blockIdx.x < a.key_groups;
    const TurnArgs &turn = is_keys ? a.keys : a.queries;
    const int index = (int)(blockIdx.x - (is_keys ? 0 : a.key_groups)), blocks = is_keys ? a.key_blocks : a.query_blocks;
    const int group = index / blocks, first = (index - group * blocks) * turn.block_tokens;
    int b = 0;
    if (a.at.starts) b = sequence_of_block(a.at, first);
    if ((int)threadIdx.x < turn.block_tokens) {
        const int token = first + (int)threadIdx.x;
        int place = -1;
        if (token < a.at.tokens) place = token_position(a.at, token, b);
        s_sequence[threadIdx.x] = b, s_place[threadIdx.x] = place;
    }
    __syncthreads();
    work_out_turns<false>(turn, s_turn, [&](int nth, double &at) {
        const int place = s_place[nth];
        if (place < 0) return false;
        at = !a.positions ? (double)place : a.long_positions ? (double)((const long long *)a.positions)[first + nth] : (double)((const int *)a.positions)[first + nth];
        return true;
    });
    __syncthreads();
    const TurnThread t = turn_thread<BF16>(turn);
    const bool mine = t.row < turn.rows && first + t.nth < a.at.tokens;
    const int token = mine ? first + t.nth : 0, valid = mine ? max(0, turn.head_dim - t.first) : 0;
    const int place = mine ? s_place[t.nth] : -1;
    LaneTurn<BF16> lane;
    lane.set(turn, s_turn + (mine ? t.nth : 0) * turn.pairs, t.first);
    if (!is_keys) {
        const uint8_t *from = (const uint8_t *)a.q + token * a.q_token * (BF16 ? 2 : 4);
        uint8_t *to = (uint8_t *)a.out + token * a.out_token * (BF16 ? 2 : 4);
        if (valid <= 0) return;
        const int last = min(a.heads, (group + 1) * turn.rows * a.queries_each);
        for (int h = group * turn.rows * a.queries_each + t.row; h < last; h += kAtOnce * turn.rows) {
            uint4 own[kAtOnce], other[kAtOnce];
            const uint8_t *row[kAtOnce];
#pragma unroll
            for (int n = 0; n < kAtOnce; ++n) {
                row[n] = from + min(h + n * turn.rows, last - 1) * a.q_head * (BF16 ? 2 : 4);
                own[n] = load_any<BF16>(row[n], t.first, valid), other[n] = lane.load_partner(row[n]);
            }
#pragma unroll
            for (int n = 0; n < kAtOnce; ++n) {
                if (h + n * turn.rows >= last) break;
                uint4 y = make_uint4(0, 0, 0, 0);
                if (place >= 0) {
                    float turned[kEach];
                    lane.apply(turn, own[n], other[n], row[n], turned);
                    y = pack_lane<BF16>(turned);
                }
                store_any<BF16>(to + (h + n * turn.rows) * a.out_head * (BF16 ? 2 : 4), t.first, valid, y);
            }
        }
        return;
    }
    // (lanes of a segment stay together: what has no place is worked out with them and not stored)
    long long line = -1, inside = 0;
    const int nth = place >> a.shape.page_shift;
    if (place >= 0 && nth < a.at.table_pages) {
        const int page = a.at.table[s_sequence[t.nth] * a.at.table_stride + nth];
        if ((unsigned)page < (unsigned)a.shape.pages) {
            line = ((long long)page * a.shape.kv_heads) << a.shape.page_shift;
            inside = place & ((1 << a.shape.page_shift) - 1);
        }
    }
    const int segment = t.first >> a.shape.segment_shift;
    for (int n = 0; n < a.keys_each; n += kHeads) {
        uint4 own[kHeads][2], other[kHeads];
        const uint8_t *row[kHeads];
#pragma unroll
        for (int e = 0; e < kHeads; ++e) {
            const int h = min((group * a.keys_each + n + e) * turn.rows + t.row, a.shape.kv_heads - 1);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint8_t *p = (const uint8_t *)a.vectors[i] + (token * a.token_stride[i] + h * a.head_stride[i]) * (BF16 ? 2 : 4);
                own[e][i] = load_any<BF16>(p, t.first, valid);
                if (i == 0) row[e] = p, other[e] = valid > 0 ? lane.load_partner(p) : make_uint4(0, 0, 0, 0);
            }
        }
#pragma unroll
        for (int e = 0; e < kHeads; ++e) {
            if (n + e >= a.keys_each) break;
            const int h = (group * a.keys_each + n + e) * turn.rows + t.row;
            const bool there = line >= 0 && h < a.shape.kv_heads && valid > 0;
            const long long head_line = line + ((long long)h << a.shape.page_shift);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float x[kEach];
                if (i == 0 && valid > 0) {
                    float turned[kEach];
                    lane.apply(turn, own[e][0], other[e], row[e], turned);
                    unpack_lane<BF16>(pack_lane<BF16>(turned), x);
#pragma unroll
                    for (int k = 0; k < kEach; ++k) x[k] = k < valid ? x[k] : 0.0f;
                } else {
                    unpack_lane<BF16>(own[e][i], x);
                }
                uint32_t top = 0;
#pragma unroll
                for (int k = 0; k < kEach; ++k) top = max(top, __float_as_uint(x[k]) & 0x7fffffffu);
                top = segment_max(top, a.segment_lanes);
                float scale;
                const uint32_t word = encode_fp4<kEach>(x, top, scale);
                if (there && t.first < 2 * a.shape.row_bytes) store_codes<BF16>(a.codes[i] + (head_line + inside) * a.shape.row_bytes + t.first / 2, word);
                if (there && (t.first & ((1 << a.shape.segment_shift) - 1)) == 0)
                    a.scales[i][head_line * a.shape.segments + ((long long)segment << a.shape.page_shift) + inside] = scale;
            }
        }
    }
}

bool turn_args(const char *what, const qtensor_rotary *r, int head_dim, bool bf16, int lanes, int block_tokens, TurnArgs &t) {
    if (!r || !r->frequencies) { set_error(kNullPointer, "%s: null frequencies", what); return false; }
    if (r->dims < 2 || (r->dims & 1) || r->dims > head_dim) {
        set_error(kBadArgument, "%s: needs an even number of elements to turn, 2 to the %d of a head (got %d)", what, head_dim, r->dims);
        return false;
    }
    if (!is_aligned(r->frequencies, 8)) { set_error(kBadArgument, "%s: unaligned frequencies", what); return false; }
    t.frequencies = r->frequencies, t.magnitude = r->magnitude, t.sine = r->back ? -r->magnitude : r->magnitude;
    t.pairs = r->dims / 2, t.interleaved = r->interleaved != 0, t.head_dim = head_dim;
    t.lanes = lanes, t.block_tokens = block_tokens, t.rows = kTurnThreads / (lanes * block_tokens);
    t.by_lanes = make_fastdiv((uint32_t)lanes), t.by_tokens = make_fastdiv((uint32_t)block_tokens), t.by_pairs = make_fastdiv((uint32_t)t.pairs);
    return true;
}

}  // namespace
}  // namespace qt

extern "C" void qtensor_hip_rotary_turn(const qtensor_rotary *rotary, const qtensor_rotary_call *call, void *stream) {
    using namespace qt;
    const char *what = "rotary_turn";
    clear_error();
    if (!call || call->parts < 1 || call->parts > 2) { set_error(kBadArgument, "%s: needs one or two tensors", what); return; }
    const bool bf16 = call->is_bf16 != 0;
    const int size = bf16 ? 2 : 4, head_dim = call->head_dim;
    if (head_dim < 1 || head_dim > 1024 || call->batch < 0 || call->tokens < 0 || (call->tokens > 0 && call->batch > 0x7fffffffffffLL / call->tokens)) {
        set_error(kBadArgument, "%s: needs heads of 1 to 1024 elements and sequences of tokens (got %d, %lld, %lld)", what, head_dim, call->batch, call->tokens);
        return;
    }
    const long long vectors = call->batch * call->tokens;
    const int lanes = (head_dim + (bf16 ? 7 : 3)) / (bf16 ? 8 : 4);
    const int block_tokens = kTurnThreads / lanes < 4 ? kTurnThreads / lanes : 4;
    TurnCall a = {};
    if (!turn_args(what, rotary, head_dim, bf16, lanes, block_tokens, a.turn)) return;
    if (vectors == 0) return;
    if (!call->positions || !is_aligned(call->positions, call->long_positions ? 8 : 4)) { set_error(kNullPointer, "%s: null or unaligned positions", what); return; }
    long long groups = 0;
    a.heads_each = 4;
    for (int i = 0; i < call->parts; ++i) {
        const qtensor_rotary_part &p = call->part[i];
        if (p.heads < 1 || p.heads > 32767 || !p.from || !p.to || !is_aligned(p.from, size) || !is_aligned(p.to, size)) {
            set_error(kBadArgument, "%s: needs 1 to 32767 heads and tensors aligned to an element (got %d)", what, p.heads);
            return;
        }
        a.part[i] = {p.from, p.to, p.from_batch, p.from_token, p.from_head, p.to_batch, p.to_token, p.to_head, p.heads};
        if (i == 1) a.first_group = (int)groups;
        groups += (p.heads + a.turn.rows * a.heads_each - 1) / (a.turn.rows * a.heads_each);
    }
    if (call->parts == 1) a.first_group = (int)groups;
    a.positions = call->positions, a.position_batch = call->position_batch, a.long_positions = call->long_positions != 0;
    a.tokens = call->tokens, a.vectors = vectors;
    const long long blocks = (vectors + block_tokens - 1) / block_tokens;
    const long long most = kMostThreads / kTurnThreads - 1;
    for (; a.first_block < blocks; a.first_block += most) {
        const dim3 grid((unsigned)(blocks - a.first_block < most ? blocks - a.first_block : most), (unsigned)groups);
        if (bf16) hipLaunchKernelGGL(turn_kernel<true>, grid, dim3(kTurnThreads), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL(turn_kernel<false>, grid, dim3(kTurnThreads), 0, (hipStream_t)stream, a);
        if (!launch_ok(what)) return;
    }
}

extern "C" void qtensor_hip_cache_write_turned(const qtensor_cache *cache, const qtensor_cache_places *places, const qtensor_rotary *rotary,
                                               const qtensor_cache_vectors *q, const qtensor_cache_vectors *out, int heads, const qtensor_cache_vectors *keys,
                                               const qtensor_cache_vectors *values, const void *positions, int long_positions, void *stream) {
    using namespace qt;
    const char *what = "cache_write_turned";
    clear_error();
    TurnWrite a = {};
    if (!cache_shape(what, cache, a.shape) || !cache_places(what, places, a.at)) return;
    if (!q || !out || !keys || !values || (a.at.tokens > 0 && (!q->base || !out->base || !keys->base || !values->base))) { set_error(kNullPointer, "%s: null vectors", what); return; }
    const bool bf16 = q->is_bf16 != 0;
    const qtensor_cache_vectors *all[4] = {q, out, keys, values};
    for (const qtensor_cache_vectors *v : all)
        if ((v->is_bf16 != 0) != bf16 || !is_aligned(v->base, bf16 ? 2 : 4)) { set_error(kBadArgument, "%s: queries, keys and values of one type, aligned to an element", what); return; }
    if (heads < 1 || heads > 32767) { set_error(kBadArgument, "%s: needs 1 to 32767 heads (got %d)", what, heads); return; }
    if (positions && !is_aligned(positions, long_positions ? 8 : 4)) { set_error(kBadArgument, "%s: unaligned positions", what); return; }
    a.segment_lanes = cache_segment_lanes(a.shape, bf16);
    const int lanes = a.segment_lanes * a.shape.segments;
    // Few tokens: as many workgroups as there are.  Many, from about a thousand: 1050 tokens of 32 heads of 128 in bf16 13.8 us against 19.1, 529 11.8
    // against 11.6, 18378 102 against 275.
    const long long elements = (long long)a.at.tokens * heads * a.shape.head_dim;
    const bool large = elements >= 1LL << 22;
    const int most = kTurnThreads / lanes, keys_tokens = large ? 8 : 4, few = most < 4 ? most : 4;
    if (!turn_args(what, rotary, a.shape.head_dim, bf16, lanes, most < keys_tokens ? most : keys_tokens, a.keys) ||
        !turn_args(what, rotary, a.shape.head_dim, bf16, lanes, few, a.queries))
        return;
    a.keys_each = large ? 4 : 1, a.queries_each = large ? 8 : 1;
    if (a.at.tokens == 0) return;
    a.q = q->base, a.out = out->base, a.q_token = q->token_stride, a.q_head = q->head_stride, a.out_token = out->token_stride, a.out_head = out->head_stride;
    const qtensor_cache_vectors *both[2] = {keys, values};
    for (int i = 0; i < 2; ++i) {
        a.vectors[i] = both[i]->base, a.token_stride[i] = both[i]->token_stride, a.head_stride[i] = both[i]->head_stride;
        a.codes[i] = cache->codes[i], a.scales[i] = cache->scales[i];
    }
    a.heads = heads, a.positions = positions, a.long_positions = long_positions != 0;
    const auto cut = [](long long n, long long by) { return (n + by - 1) / by; };
    a.key_blocks = (int)cut(a.at.tokens, a.keys.block_tokens), a.query_blocks = (int)cut(a.at.tokens, a.queries.block_tokens);
    a.key_groups = a.key_blocks * cut(a.shape.kv_heads, a.keys.rows * a.keys_each);
    const long long workgroups = a.key_groups + a.query_blocks * cut(heads, a.queries.rows * a.queries_each);
    if (workgroups >= kMostThreads / kTurnThreads) { set_error(kBadArgument, "%s: too many tokens and heads (%d, %d)", what, a.at.tokens, heads); return; }
    const dim3 grid((unsigned)workgroups);
    if (bf16 && large) hipLaunchKernelGGL((turn_write_kernel<true, true>), grid, dim3(kTurnThreads), 0, (hipStream_t)stream, a);
    else if (bf16) hipLaunchKernelGGL((turn_write_kernel<true, false>), grid, dim3(kTurnThreads), 0, (hipStream_t)stream, a);
    else if (large) hipLaunchKernelGGL((turn_write_kernel<false, true>), grid, dim3(kTurnThreads), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((turn_write_kernel<false, false>), grid, dim3(kTurnThreads), 0, (hipStream_t)stream, a);
    launch_ok(what);
}
