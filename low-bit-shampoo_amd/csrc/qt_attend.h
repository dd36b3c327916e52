// What the attention kernels over a 4-bit cache (layout: qt_cache.h) share: arguments, which tokens a sequence's queries see,
// and the split of fp32 numbers into 6-bit ones, which the matrix instructions multiply with the cache's 4-bit numbers.
#pragma once

#include "qt_cache.h"

namespace qt {

struct AttendArgs {
    CacheShape shape;
    CachePlaces at;
    const uint8_t *codes[2];
    const float *scales[2];
    const void *q;
    void *out;
    long long q_token, q_head, out_token, out_head;
    int group;              // query heads that share one of the cache
    int q_in_eights;        // not 0: eight elements of a query from a multiple of eight on are there together, and aligned to 16 bytes
    float factor;           // scale * log2 e
    int window, sinks;      // window 0: no window
    int few_rows;           // sequences with up to so many queries (times heads that share one of the cache) go to the kernel for few, others to
                            // the one for many
    int slots;              // workgroups that the kernel's work is cut for
    int least;              // tiles below which a piece is not worth having
    float *partial;         // attend_places(slots) pieces of (rows x (DP + 2)) floats
};

// Pieces of rows of tiles that were cut, at most (see find_work).
constexpr int attend_places(int slots) { return 2 * slots; }

constexpr int attend_dim(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

constexpr int kRowsOfMany = 128;    // queries that a workgroup of the kernel for many takes
int attend_many_slots(int dim);
// Launches the kernel for sequences of many queries (and what joins its pieces): `rows_of_tiles` at most.
void launch_attend_many(AttendArgs a, unsigned rows_of_tiles, bool may_cut, hipStream_t stream);

#if defined(__HIPCC__)
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x32 __attribute__((ext_vector_type(32)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x6 __attribute__((ext_vector_type(6)));

#define QT_LDS __attribute__((address_space(3)))
#define QT_GLOBAL __attribute__((address_space(1)))
#define QT_CONSTANT __attribute__((address_space(4)))

constexpr int kFp4 = 4, kFp6 = 2;               // operand formats of the scaled matrix instructions
constexpr int kOne = 0x7f7f7f7f;                // scale bytes that stand for 2^0

// 32 numbers as 6-bit floating ones (two bits of exponent, three of mantissa, at most 7.5) times the scale's power of two, in the
// order x[0], y[0], x[1], y[1] ...; these instructions write their result while they still read, which the compiler does not know: all
// operands are kept alive behind them, so that none shares a register with the result.
__device__ __forceinline__ u32x6 to_fp6(const f32x16 &x, const f32x16 &y, float scale) {
    u32x6 out = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(x, y, scale);
    asm volatile("" : "+v"(out) : "v"(x), "v"(y), "v"(scale));
    return out;
}
__device__ __forceinline__ f32x32 from_fp6(const u32x6 &piece, float scale) {
    f32x32 out = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(piece, scale);
    asm volatile("" : "+v"(out) : "v"(piece), "v"(scale));
    return out;
}

// 32 numbers as a sum of N pieces of 6 bits.  The first piece's scale puts the largest number in [2, 4), where pieces are 1/4 apart;
// every further piece takes what is left at 2^-5 of the scale before: a rest is at most 4 in units of its scale.  What N pieces
// leave is below 2^-(4 + 5 (N - 1)) of the largest number: 2^-14 for three, 2^-24 for five.  `top`: bits of the largest
// magnitude.  scale[i]: the matrix instruction's byte for piece i; 255, its NaN, where the numbers are not finite.
template <int N>
__device__ __forceinline__ void split_fp6(f32x16 x, f32x16 y, uint32_t top, u32x6 *piece, int *scale) {
    const int exponent = (int)((top >> 23) & 0xff);
    const int first = max(exponent - 1, 5 * N);     // (numbers below 2^-100: in steps of the least scale)
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float by = __uint_as_float((uint32_t)(first - 5 * i) << 23);
        piece[i] = to_fp6(x, y, by);
        scale[i] = exponent == 255 ? 255 : first - 5 * i;
        if (i + 1 < N) {
            const f32x32 back = from_fp6(piece[i], by);
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] -= back[2 * e], y[e] -= back[2 * e + 1];
        }
    }
}

__device__ __forceinline__ i32x8 as_operand(const u32x6 &p) {
    return (i32x8){(int)p[0], (int)p[1], (int)p[2], (int)p[3], (int)p[4], (int)p[5], 0, 0};
}
__device__ __forceinline__ i32x8 as_operand(const i32x4 &p) { return (i32x8){p[0], p[1], p[2], p[3], 0, 0, 0, 0}; }

// The tokens that the new ones of a sequence see: all of it up to them, or with a window its first `sinks` and the window of the
// first of them, in tiles of 2^SHIFT: `sink_tiles` from token 0, then those from `first_tile` on.
struct SequenceView {
    int start, count;                   // its rows of the call
    int first_position, end;            // position of the first; tokens of the sequence that its table can hold
    int sink_tiles, first_tile, tiles;
};

// Tiles of what queries from `first` on see of the tokens before `end`.
template <int SHIFT>
__device__ __forceinline__ void view_tokens(const AttendArgs &a, SequenceView &v, int first, int end) {
    constexpr int kRound = (1 << SHIFT) - 1;
    int low = 0;
    if (a.window) low = min(end, max(0, max(first, 0) - (a.window - 1)));
    v.first_tile = low >> SHIFT;
    v.sink_tiles = min((int)(((long long)min(a.sinks, low) + kRound) >> SHIFT), v.first_tile);
    v.tiles = v.sink_tiles + ((end + kRound) >> SHIFT) - v.first_tile;
}

template <int SHIFT>
__device__ __forceinline__ SequenceView view_sequence(const AttendArgs &a, int b) {
    SequenceView v;
    const int length = a.at.lengths[b];
    v.start = a.at.starts ? a.at.starts[b] : b;
    v.count = a.at.starts ? a.at.starts[b + 1] - v.start : 1;
    if (v.start < 0 || v.count < 0 || (long long)v.start + v.count > a.at.tokens) v.count = 0;      // (not a list of starts: nothing)
    v.first_position = length - v.count;
    const long long covered = (long long)a.at.table_pages << a.shape.page_shift;
    v.end = (int)min((long long)max(length, 0), min(covered, 0x7fffff00LL));
    view_tokens<SHIFT>(a, v, v.first_position, v.end);
    return v;
}
struct AttendWork {
    int b, head, row_tile, piece, pieces, slot;      // slot: first partial result of this row of tiles
    int per_piece;                                   // tiles of one piece
};

// Sum over the lanes up to this one (64 lanes), additions inside rows of sixteen and of their last lanes without LDS.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_or_zero(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
    x += dpp_or_zero<0x111, 0xf>(x);        // row_shr 1, 2, 4, 8
    x += dpp_or_zero<0x112, 0xf>(x);
    x += dpp_or_zero<0x114, 0xf>(x);
    x += dpp_or_zero<0x118, 0xf>(x);
    x += dpp_or_zero<0x142, 0xa>(x);        // row_bcast 15: into rows 1 and 3
    x += dpp_or_zero<0x143, 0xc>(x);        // row_bcast 31: into rows 2 and 3
    return x;
}

// Rows of tiles of a sequence's queries; none if the sequence is the other kernel's.
template <int ROWS>
__device__ __forceinline__ int row_tiles(const AttendArgs &a, const SequenceView &v) {
    const int rows = v.count * a.group;
    return (rows > a.few_rows) == (ROWS == kRowsOfMany) ? (rows + ROWS - 1) / ROWS : 0;
}

// First row of a row of tiles: of many, the last ones first, as they see most.
template <int ROWS>
__device__ __forceinline__ int first_row_of(int rows, int row_tile) {
    return (ROWS == kRowsOfMany ? (rows + ROWS - 1) / ROWS - 1 - row_tile : row_tile) * ROWS;
}

// Pieces of a row of `tiles` tiles: of up to one and a half times `most`, as half a piece is not worth its part in the join; but where
// units would stay idle (`most` is the least), of no more than that.
__device__ __forceinline__ int pieces_of(const AttendArgs &a, int tiles, int most) { return max(1, (tiles + (most > a.least ? most / 2 : most - 1)) / most); }

// How a kernel's work is cut: a row of tiles (a sequence, a head of the cache, ROWS queries) into pieces of about as many tiles as all the work
// has per slot.  Finds the `index`th piece (BY_PIECE) or the first piece of the `index`th row of tiles; false beyond the last, where w.piece says by how
// many and w.pieces is 0.  Every wave works it out for itself, a sequence per lane.
//
// Pieces behind the first of a row are at most tiles / most, so there are no more than slots of them; and rows that are cut have fewer than 2 tiles /
// most pieces each, fewer than 2 slots in all.  `most` may round below the exact quotient by a few 2^-24 (a sum in fp32): a row whose
// partial results would lie behind the workspace's places (two per slot) is refused below, whatever the lengths say.
template <int ROWS, int SHIFT, bool BY_PIECE>
__device__ __forceinline__ bool find_work(const AttendArgs &a, uint32_t index, AttendWork &w, SequenceView &v) {
    const int lane = threadIdx.x & 63;
    const bool few = a.at.batch <= 64;          // (every lane keeps its only sequence)
    SequenceView mine = {};
    float all = 0.0f;
    for (int first = 0; first < a.at.batch; first += 64) {
        if (first + lane < a.at.batch) {
            mine = view_sequence<SHIFT>(a, first + lane);
            all += (float)(row_tiles<ROWS>(a, mine) * a.shape.kv_heads) * (float)mine.tiles;
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) all += __shfl_xor(all, off, 64);
    const int most = max(a.least, (int)min(ceilf(all / (float)a.slots), 1.0e9f));
    uint32_t before = 0, partial = 0;           // pieces or rows of tiles, and partial results, of the sequences before
    for (int first = 0; first < a.at.batch; first += 64) {
        int items = 0, pieces = 1;
        if (first + lane < a.at.batch) {
            if (!few) mine = view_sequence<SHIFT>(a, first + lane);
            items = row_tiles<ROWS>(a, mine) * a.shape.kv_heads;
            pieces = pieces_of(a, mine.tiles, most);
        }
        const uint32_t here = (uint32_t)(BY_PIECE ? items * pieces : items), parts = pieces > 1 ? (uint32_t)(items * pieces) : 0u;
        const uint32_t upto = before + wave_scan(here), parts_upto = partial + wave_scan(parts);
        const unsigned long long at = __ballot(index < upto);
        if (at) {
            const int found = __builtin_ctzll(at);
            const uint32_t from = __builtin_amdgcn_readlane(upto - here, found);
            v.start = __builtin_amdgcn_readlane(mine.start, found), v.count = __builtin_amdgcn_readlane(mine.count, found);
            v.first_position = __builtin_amdgcn_readlane(mine.first_position, found), v.end = __builtin_amdgcn_readlane(mine.end, found);
            v.sink_tiles = __builtin_amdgcn_readlane(mine.sink_tiles, found), v.first_tile = __builtin_amdgcn_readlane(mine.first_tile, found);
            v.tiles = __builtin_amdgcn_readlane(mine.tiles, found);
            w.b = first + found;
            w.pieces = __builtin_amdgcn_readlane(pieces, found);
            const int local = (int)(index - from), item = BY_PIECE ? local / w.pieces : local;
            w.row_tile = item / a.shape.kv_heads;
            w.head = item - w.row_tile * a.shape.kv_heads;
            w.piece = BY_PIECE ? local - item * w.pieces : 0;
            w.slot = (int)__builtin_amdgcn_readlane(parts_upto - parts, found) + item * w.pieces;
            w.per_piece = (v.tiles + w.pieces - 1) / w.pieces;
            return w.pieces == 1 || (w.slot >= 0 && w.slot + w.pieces <= attend_places(a.slots));
        }
        before = __builtin_amdgcn_readlane(upto, 63);
        partial = __builtin_amdgcn_readlane(parts_upto, 63);
    }
    w.piece = (int)(index - before), w.pieces = 0;
    return false;
}

// What lane LANE of the lane's row of sixteen holds: an operand of the instruction that takes it.
template <int LANE>
__device__ __forceinline__ float of_row(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x150 + LANE, 0xf, 0xf, false));
}
// 32 consecutive elements of a query from element d on, zeros behind its end: as they lie in memory, and as fp32 numbers of even and odd place.
template <bool BF16>
__device__ __forceinline__ void load_query(const AttendArgs &a, long long at, int d, bool there, uint4 *raw) {
    const int valid = there ? a.shape.head_dim - d : 0;
    constexpr int kWords = BF16 ? 4 : 8;
    const uint8_t *p = (const uint8_t *)a.q + (at + d) * (BF16 ? 2 : 4);
    if (valid >= 32 && is_aligned16(p)) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) raw[i] = ((const uint4 *)p)[i];
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
__device__ __forceinline__ void unpack_query(const uint4 *raw, f32x16 &even, f32x16 &odd) {
#pragma unroll
    for (int i = 0; i < (BF16 ? 4 : 8); ++i) {
        const uint32_t word[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        if (BF16) {
#pragma unroll
            for (int e = 0; e < 4; ++e) even[4 * i + e] = __uint_as_float(word[e] << 16), odd[4 * i + e] = __uint_as_float(word[e] & 0xffff0000u);
        } else {
            even[2 * i] = __uint_as_float(word[0]), odd[2 * i] = __uint_as_float(word[1]);
            even[2 * i + 1] = __uint_as_float(word[2]), odd[2 * i + 1] = __uint_as_float(word[3]);
        }
    }
}

template <bool BF16>
__device__ __forceinline__ void store_result(const AttendArgs &a, long long at, float y) {
    if (BF16) ((uint16_t *)a.out)[at] = float_to_bf16_bits(y);
    else ((float *)a.out)[at] = y;
}

// Order of the 16-byte chunks of row `row` of a tile's codes in LDS: chunk c stands at c ^ swap.  Sixteen rows' chunks of one place fall on all
// banks then, and of the 64 rows that a transposed read takes eight bytes each from, four share a bank, as few as 512 bytes can.
template <int DP>
__device__ __forceinline__ int swap_of(int row) {
    return DP == 64 ? (row >> 3) & 1 : DP == 128 ? (row >> 2) & 3 : (row >> 1) & 7;
}

#endif  // __HIPCC__

}  // namespace qt
