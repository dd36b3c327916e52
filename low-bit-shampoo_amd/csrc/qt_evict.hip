// Eviction from a 4-bit attention cache: of every sequence and head the tokens whose totals are largest stay, in their order.
//
// A token is there if its page is.  `keep` of them stay (all, where there are no more): the first `sinks` and the last `recent` places
// of the sequence, then those with the largest totals, ties to the earlier one.  The nth token that stays moves to the place of the nth
// token that is there, which is never behind it.
//
// The choice (a workgroup a sequence and head), which lists where tokens come from and go to, then the moves.
#include "qt_cache.h"

namespace qt {
namespace {

constexpr int kChooseThreads = 1024, kChooseWaves = kChooseThreads / 64;
constexpr int kMoveThreads = 512;
constexpr long long kMostTokens = 0x7fff0000;       // of a sequence: whole chunks (below), so that places do not pass 32 bits

struct EvictArgs {
    CacheShape shape;
    const int *table, *lengths;
    long long table_stride;
    int table_pages, batch;
    uint8_t *codes[2];
    float *scales[2];
    float *totals;
    long long total_sequence, total_head;
    int keep, recent, sinks;            // keep: no more than the table holds
    int *new_lengths;
    // scratch, an entry a token that stays, of [batch][kv_heads][keep]
    int *from, *to, *count;             // places; how many stay of a sequence
    uint8_t *apart[4];                  // room for what moves: codes of keys and of values, scales (with the keys' totals)
};

__device__ __forceinline__ int evict_end(const EvictArgs &a, int b) {
    const long long covered = (long long)a.table_pages << a.shape.page_shift;
    return (int)min((long long)max(a.lengths[b], 0), min(covered, kMostTokens));
}
// First row of head 0 of the page of a place; negative: there is none.
__device__ __forceinline__ long long evict_line(const EvictArgs &a, int b, int place) {
    const int page = a.table[b * a.table_stride + (place >> a.shape.page_shift)];
    return (unsigned)page < (unsigned)a.shape.pages ? ((long long)page * a.shape.kv_heads) << a.shape.page_shift : -1;
}
// Totals in order: NaN above all, zeroes alike.
__device__ __forceinline__ uint32_t total_key(float x) {
    return __builtin_isunordered(x, x) ? 0xffffffffu : float_to_key(x + 0.0f);
}

// A workgroup looks at kChunk tokens at a time, up to kEach side by side a thread, whose keys stay in LDS where they are all of the sequence.  (32 a thread: 131 us
// for 9 sequences of 58000 tokens, 16 124.)
constexpr int kEach = 16, kChunk = kEach * kChooseThreads;
constexpr int kCopies = 4;             // of the counts: waves that take one in turn wait for each other less

// Sums over the threads in front of this one, and over all, of two counts below 2^16 (in the halves of x); `s_waves`: scratch.
__device__ __forceinline__ uint32_t sum_before(uint32_t x, uint32_t *s_waves, uint32_t &all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t upto = x;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
        const uint32_t other = (uint32_t)__shfl_up((int)upto, off, 64);
        if (lane >= off) upto += other;
    }
    __syncthreads();
    if (lane == 63) s_waves[wave] = upto;
    __syncthreads();
    uint32_t before = upto - x;
    all = 0;
#pragma unroll 1
    for (int w = 0; w < kChooseWaves; ++w) {
        const uint32_t n = s_waves[w];
        before += w < wave ? n : 0;
        all += n;
    }
    return before;
}

// Bound by the latency of its steps, and of fetching its instructions, which run once: loops stay loops (16384 keys in registers, all unrolled: 27 us for the
// fewest tokens, 37 for 24 x 8 of 12000; so 13.5 and 23; with loads and LDS reads asked for together, four copies of the counts, no look at ties that all
// stay and the first digit counted with the tokens that are there, 20.2).  The least key of those that stay is found eight bits at a time, from counts in LDS;
// lanes that have the digit of the first one among them are counted together, as totals of one size are most of them.
__global__ __launch_bounds__(kChooseThreads) void evict_choose_kernel(const EvictArgs a) {
    __shared__ uint32_t s_key[kEach][kChooseThreads], s_waves[kChooseWaves];
    __shared__ int s_count[kCopies][256], s_digit, s_above, s_same, s_all[2];
    const int head = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 63;
    const int length = max(a.lengths[b], 0), end = evict_end(a, b);
    const float *totals = a.totals + b * a.total_sequence + head * a.total_head;
    const int chunks = max(1, (end + kChunk - 1) / kChunk);
    // tokens of a thread in every chunk: all kEach but where there is only one
    const int each = chunks > 1 ? kEach : ((end + kChooseThreads - 1) / kChooseThreads + 3) & ~3;
    // bits of a thread's tokens: those that are there, those that stay whatever their totals are
    uint32_t there = 0, anyhow = 0;
    const auto load = [&](int chunk) {
        const int first = chunk * kChunk + (int)threadIdx.x * each, last = max(end - 1, 0) & ~3;
        there = anyhow = 0;
        // (four places are of one page, and totals are as long as the pages: what is not looked at is read from the last places instead)
        int page[kEach / 4];
        qt_u32x4 total[kEach / 4];
#pragma unroll
        for (int i = 0; i < kEach / 4; ++i) {
            if (4 * i >= each) break;
            const int place = min(first + 4 * i, last);
            page[i] = a.table[b * a.table_stride + (place >> a.shape.page_shift)];
            total[i] = ((const Unaligned16of4 *)(totals + place))->v;
        }
#pragma unroll
        for (int i = 0; i < kEach / 4; ++i) {
            if (4 * i >= each) break;
            const bool is = (unsigned)page[i] < (unsigned)a.shape.pages;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int here = first + 4 * i + e;
                if (is && here < end) {
                    there |= 1u << (4 * i + e);
                    if (here < a.sinks || here >= length - a.recent) anyhow |= 1u << (4 * i + e);
                }
                s_key[4 * i + e][threadIdx.x] = total_key(__uint_as_float(total[i][e]));
            }
        }
    };
    int stay = 0, wanted = 0;                   // of the tokens that are there; by their totals
    // the least key of those that stay, and how many of the tokens with that key do
    uint32_t least = 0;
    bool all_ties = false;
    const int copy = (threadIdx.x >> 6) % kCopies;
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < kCopies * 256) (&s_count[0][0])[threadIdx.x] = 0;
        if (shift == 24 && threadIdx.x < 2) s_all[threadIdx.x] = 0;
        __syncthreads();
#pragma unroll 1
        for (int chunk = 0; chunk < chunks; ++chunk) {
            if (chunks > 1 || shift == 24) load(chunk);
            if (shift == 24) {
                uint32_t n = (uint32_t)__popc(there) | (uint32_t)__popc(anyhow) << 16;
#pragma unroll
                for (int off = 1; off < 64; off *= 2) n += (uint32_t)__shfl_xor((int)n, off, 64);
                if (lane < 2) atomicAdd(&s_all[lane], (int)(lane ? n >> 16 : n & 0xffff));
            }
#pragma unroll 1
            for (int first = 0; first < each; first += 4) {
                uint32_t key[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) key[i] = s_key[first + i][threadIdx.x];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool counts = ((there & ~anyhow) >> (first + i) & 1) && (shift == 24 || (key[i] >> (shift + 8)) == (least >> (shift + 8)));
                    const int digit = (key[i] >> shift) & 255;
                    const unsigned long long some = __ballot(counts);
                    if (!some) continue;
                    const int common = __builtin_amdgcn_readlane(digit, __builtin_ctzll(some));
                    const unsigned long long same = __ballot(counts && digit == common);
                    if (lane == 0) atomicAdd(&s_count[copy][common], __popcll(same));
                    if (counts && digit != common) atomicAdd(&s_count[copy][digit], 1);
                }
            }
        }
        __syncthreads();
        if (shift == 24) stay = min(s_all[0], a.keep), wanted = stay - s_all[1];
        if (threadIdx.x < 64) {
            // counts of the digits from this lane's four on
            int mine[4], above = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                mine[i] = 0;
#pragma unroll
                for (int c = 0; c < kCopies; ++c) mine[i] += s_count[c][4 * lane + i];
                above += mine[i];
            }
#pragma unroll
            for (int off = 1; off < 64; off *= 2) {
                const int other = __shfl_down(above, off, 64);
                if (lane + off < 64) above += other;
            }
            // the digit at which the wanted are reached from above (the largest if nothing is wanted)
            const unsigned long long reach = __ballot(above >= wanted);
            if (lane == 63 - __builtin_clzll(reach)) {
                int digit = 0, before = above - mine[0];
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    if (before >= wanted) digit = i + 1, before -= mine[i + 1];
                s_digit = 4 * lane + digit, s_above = before, s_same = mine[digit];
            }
        }
        __syncthreads();
        least |= (uint32_t)s_digit << shift;
        wanted -= s_above;
        // (all keys with these digits stay: the others, which are 0 here, need not be found)
        all_ties = s_same == wanted;
        if (all_ties) break;
    }
    int *from = a.from + ((long long)b * a.shape.kv_heads + head) * a.keep, *to = a.to + ((long long)b * a.shape.kv_heads + head) * a.keep;
    int there_before = 0, stay_before = 0, ties_before = 0;
#pragma unroll 1
    for (int chunk = 0; chunk < chunks; ++chunk) {
        if (chunks > 1) load(chunk);
        uint32_t tie = 0, stays = anyhow, all;
#pragma unroll 1
        for (int i = 0; i < each; ++i) {
            const uint32_t key = s_key[i][threadIdx.x], is = (there & ~anyhow) >> i & 1;
            tie |= (is & (uint32_t)(key == least)) << i, stays |= (is & (uint32_t)(key > least)) << i;
        }
        if (all_ties) {
            stays |= tie;
        } else {
            int ties = ties_before + (int)sum_before((uint32_t)__popc(tie), s_waves, all);
            ties_before += (int)all;
#pragma unroll 1
            for (; tie && ties < wanted; ++ties, tie &= tie - 1) stays |= tie & -tie;
        }
        const uint32_t before = sum_before((uint32_t)__popc(stays) | (uint32_t)__popc(there) << 16, s_waves, all);
        int nth = stay_before + (int)(before & 0xffff), slot = there_before + (int)(before >> 16);
        stay_before += (int)(all & 0xffff), there_before += (int)(all >> 16);
        const int first = chunk * kChunk + (int)threadIdx.x * each;
#pragma unroll 1
        for (; stays && nth < stay; stays &= stays - 1, ++nth) from[nth] = first + __builtin_ctz(stays);
        uint32_t places = there;
#pragma unroll 1
        for (; places && slot < stay; places &= places - 1, ++slot) {
            const int place = first + __builtin_ctz(places);
            to[slot] = place;
            if (slot == stay - 1 && head == 0) a.new_lengths[b] = place + 1;
        }
    }
    if (threadIdx.x == 0 && head == 0) {
        a.count[b] = stay;
        if (stay == 0) a.new_lengths[b] = 0;
    }
}

// The tokens that stay of a sequence and head by one workgroup in their order, kItems pieces a thread at a time: of keys' or values' codes sixteen
// bytes of a token each, of their scales (or, with the keys', totals) one number.
//
// In place: a token goes to a place that is not behind its own, so what is written is behind no token that has been read, and only the tokens
// that are read at the same time may lie there: they are all in registers before any is written.
//
// Bound by the lines that are touched: 2048 tokens of each of 24 sequences and 8 heads of 128 37 us for 113 MB, 3.1 TB/s, as a scale that stays alone costs its
// line.  2 or 8 pieces a thread and 1024 threads are no faster.
constexpr int kItems = 4;
template <typename Piece, typename Address>
__device__ __forceinline__ void move_pieces(int count, int parts, const int *from, const int *to, const Address &address) {
    const int each = kMoveThreads / parts, nth = (int)threadIdx.x / parts, part = (int)threadIdx.x - nth * parts;
    const int step = kItems * each;
    Piece *source[kItems], *target[kItems], held[kItems];
    // (null: nothing to do)
    const auto find = [&](int first) {
        int place[kItems], there[kItems];
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            const int at = min(first + k * each + nth, count - 1);
            place[k] = from[at], there[k] = to[at];
        }
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            const bool moves = nth < each && first + k * each + nth < count && place[k] != there[k];
            source[k] = address(place[k], part), target[k] = moves ? address(there[k], part) : nullptr;
        }
    };
    find(0);
    for (int first = 0; first < count; first += step) {
        Piece *now[kItems];
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            now[k] = target[k];
            if (now[k]) held[k] = *source[k];
        }
        if (first + step < count) find(first + step);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");        // (read, not only asked for)
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kItems; ++k)
            if (now[k]) *now[k] = held[k];
    }
}

__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(const EvictArgs a) {
    const int what = blockIdx.x, values = what & 1, head = blockIdx.y, b = blockIdx.z;
    const long long sequence = (long long)b * a.shape.kv_heads + head;
    const int *from = a.from + sequence * a.keep, *to = a.to + sequence * a.keep;
    const int count = a.count[b];
    if (count == 0) return;
    const auto inside = [&](int place) { return place & ((1 << a.shape.page_shift) - 1); };
    const auto line = [&](int place) { return evict_line(a, b, place) + ((long long)head << a.shape.page_shift); };
    if (what < 2) {
        uint8_t *codes = a.codes[values];
        move_pieces<qt_u32x4>(count, a.shape.row_bytes / 16, from, to,
                              [&](int place, int part) { return (qt_u32x4 *)(codes + (line(place) + inside(place)) * a.shape.row_bytes) + part; });
    } else {
        // (a token's segments, and behind the keys' its total)
        float *scales = a.scales[values], *totals = a.totals + b * a.total_sequence + head * a.total_head;
        move_pieces<float>(count, a.shape.segments + 1 - values, from, to, [&](int place, int part) {
            return part == a.shape.segments ? totals + place : scales + line(place) * a.shape.segments + ((long long)part << a.shape.page_shift) + inside(place);
        });
    }
}

// The same for few sequences and heads, through room of their own, by all units: out of the cache, then back.  8 sequences and heads, 26000 tokens of
// 128 chosen, moved and read back 155 us, in place 245; 2048 36 and 39; 32 of 2048 46 and 43, 8 of 1100 35 and 33.
constexpr int kCopyThreads = 256, kCopyItems = 4;
template <bool BACK, typename Piece, typename Address>
__device__ __forceinline__ void copy_pieces(int count, int parts, const int *from, const int *to, Piece *apart, const Address &address) {
    const int *place = BACK ? to : from;
#pragma unroll
    for (int k = 0; k < kCopyItems; ++k) {
        const long long i = ((long long)blockIdx.x * kCopyItems + k) * kCopyThreads + threadIdx.x;
        const int nth = (int)(i / parts), part = (int)(i - (long long)nth * parts);
        if (nth >= count) break;
        if (from[nth] == to[nth]) continue;
        Piece *there = address(place[nth], part);
        if (BACK) *there = apart[i];
        else apart[i] = *there;
    }
}
template <bool BACK>
__global__ __launch_bounds__(kCopyThreads) void evict_copy_kernel(const EvictArgs a) {
    const int what = blockIdx.y & 3, values = what & 1, head = blockIdx.y >> 2, b = blockIdx.z;
    const long long sequence = (long long)b * a.shape.kv_heads + head;
    const int *from = a.from + sequence * a.keep, *to = a.to + sequence * a.keep;
    const int count = a.count[b];
    const auto inside = [&](int place) { return place & ((1 << a.shape.page_shift) - 1); };
    const auto line = [&](int place) { return evict_line(a, b, place) + ((long long)head << a.shape.page_shift); };
    if (what < 2) {
        uint8_t *codes = a.codes[values];
        const int parts = a.shape.row_bytes / 16;
        copy_pieces<BACK>(count, parts, from, to, (qt_u32x4 *)a.apart[values] + sequence * a.keep * parts,
                          [&](int place, int part) { return (qt_u32x4 *)(codes + (line(place) + inside(place)) * a.shape.row_bytes) + part; });
    } else {
        float *scales = a.scales[values], *totals = a.totals + b * a.total_sequence + head * a.total_head;
        const int parts = a.shape.segments + 1 - values;
        copy_pieces<BACK>(count, parts, from, to, (float *)a.apart[2 + values] + sequence * a.keep * parts, [&](int place, int part) {
            return part == a.shape.segments ? totals + place : scales + line(place) * a.shape.segments + ((long long)part << a.shape.page_shift) + inside(place);
        });
    }
}

long long rounded(long long bytes) { return (bytes + 255) & ~255LL; }

struct EvictSizes { long long lists, count, codes, scales[2], all; };
EvictSizes evict_sizes(const CacheShape &shape, int batch, long long keep) {
    const long long kept = (long long)batch * shape.kv_heads * keep;
    EvictSizes s = {rounded(4 * kept), rounded(4LL * batch), 0, {0, 0}, 0};
    const long long workers = (long long)batch * shape.kv_heads;
    if (8 * workers < compute_units() && keep >= 1536 && keep >= 256 * workers)
        s.codes = rounded(kept * shape.row_bytes), s.scales[0] = rounded(4 * kept * (shape.segments + 1)), s.scales[1] = rounded(4 * kept * shape.segments);
    s.all = 2 * s.lists + s.count + 2 * s.codes + s.scales[0] + s.scales[1];
    return s;
}

bool evict_shape(const char *what, const qtensor_cache *cache, const qtensor_cache_places *places, long long keep, CacheShape &shape, CachePlaces &at) {
    if (!cache_shape(what, cache, shape) || !cache_places(what, places, at)) return false;
    if (keep < 1) { set_error(kBadArgument, "%s: needs at least a token to keep (got %lld)", what, keep); return false; }
    if (at.batch > 65535 || shape.kv_heads > 65535) { set_error(kBadArgument, "%s: too many sequences or heads (%d, %d)", what, at.batch, shape.kv_heads); return false; }
    return true;
}
long long evict_keep(const CacheShape &shape, const CachePlaces &at, long long keep) {
    const long long covered = (long long)at.table_pages << shape.page_shift, most = covered < kMostTokens ? covered : kMostTokens;
    return keep < most ? keep : most;
}

}  // namespace
}  // namespace qt

extern "C" long long qtensor_hip_cache_evict_workspace(const qtensor_cache *cache, const qtensor_cache_places *places, long long keep) {
    using namespace qt;
    clear_error();
    CacheShape shape;
    CachePlaces at;
    if (!evict_shape("cache_evict", cache, places, keep, shape, at)) return 0;
    return evict_sizes(shape, at.batch, evict_keep(shape, at, keep)).all;
}

extern "C" void qtensor_hip_cache_evict(const qtensor_cache *cache, const qtensor_cache_places *places, float *totals, long long total_sequence, long long total_head,
                                        long long keep, long long recent, long long sinks, int *new_lengths, void *workspace, long long workspace_bytes, void *stream) {
    using namespace qt;
    const char *what = "cache_evict";
    clear_error();
    EvictArgs a;
    CachePlaces at;
    if (!evict_shape(what, cache, places, keep, a.shape, at)) return;
    if (!totals || !new_lengths || !workspace) { set_error(kNullPointer, "%s: null pointer", what); return; }
    if (recent < 0 || sinks < 0 || recent > keep || sinks > keep - recent || total_sequence < 0 || total_head < 0 || !is_aligned(totals, 4) || !is_aligned(new_lengths, 4) ||
        !is_aligned(workspace, 16)) {
        set_error(kBadArgument, "%s: needs aligned tensors, and no more first and last tokens than are kept (got %lld and %lld of %lld)", what, sinks, recent, keep);
        return;
    }
    if (new_lengths == at.lengths) { set_error(kBadArgument, "%s: new lengths in the place of the lengths, which are still read", what); return; }
    const long long kept = evict_keep(a.shape, at, keep);
    const EvictSizes size = evict_sizes(a.shape, at.batch, kept);
    if (workspace_bytes < size.all) { set_error(kBadArgument, "%s: needs %lld bytes of workspace, got %lld", what, size.all, workspace_bytes); return; }
    a.table = at.table, a.lengths = at.lengths, a.table_stride = at.table_stride, a.table_pages = at.table_pages, a.batch = at.batch;
    uint8_t *p = (uint8_t *)workspace;
    a.from = (int *)p, a.to = (int *)(p + size.lists), a.count = (int *)(p + 2 * size.lists);
    p += 2 * size.lists + size.count;
    a.apart[0] = p, a.apart[1] = p + size.codes, a.apart[2] = p + 2 * size.codes, a.apart[3] = a.apart[2] + size.scales[0];
    for (int i = 0; i < 2; ++i) a.codes[i] = cache->codes[i], a.scales[i] = cache->scales[i];
    a.totals = totals, a.total_sequence = total_sequence, a.total_head = total_head;
    const long long most = 0x7fffffff;
    a.keep = (int)kept, a.recent = (int)(recent < most ? recent : most), a.sinks = (int)(sinks < most ? sinks : most);
    a.new_lengths = new_lengths;
    hipLaunchKernelGGL(evict_choose_kernel, dim3((unsigned)a.shape.kv_heads, (unsigned)a.batch), dim3(kChooseThreads), 0, (hipStream_t)stream, a);
    if (size.codes) {
        const long long pieces = kept * (a.shape.row_bytes / 16 > a.shape.segments + 1 ? a.shape.row_bytes / 16 : a.shape.segments + 1), each = kCopyThreads * kCopyItems;
        const dim3 grid((unsigned)((pieces + each - 1) / each), 4 * (unsigned)a.shape.kv_heads, (unsigned)a.batch);
        hipLaunchKernelGGL(evict_copy_kernel<false>, grid, dim3(kCopyThreads), 0, (hipStream_t)stream, a);
        hipLaunchKernelGGL(evict_copy_kernel<true>, grid, dim3(kCopyThreads), 0, (hipStream_t)stream, a);
    } else {
        hipLaunchKernelGGL(evict_move_kernel, dim3(4, (unsigned)a.shape.kv_heads, (unsigned)a.batch), dim3(kMoveThreads), 0, (hipStream_t)stream, a);
    }
    launch_ok(what);
}
