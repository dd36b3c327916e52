// Eviction from a 4-bit attention cache: of every sequence and head the tokens whose totals are largest stay, in their order.
//
// A token is there if its page is.  `keep` of them stay (all, where there are no more): the first `sinks` and the last `recent` places
// of the sequence, then those with the largest totals, ties to the earlier one.  The nth token that stays moves to the place of the nth
// token that is there, which is never behind it.  As heads keep different tokens and every place may be read for one that is written
// before it, all that moves goes through scratch memory: gathered, then put down.
//
// Three launches: the choice (a workgroup a sequence and head), which lists where tokens come from and go to; gathering; putting down.
#include "qt_cache.h"

namespace qt {
namespace {

constexpr int kChooseThreads = 1024, kChooseWaves = kChooseThreads / 64;
constexpr int kMoveThreads = 256;

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
    uint8_t *held_codes[2];
    float *held_scales[2], *held_totals;
};

__device__ __forceinline__ int evict_end(const EvictArgs &a, int b) {
    const long long covered = (long long)a.table_pages << a.shape.page_shift;
    return (int)min((long long)max(a.lengths[b], 0), min(covered, 0x7fffff00LL));
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

// Sum over the threads in front of this one, and over all; `s_waves`: scratch.
__device__ __forceinline__ int flags_before(bool flag, int *s_waves, int &all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned long long at = __ballot(flag);
    __syncthreads();
    if (lane == 0) s_waves[wave] = __popcll(at);
    __syncthreads();
    int before = __popcll(at & ((1ull << lane) - 1));
    all = 0;
#pragma unroll
    for (int w = 0; w < kChooseWaves; ++w) {
        const int n = s_waves[w];
        before += w < wave ? n : 0;
        all += n;
    }
    return before;
}

__global__ __launch_bounds__(kChooseThreads) void evict_choose_kernel(const EvictArgs a) {
    __shared__ int s_count[256], s_waves[kChooseWaves], s_there, s_kept_anyhow, s_digit, s_above;
    const int head = blockIdx.x, b = blockIdx.y;
    const int length = max(a.lengths[b], 0), end = evict_end(a, b);
    const float *totals = a.totals + b * a.total_sequence + head * a.total_head;
    const auto anyhow = [&](int place) { return place < a.sinks || place >= length - a.recent; };
    if (threadIdx.x == 0) s_there = 0, s_kept_anyhow = 0;
    __syncthreads();
    int there = 0, protect = 0;
    for (int place = threadIdx.x; place < end; place += kChooseThreads) {
        const bool is = evict_line(a, b, place) >= 0;
        there += is, protect += is && anyhow(place);
    }
    atomicAdd(&s_there, there), atomicAdd(&s_kept_anyhow, protect);
    __syncthreads();
    const int stay = min(s_there, a.keep);
    int wanted = stay - s_kept_anyhow;          // by their totals
    // the least key of those that stay, eight bits at a time, and how many of the tokens with that key do
    uint32_t least = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < 256) s_count[threadIdx.x] = 0;
        __syncthreads();
        for (int place = threadIdx.x; place < end; place += kChooseThreads) {
            if (anyhow(place) || evict_line(a, b, place) < 0) continue;
            const uint32_t key = total_key(totals[place]);
            if (shift == 24 || (key >> (shift + 8)) == (least >> (shift + 8))) atomicAdd(&s_count[(key >> shift) & 255], 1);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int above = 0, digit = 255;
            for (; digit > 0 && above + s_count[digit] < wanted; --digit) above += s_count[digit];
            s_digit = digit, s_above = above;
        }
        __syncthreads();
        least |= (uint32_t)s_digit << shift;
        wanted -= s_above;
    }
    int *from = a.from + ((long long)b * a.shape.kv_heads + head) * a.keep, *to = a.to + ((long long)b * a.shape.kv_heads + head) * a.keep;
    int there_before = 0, stay_before = 0, ties_before = 0;
    for (int first = 0; first < end; first += kChooseThreads) {
        const int place = first + (int)threadIdx.x;
        const bool is = place < end && evict_line(a, b, place) >= 0;
        const bool by_total = is && !anyhow(place);
        const uint32_t key = by_total ? total_key(totals[place]) : 0u;
        int all;
        const bool tie = by_total && key == least;
        const int ties = ties_before + flags_before(tie, s_waves, all);
        ties_before += all;
        const bool stays = is && (!by_total || key > least || (tie && ties < wanted));
        const int nth = stay_before + flags_before(stays, s_waves, all);
        stay_before += all;
        if (stays && nth < stay) from[nth] = place;
        const int slot = there_before + flags_before(is, s_waves, all);
        there_before += all;
        if (is && slot < stay) {
            to[slot] = place;
            if (slot == stay - 1 && head == 0) a.new_lengths[b] = place + 1;
        }
    }
    if (threadIdx.x == 0 && head == 0) {
        a.count[b] = stay;
        if (stay == 0) a.new_lengths[b] = 0;
    }
}

// A thread moves sixteen bytes of keys and of values, or (the first one of a token behind those) its scales and total.
template <bool GATHER>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(const EvictArgs a) {
    const int head = blockIdx.y, b = blockIdx.z;
    const int parts = a.shape.row_bytes / 16 + 1;
    const long long index = (long long)blockIdx.x * kMoveThreads + threadIdx.x;
    const int nth = (int)(index / parts), part = (int)(index - (long long)nth * parts);
    if (nth >= a.count[b]) return;
    const long long sequence = (long long)b * a.shape.kv_heads + head, entry = sequence * a.keep + nth;
    const int from = a.from[entry], to = a.to[entry];
    if (from == to) return;
    const int place = GATHER ? from : to;
    const long long line = evict_line(a, b, place) + ((long long)head << a.shape.page_shift), inside = place & ((1 << a.shape.page_shift) - 1);
    if (part < parts - 1) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            qt_u32x4 *there = (qt_u32x4 *)(a.codes[i] + (line + inside) * a.shape.row_bytes + 16 * part), *held = (qt_u32x4 *)(a.held_codes[i] + entry * a.shape.row_bytes + 16 * part);
            if (GATHER) *held = *there;
            else *there = *held;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            for (int g = 0; g < a.shape.segments; ++g) {
                float *there = a.scales[i] + line * a.shape.segments + ((long long)g << a.shape.page_shift) + inside, *held = a.held_scales[i] + entry * a.shape.segments + g;
                if (GATHER) *held = *there;
                else *there = *held;
            }
        float *there = a.totals + b * a.total_sequence + head * a.total_head + place, *held = a.held_totals + entry;
        if (GATHER) *held = *there;
        else *there = *held;
    }
}

long long rounded(long long bytes) { return (bytes + 255) & ~255LL; }

struct EvictSizes { long long lists, count, codes, scales, totals, all; };
EvictSizes evict_sizes(const CacheShape &shape, int batch, long long keep) {
    const long long entries = (long long)batch * shape.kv_heads * keep;
    EvictSizes s = {rounded(4 * entries), rounded(4LL * batch), rounded(entries * shape.row_bytes), rounded(4 * entries * shape.segments), rounded(4 * entries), 0};
    s.all = 2 * s.lists + s.count + 2 * s.codes + 2 * s.scales + s.totals;
    return s;
}

bool evict_shape(const char *what, const qtensor_cache *cache, const qtensor_cache_places *places, long long keep, CacheShape &shape, CachePlaces &at) {
    if (!cache_shape(what, cache, shape) || !cache_places(what, places, at)) return false;
    if (keep < 1) { set_error(kBadArgument, "%s: needs at least a token to keep (got %lld)", what, keep); return false; }
    if (at.batch > 65535 || shape.kv_heads > 65535) { set_error(kBadArgument, "%s: too many sequences or heads (%d, %d)", what, at.batch, shape.kv_heads); return false; }
    return true;
}
long long evict_keep(const CacheShape &shape, const CachePlaces &at, long long keep) {
    const long long covered = (long long)at.table_pages << shape.page_shift, most = covered < 0x7fffff00LL ? covered : 0x7fffff00LL;
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
    const auto take = [&](long long bytes) { uint8_t *here = p; p += bytes; return here; };
    a.from = (int *)take(size.lists), a.to = (int *)take(size.lists), a.count = (int *)take(size.count);
    for (int i = 0; i < 2; ++i) {
        a.codes[i] = cache->codes[i], a.scales[i] = cache->scales[i];
        a.held_codes[i] = take(size.codes), a.held_scales[i] = (float *)take(size.scales);
    }
    a.held_totals = (float *)take(size.totals);
    a.totals = totals, a.total_sequence = total_sequence, a.total_head = total_head;
    const long long most = 0x7fffffff;
    a.keep = (int)kept, a.recent = (int)(recent < most ? recent : most), a.sinks = (int)(sinks < most ? sinks : most);
    a.new_lengths = new_lengths;
    const long long blocks = (kept * (a.shape.row_bytes / 16 + 1) + kMoveThreads - 1) / kMoveThreads;
    if (blocks > 0x7fffffffLL) { set_error(kBadArgument, "%s: too many tokens to keep (%lld)", what, kept); return; }
    const dim3 grid((unsigned)blocks, (unsigned)a.shape.kv_heads, (unsigned)a.batch);
    hipLaunchKernelGGL(evict_choose_kernel, dim3((unsigned)a.shape.kv_heads, (unsigned)a.batch), dim3(kChooseThreads), 0, (hipStream_t)stream, a);
    hipLaunchKernelGGL((evict_move_kernel<true>), grid, dim3(kMoveThreads), 0, (hipStream_t)stream, a);
    hipLaunchKernelGGL((evict_move_kernel<false>), grid, dim3(kMoveThreads), 0, (hipStream_t)stream, a);
    launch_ok(what);
}
