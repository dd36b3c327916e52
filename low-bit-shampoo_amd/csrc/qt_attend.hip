// Attention over a cache held in 4 bits (layout: qt_cache.h): out_i = sum_j p_ij v_j, p_ij = softmax_j(scale q_i . k_j) over the
// tokens j that query i sees: j <= i and, with a window, i - j < window or j < sinks.
#include "qt_cache.h"

namespace qt {
namespace {

struct AttendArgs {
    CacheShape shape;
    CachePlaces at;
    const uint8_t *codes[2];
    const float *scales[2];
    const void *q;
    void *out;
    long long q_token, q_head, out_token, out_head;
    int heads, group;
    float factor;           // scale * log2 e
    int window, sinks;      // window 0: no window
};

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, 64));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
    return x;
}

// One wave per query and head: a token per lane for the scores of 64 tokens, then two elements per lane and byte for their values.
template <bool BF16>
__global__ __launch_bounds__(256) void attend_kernel(const AttendArgs a) {
    __shared__ float s_q[4][256];
    __shared__ float s_p[4][64][4];         // weight times the value's scale, per segment
    __shared__ long long s_row[4][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int token = blockIdx.x, head = blockIdx.y * 4 + wave;
    int b = token;
    if (a.at.starts) b = sequence_of_block(a.at, token);
    if (head >= a.heads || b >= a.at.batch) return;
    if (a.at.starts && token < a.at.starts[b]) return;
    const int dim = a.shape.head_dim, kv = head / a.group;
    const int position = a.at.starts ? a.at.lengths[b] - (a.at.starts[b + 1] - token) : a.at.lengths[b] - 1;
    for (int d = lane; d < 256; d += 64) {
        const long long at = token * a.q_token + head * a.q_head + d;
        s_q[wave][d] = d >= dim ? 0.0f : BF16 ? bf16_bits_to_float(((const uint16_t *)a.q)[at]) : ((const float *)a.q)[at];
    }
    wave_lds_sync();
    float best = -__builtin_inff(), sum = 0.0f;
    float acc[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
    int first = 0;
    const long long covered = (long long)a.at.table_pages << a.shape.page_shift;      // (lengths beyond the table: nothing is there)
    const int end = (int)min((long long)position + 1, covered);
    while (first < end) {
        const int j = first + lane;
        const bool seen = j < end && (!a.window || position - j < a.window || j < a.sinks);
        const long long row = seen ? cache_row(a.shape, a.at, b, j, kv) : -1;
        float score = -__builtin_inff();
        if (row >= 0) {
            const uint8_t *codes = a.codes[0] + row * a.shape.row_bytes;
            const float *scale = a.scales[0] + cache_scale_at(a.shape, row);
            score = 0.0f;
            for (int c = 0; c < a.shape.row_bytes; c += 16) {
                const uint4 w = *(const uint4 *)(codes + c);
                const uint32_t v[4] = {w.x, w.y, w.z, w.w};
                float part = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float *q = &s_q[wave][2 * c + 8 * i];
                    const cache_f32x2 e0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v[i], 1.0f, 0), e1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v[i], 1.0f, 1),
                                      e2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v[i], 1.0f, 2), e3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v[i], 1.0f, 3);
                    part += e0.x * q[0] + e0.y * q[1] + e1.x * q[2] + e1.y * q[3] + e2.x * q[4] + e2.y * q[5] + e3.x * q[6] + e3.y * q[7];
                }
                score += part * scale[(long long)((2 * c) >> a.shape.segment_shift) << a.shape.page_shift];
            }
            score *= a.factor;
        }
        const float top = fmaxf(best, wave_max(score));
        const float base = top == -__builtin_inff() ? 0.0f : top;
        const float fade = __builtin_amdgcn_exp2f(best - base);
        const float p = row >= 0 ? __builtin_amdgcn_exp2f(score - base) : 0.0f;
        sum = sum * fade + wave_sum(p);
        best = top;
        s_row[wave][lane] = row;
        if (row >= 0)
            for (int i = 0; i < a.shape.segments; ++i)
                s_p[wave][lane][i] = p * a.scales[1][cache_scale_at(a.shape, row) + ((long long)i << a.shape.page_shift)];
        wave_lds_sync();
#pragma unroll
        for (int i = 0; i < 2; ++i) acc[i][0] *= fade, acc[i][1] *= fade;
        const int count = min(64, end - first);
        for (int t = 0; t < count; ++t) {
            const long long here = s_row[wave][t];
            if (here < 0) continue;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int byte = lane + 64 * i;
                if (byte >= a.shape.row_bytes) continue;
                const float w = s_p[wave][t][(2 * byte) >> a.shape.segment_shift];
                const cache_f32x2 e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4((uint32_t)a.codes[1][here * a.shape.row_bytes + byte], 1.0f, 0);
                acc[i][0] += w * e.x;
                acc[i][1] += w * e.y;
            }
        }
        wave_lds_sync();
        first += 64;
        if (a.window && first >= a.sinks) first = max(first, (position + 1 - a.window) & ~63);
    }
    const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int d = 2 * (lane + 64 * i) + e;
            if (d >= dim) continue;
            const long long at = token * a.out_token + head * a.out_head + d;
            const float y = sum == 0.0f ? 0.0f : acc[i][e] * by;
            if (BF16) ((uint16_t *)a.out)[at] = float_to_bf16_bits(y);
            else ((float *)a.out)[at] = y;
        }
}

}  // namespace
}  // namespace qt

extern "C" void qtensor_hip_cache_attend(const qtensor_cache *cache, const qtensor_cache_places *places, const qtensor_cache_vectors *q,
                                         const qtensor_cache_vectors *out, int heads, float scale, int window, int sinks, void *stream) {
    using namespace qt;
    clear_error();
    AttendArgs a;
    if (!cache_shape("cache_attend", cache, a.shape) || !cache_places("cache_attend", places, a.at)) return;
    if (!q || !out || (a.at.tokens > 0 && (!q->base || !out->base))) { set_error(kNullPointer, "cache_attend: null queries or result"); return; }
    if (heads < 1 || heads > 65535 || heads % a.shape.kv_heads || window < 0 || sinks < 0 || !(scale - scale == 0.0f) || q->is_bf16 != out->is_bf16) {
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
    a.heads = heads, a.group = heads / a.shape.kv_heads;
    a.factor = scale * 1.4426950408889634f;
    a.window = window, a.sinks = sinks;
    const dim3 grid(a.at.tokens, (heads + 3) / 4);
    if (q->is_bf16) hipLaunchKernelGGL(attend_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(attend_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, a);
    launch_ok("cache_attend");
}
