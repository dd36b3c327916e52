// Weights held in 4 bits: encoding, decoding, products with few tokens (layout: qt_linear.h).
#include "qt_linear.h"

namespace qt {
namespace {

constexpr int kCodeThreads = 256;

struct LinearCopy {
    uint8_t *codes;
    float *scales;
    void *weight;
    long long row_stride;
    int inputs, outputs, blocks, segments, blocksize;
};

// A wave takes 16 outputs x 256 inputs: two blocks, which hold whole segments of every size: a segment's largest is among four lanes, and what is written is what the
// products read, 1 KB a block.  Bound by memory: 28672 x 8192 of bf16 encoded in 108 us, 5.6 TB/s, of fp32 in 205, 5.2; weights are laid out
// once.  Decoded in 185 us, 3.3 TB/s, and 286, 3.7: a wave stores 64 bytes (fp32 128) of each of sixteen rows at a time.
template <bool BF16, bool WRITE>
__global__ __launch_bounds__(kCodeThreads) void linear_copy_kernel(const LinearCopy a) {
    const int lane = threadIdx.x & 63, quarter = lane >> 4;
    const int pairs = (a.blocks + 1) >> 1;
    const long long work = (long long)blockIdx.x * (kCodeThreads / 64) + (threadIdx.x >> 6);
    const long long tile = work / pairs;
    const int pair = (int)(work - tile * pairs);
    const long long output = tile * kLinearOutputs + (lane & 15);
    if (tile * kLinearOutputs >= a.outputs) return;
    const bool there = output < a.outputs;
    uint8_t *row = (uint8_t *)a.weight + output * a.row_stride * (BF16 ? 2 : 4);
    uint8_t *codes = a.codes + ((tile * a.blocks + 2 * pair) << 10) + 16 * lane;
    if constexpr (WRITE) {
        Eight<BF16> raw[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) raw[j].load(row, 256 * pair + 32 * j + 8 * quarter, there ? a.inputs : 0);
        float x[8][8];
        uint32_t top[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            top[j] = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[j][e] = BF16 ? __uint_as_float(e & 1 ? raw[j].raw[e / 2] & 0xffff0000u : raw[j].raw[e / 2] << 16) : __uint_as_float(raw[j].raw[BF16 ? 0 : e]);
                top[j] = max(top[j], __float_as_uint(x[j][e]) & 0x7fffffffu);
            }
        }
        const int each = a.blocksize >> 5;              // steps of 32 inputs of a segment
#pragma unroll
        for (int half = 1; half < 8; half *= 2)
            if (half < each) {
                uint32_t other[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) other[j] = top[j ^ half];
#pragma unroll
                for (int j = 0; j < 8; ++j) top[j] = max(top[j], other[j]);
            }
        uint32_t word[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            top[j] = max(top[j], (uint32_t)__shfl_xor((int)top[j], 16, 64));
            top[j] = max(top[j], (uint32_t)__shfl_xor((int)top[j], 32, 64));
            float scale;
            word[j] = encode_fp4<8>(x[j], top[j], scale);
            const int segment = (256 * pair + 32 * j) / a.blocksize;
            if (quarter == 0 && (32 * j) % a.blocksize == 0 && segment < a.segments) a.scales[(tile * a.segments + segment) * kLinearOutputs + (lane & 15)] = scale;
        }
        *(qt_u32x4 *)codes = (qt_u32x4){word[0], word[1], word[2], word[3]};
        if (2 * pair + 1 < a.blocks) *(qt_u32x4 *)(codes + 1024) = (qt_u32x4){word[4], word[5], word[6], word[7]};
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (2 * pair + i >= a.blocks) break;
            const qt_u32x4 words = *(const qt_u32x4 *)(codes + 1024 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int first = 256 * pair + 128 * i + 32 * j + 8 * quarter;
                const float scale = a.scales[(tile * a.segments + min(first / a.blocksize, a.segments - 1)) * kLinearOutputs + (lane & 15)];
                const bf16x8 numbers = fp4_to_bf16(words[j]);
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = (float)numbers[e] * scale;
                if (!there || first >= a.inputs) continue;
                if (first + 8 <= a.inputs) {
                    if constexpr (BF16) {
                        ((Unaligned16 *)((uint16_t *)row + first))->v = (qt_u32x4){floats_to_bf16_pair(y[0], y[1]), floats_to_bf16_pair(y[2], y[3]), floats_to_bf16_pair(y[4], y[5]),
                                                                                   floats_to_bf16_pair(y[6], y[7])};
                    } else {
#pragma unroll
                        for (int h = 0; h < 8; h += 4)
                            ((Unaligned16of4 *)((float *)row + first + h))->v =
                                (qt_u32x4){__float_as_uint(y[h]), __float_as_uint(y[h + 1]), __float_as_uint(y[h + 2]), __float_as_uint(y[h + 3])};
                    }
                    continue;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (first + e >= a.inputs) continue;
                    if (BF16) ((uint16_t *)row)[first + e] = float_to_bf16_bits(y[e]);
                    else ((float *)row)[first + e] = y[e];
                }
            }
        }
    }
}

// Products of few tokens: a wave multiplies R tiles of 16 outputs with T of 16 tokens, and the WAVES waves of a workgroup take the blocks of 128
// inputs in turn; their sums are joined through LDS, in the order of the waves.
//
// Bound by reading the weights, which a single token's calls do past the L2: 1 token through 28672 x 8192 in bf16, a scale for 128, 23 us, 5.3 TB/s; 32 tokens through
// 14336 x 4096 9.9 us, 3.5 TB/s, of which 3 are the launch, the first loads and the join; small ones by the launch (2304 x 768 4.4 us a call).  Tried: the next block's
// loads in front of this one's products (no faster: waves of a unit do that for each other), sums joined by one wave (15.8 us for the
// 32 tokens, by all 12.1, before tokens were loaded line by line).
template <bool BF16, int T, int R, int WAVES, int GROUPS, bool STREAM>
__global__ __launch_bounds__(64 * WAVES) void linear_few_kernel(const LinearArgs a) {
    constexpr int P = Eight<BF16>::kPieces, J = 4 / GROUPS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quarter = lane >> 4;
    const int tiles = (a.outputs + kLinearOutputs - 1) / kLinearOutputs;
    const int first_tile = blockIdx.x * R, first_token = blockIdx.y * 16 * T;
    __shared__ fp4_f32x4 s_part[WAVES][R * T][64];
    const uint32_t code_at = 16 * lane, scale_at = lane & 15;
    // (tokens and tiles behind the last are the last one again: what comes of them is not stored)
    // (four lanes side by side load a row's line: 16 tokens through 4096 x 4096 in bf16 5.5 us, else 6.6, in fp32 8.8 and 10.4; two in fp32 7.9 and 7.0)
    const bool apart = a.tokens > (BF16 ? 4 : 8);
    const int eighth = 8 * (apart ? lane & 3 : quarter);
    const uint8_t *x[T];
#pragma unroll
    for (int t = 0; t < T; ++t)
        x[t] = (const uint8_t *)a.x + ((long long)min(first_token + 16 * t + (apart ? lane >> 2 : lane & 15), a.tokens - 1) * a.x_stride + eighth) * (BF16 ? 2 : 4);
    fp4_f32x4 sum[R][T];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < T; ++t) sum[r][t] = (fp4_f32x4){0.f, 0.f, 0.f, 0.f};
    for (int block = wave; block < a.blocks; block += WAVES) {
        qt_u32x4 word[R];
        float scale[R][GROUPS];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const long long tile = min(first_tile + r, tiles - 1);
            word[r] = __builtin_bit_cast(qt_u32x4, load_u32x4<STREAM>(a.codes + ((tile * a.blocks + block) << 10) + code_at));
#pragma unroll
            for (int g = 0; g < GROUPS; ++g)
                scale[r][g] = (a.scales + (tile * a.segments + min((block * GROUPS + g) >> a.scales_shift, a.segments - 1)) * kLinearOutputs)[scale_at];
        }
        Eight<BF16> raw[T][4];
        const int at = block * kLinearInputs;
        if (at + kLinearInputs <= a.inputs) {
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) raw[t][j].load(x[t], at + 32 * j);
        } else {
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) raw[t][j].load(x[t], at + 32 * j, a.inputs - eighth);
        }
        if (apart) {
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) raw[t][j].exchange();
        }
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            bf16x8 numbers[R][J];
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int j = 0; j < J; ++j) numbers[r][j] = fp4_to_bf16(word[r][g * J + j]);
#pragma unroll
            for (int t = 0; t < T; ++t) {
                fp4_f32x4 part[R];
#pragma unroll
                for (int r = 0; r < R; ++r) part[r] = (fp4_f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    bf16x8 pieces[P];
                    raw[t][g * J + j].pieces(pieces);
#pragma unroll
                    for (int r = 0; r < R; ++r) part[r] = multiply_pieces<P>(pieces, numbers[r][j], part[r]);
                }
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[r][t][i] = __builtin_fmaf(scale[r][g], part[r][i], sum[r][t][i]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < T; ++t) s_part[wave][r * T + t][lane] = sum[r][t];
    __syncthreads();
    // every wave joins tiles of its own
#pragma unroll
    for (int n = 0; n < (R * T + WAVES - 1) / WAVES; ++n) {
        const int tile = n * WAVES + wave;
        if (tile >= R * T) break;
        fp4_f32x4 y = s_part[0][tile][lane];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) y += s_part[w][tile][lane];
        const int output = (first_tile + tile / T) * kLinearOutputs + (lane & 15), token = first_token + 16 * (tile % T) + 4 * quarter;
        if (output >= a.outputs) continue;
        const float bias = linear_bias(a, output);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (token + i < a.tokens) linear_store<BF16>(a, token + i, output, y[i] + bias);
    }
}

template <bool BF16, int T, int R, int WAVES>
void launch_few(const LinearArgs &a, int groups, hipStream_t stream) {
    const dim3 grid((unsigned)(((a.outputs + 15) / 16 + R - 1) / R), (unsigned)((a.tokens + 16 * T - 1) / (16 * T)));
    if (groups == 2) hipLaunchKernelGGL((linear_few_kernel<BF16, T, R, WAVES, 2, T == 1>), grid, dim3(64 * WAVES), 0, stream, a);
    else hipLaunchKernelGGL((linear_few_kernel<BF16, T, R, WAVES, 1, T == 1>), grid, dim3(64 * WAVES), 0, stream, a);
}

// One tile of tokens to a workgroup: MOST waves where more than 2048 inputs give each of them blocks, else eight.  One token, 14336 inputs, 4096 outputs in bf16 9.3 us of 16
// waves, 11.4 of 8; in fp32 4096 inputs, 4096 outputs 6.2 and 7.3, 14336 outputs 10.0 and 11.1, where bf16 has 7.3 and 7.4 (32 tokens 15.8 and 15.2).
template <bool BF16, int R, int MOST>
void launch_few_long(const LinearArgs &a, int groups, hipStream_t stream) {
    if (MOST > 8 && a.blocks > 16) launch_few<BF16, 1, R, MOST>(a, groups, stream);
    else launch_few<BF16, 1, R, 8>(a, groups, stream);
}

// Many tokens as soon as the kernel for them has a workgroup for seven of eight units: 4096 inputs in bf16, 256 tokens and 4096 outputs (128 workgroups) 15.1 us here
// and 22.2 there, 384 and 4096 (192) 21.0 and 22.4, 64 and 24000 (188) 24.7 and 22.4, in fp32 46.5 and 53.9, 54.7 and 53.8.
// Its tile is of 64 tokens: 32 tokens, 128000 outputs 74 us here and 80 there, 33 126 and 80, one in fp32 67 and 213; in fp32 from 48 on: 40 tokens 215 and 228, 48 218
// and 198, 50000 outputs 91 and 107, 92 and 94, 28672 outputs 53 and 65, 54 and 53 (1000 inputs, 128000 outputs 33 77 and 56, 48 80 and 52).
// Else the smallest tile of a workgroup whose workgroups have a unit each: every one reads all of its tokens (from L2) and joins its waves, so
// more of them than that cost more than they spread.  By tiles of outputs x tokens, before loads of tokens and joins were as they are: 16 tokens, 4096
// outputs 1 x 1 6.7 us, 2 x 1 7.9, 4 x 1 10.1; 14336 outputs 18.3, 12.6, 10.5; 64 tokens, 4096 outputs 4 x 1 10.5, 4 x 2 15.4; as they are, 64 tokens, 11008
// outputs 4 x 4 14.5, 4 x 2 16.6.  Four waves to a workgroup where there are several for each unit (32 tokens, 28672 outputs 25.1 us against 26.0 of
// eight).  In fp32 eight tiles of outputs share a token's pieces, which take as long to cut as twelve matrix instructions: 128 tokens, 4096 outputs 17.3 us, four tiles 20.9, with two
// of 16 tokens 18.8; one token, 28672 outputs 18.6 us, four tiles and waves 19.8.
template <bool BF16>
void launch_product(const LinearArgs &a, int groups, hipStream_t stream) {
    const long long tiles = (a.outputs + 15) / 16, rows = (a.tokens + 15) / 16, units = compute_units();
    if (a.tokens >= (BF16 ? 33 : 48) && 8 * linear_many_workgroups(a) >= 7 * units) return launch_linear_many(a, BF16, groups, stream);
    if (tiles * rows <= units) return launch_few_long<BF16, 1, 16>(a, groups, stream);
    if ((tiles + 1) / 2 * rows <= units) return launch_few_long<BF16, 2, BF16 ? 8 : 16>(a, groups, stream);
    if ((tiles + 3) / 4 * rows <= units) return launch_few_long<BF16, 4, BF16 ? 8 : 16>(a, groups, stream);
    if constexpr (BF16) {
        if (rows > 1 && (tiles + 3) / 4 * ((rows + 1) / 2) <= units) return launch_few<BF16, 2, 4, 8>(a, groups, stream);
        if (rows > 2 && (tiles + 3) / 4 * ((rows + 3) / 4) <= units) return launch_few<BF16, 4, 4, 8>(a, groups, stream);
        if (rows > 1) return launch_few<BF16, 2, 4, 4>(a, groups, stream);
        return launch_few<BF16, 1, 4, 4>(a, groups, stream);
    } else {
        return launch_few<BF16, 1, 8, 8>(a, groups, stream);
    }
}

bool linear_shape(const char *what, const qtensor_linear *w) {
    if (!w || !w->codes || !w->scales) { set_error(kNullPointer, "%s: null pointer in the weights", what); return false; }
    if (w->blocksize != 64 && w->blocksize != 128 && w->blocksize != 256) {
        set_error(kBadBlocksize, "%s: blocksize %d is not one of 64,128,256", what, w->blocksize);
        return false;
    }
    if (w->inputs < 1 || w->inputs > (1 << 24) || w->outputs < 1 || w->outputs > (1 << 24)) {
        set_error(kBadArgument, "%s: needs 1 to 2^24 inputs and outputs (got %d, %d)", what, w->inputs, w->outputs);
        return false;
    }
    if (!is_aligned(w->codes, 16) || !is_aligned(w->scales, 16)) { set_error(kBadArgument, "%s: unaligned weights", what); return false; }
    return true;
}

void copy_linear(const char *what, bool write, const qtensor_linear *w, void *weight, int is_bf16, long long row_stride, hipStream_t stream) {
    clear_error();
    if (!linear_shape(what, w)) return;
    if (!weight) { set_error(kNullPointer, "%s: null weight", what); return; }
    if (!is_aligned(weight, is_bf16 ? 2 : 4) || row_stride < 0) { set_error(kBadArgument, "%s: a weight aligned to an element, with rows in ascending order", what); return; }
    const int blocks = (w->inputs + kLinearInputs - 1) / kLinearInputs;
    const LinearCopy a = {w->codes, w->scales, weight, row_stride, w->inputs, w->outputs, blocks, (w->inputs + w->blocksize - 1) / w->blocksize, w->blocksize};
    const long long waves = (long long)((w->outputs + 15) / 16) * ((blocks + 1) / 2);
    const long long groups = (waves + kCodeThreads / 64 - 1) / (kCodeThreads / 64);
    if (groups >= kMostThreads / kCodeThreads) { set_error(kBadArgument, "%s: too many weights", what); return; }
    const dim3 grid((unsigned)groups);
    if (write && is_bf16) hipLaunchKernelGGL((linear_copy_kernel<true, true>), grid, dim3(kCodeThreads), 0, stream, a);
    else if (write) hipLaunchKernelGGL((linear_copy_kernel<false, true>), grid, dim3(kCodeThreads), 0, stream, a);
    else if (is_bf16) hipLaunchKernelGGL((linear_copy_kernel<true, false>), grid, dim3(kCodeThreads), 0, stream, a);
    else hipLaunchKernelGGL((linear_copy_kernel<false, false>), grid, dim3(kCodeThreads), 0, stream, a);
    launch_ok(what);
}

}  // namespace
}  // namespace qt

extern "C" void qtensor_hip_linear_quantize(const qtensor_linear *weights, const void *weight, int is_bf16, long long row_stride, void *stream) {
    qt::copy_linear("linear_quantize", true, weights, const_cast<void *>(weight), is_bf16, row_stride, (hipStream_t)stream);
}

extern "C" void qtensor_hip_linear_dequantize(const qtensor_linear *weights, void *weight, int is_bf16, long long row_stride, void *stream) {
    qt::copy_linear("linear_dequantize", false, weights, weight, is_bf16, row_stride, (hipStream_t)stream);
}

extern "C" void qtensor_hip_linear_product(const qtensor_linear *weights, const qtensor_linear_call *call, void *stream) {
    using namespace qt;
    const char *what = "linear_product";
    clear_error();
    if (!linear_shape(what, weights)) return;
    if (!call || (call->tokens > 0 && (!call->x || !call->out))) { set_error(kNullPointer, "%s: null pointer in the call", what); return; }
    const int size = call->is_bf16 ? 2 : 4;
    if (call->tokens < 0 || call->tokens > 0x7fffff00LL || call->x_stride < 0 || call->out_stride < weights->outputs || !is_aligned(call->x, size) || !is_aligned(call->out, size) ||
        (call->bias && !is_aligned(call->bias, call->bias_is_bf16 ? 2 : 4))) {
        set_error(kBadArgument, "%s: needs up to 2^31 - 256 tokens in ascending order, results that do not overlap, and tensors aligned to an element", what);
        return;
    }
    if (call->tokens == 0) return;
    const int blocks = (weights->inputs + kLinearInputs - 1) / kLinearInputs;
    const int groups = weights->blocksize == 64 ? 2 : 1;
    // (a launch takes less than 2^24 workgroups, of 64 tokens and up to 256 outputs)
    const long long most = 1LL << 24;
    for (long long first = 0; first < call->tokens; first += most) {
        const long long tokens = call->tokens - first < most ? call->tokens - first : most;
        const LinearArgs a = {weights->codes, weights->scales, (const uint8_t *)call->x + first * call->x_stride * size, call->bias, (uint8_t *)call->out + first * call->out_stride * size,
                              call->x_stride, call->out_stride, (int)tokens, weights->inputs, weights->outputs, blocks,
                              (weights->inputs + weights->blocksize - 1) / weights->blocksize, weights->blocksize == 256, call->bias_is_bf16 != 0};
        if (call->is_bf16) launch_product<true>(a, groups, (hipStream_t)stream);
        else launch_product<false>(a, groups, (hipStream_t)stream);
        if (!launch_ok(what)) return;
    }
}
