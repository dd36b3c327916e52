// Products of weights held in 4 bits with many tokens (layout: qt_linear.h).
#include <type_traits>

#include "qt_linear.h"

#define QT_LDS __attribute__((address_space(3)))
#define QT_GLOBAL __attribute__((address_space(1)))

namespace qt {
namespace {

constexpr int kManyWaves = 4, kManyThreads = 64 * kManyWaves;
constexpr int kXcds = 8;

struct ManyGrid { int rows, columns, group; };      // tiles of tokens and of outputs; rows that are gone through together

// A workgroup's tile: neighbours on an XCD (workgroups go round the XCDs in turn) take tiles that share tokens and outputs.
__device__ __forceinline__ bool many_tile(const ManyGrid &g, int &row, int &column) {
    const int all = g.rows * g.columns, each = (all + kXcds - 1) / kXcds;
    const int index = (int)(blockIdx.x % kXcds) * each + (int)(blockIdx.x / kXcds);
    if ((int)(blockIdx.x / kXcds) >= each || index >= all) return false;
    const int group = index / (g.group * g.columns), rest = index - group * g.group * g.columns;
    const int rows = min(g.group, g.rows - group * g.group);
    column = rest / rows, row = group * g.group + rest - column * rows;
    return true;
}

// A workgroup takes 16 MT tokens x 64 N outputs, each wave all of the tokens and 16 N outputs.  Tokens lie in LDS as the matrix instructions take
// them (sixteen tokens x 32 inputs are 1 KB, 16 bytes a lane), in bf16 two blocks of 128 inputs in turn, straight from memory where rows are aligned;
// numbers of the next block are on their way in registers.  They are exact in bf16, and scales multiply the sums of 64 inputs: four vector
// operations beside every two matrix ones, and as many to expand the numbers, are what a wave does beside them.
//
// Bound by the matrix instructions and the vector operations between them: 6000 tokens through 11008 x 4096 in bf16 449 to 462 us, 1170 to 1200 TFLOP/s, where the
// library's product of bf16 matrices takes 519 us; 1024 tokens through 4096 x 4096 39 us, 885 TFLOP/s; 2048 tokens through 11008 x 4096 in fp32 (three
// matrix operations for each) 498 us, 371 TFLOP/s.  Results stored two bytes a lane: 510, 43 and 508 us.  Four lanes side by side load a token's line: 547 us where sixteen tokens' lines were touched by each.  Tried: the next operands read from LDS in front of the matrix instructions (620 us: registers), the
// matrix instructions at a higher priority, in groups with the vector ones, or one tile ahead of them (512 to 529 us beside 513).  Of all cycles, at a clock that falls to 2.0 GHz, matrix instructions take 52 % and vector ones 55 %, in the
// 1.7 waves that a SIMD has on average.
//
// STAGED: tokens on their way in registers while a block is multiplied, for rows of bf16 that are not aligned to sixteen bytes.
// SPLIT: two times four waves, which take the blocks of 128 inputs in turn and join their sums through LDS.
template <bool BF16, int MT, int N, int SPLIT, bool STAGED>
__global__ __launch_bounds__(SPLIT * kManyThreads, SPLIT == 1 && BF16 && MT == 4 ? 3 : 2) void linear_many_kernel(const LinearArgs a, const ManyGrid grid, const int shift) {
    constexpr int P = Eight<BF16>::kPieces, GROUPS = 2, J = 4 / GROUPS, kBuffers = BF16 ? 2 : 1;
    constexpr int kPlane = MT * 4 * 64;             // sixteen bytes each
    __shared__ qt_u32x4 s_all[SPLIT][kBuffers * P * kPlane];
    const int lane = threadIdx.x & 63, turn = __builtin_amdgcn_readfirstlane(threadIdx.x / kManyThreads), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % kManyWaves;
    const int quarter = lane >> 4;
    qt_u32x4 *const s_x = s_all[turn];
    int row, column;
    if (!many_tile(grid, row, column)) return;
    const int first_token = row * 16 * MT, first_tile = column * (kManyWaves * N) + wave * N;
    const int tiles = (a.outputs + 15) >> 4;
    const uint32_t code_at = 16 * lane, scale_at = lane & 15;
    qt_u32x4 word[N];
    float scale[N][GROUPS];
    const auto load_weights = [&](int block) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const long long tile = min(first_tile + n, tiles - 1);
            word[n] = *(const qt_u32x4 *)(a.codes + ((tile * a.blocks + block) << 10) + code_at);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g)
                scale[n][g] = (a.scales + (tile * a.segments + min((block * GROUPS + g) >> shift, a.segments - 1)) * kLinearOutputs)[scale_at];
        }
    };
    // a wave's part of a block of tokens: MT of the 4 MT pieces of 1 KB
    Eight<BF16> raw[STAGED || !BF16 ? MT : 1];
    // (four lanes side by side load 64 bytes of a token, in an order that keeps the lanes which read them off each other's banks)
    const int eighth = 8 * ((lane & 3) ^ quarter), mine = 4 * (lane & 15) + (quarter ^ ((lane >> 2) & 3));
    const uint8_t *from[MT / 4];
    int valid[MT / 4];
#pragma unroll
    for (int i = 0; i < MT / 4; ++i) {
        const int token = first_token + 16 * (wave * (MT / 4) + i) + (lane >> 2);
        valid[i] = token < a.tokens ? a.inputs : 0;
        from[i] = (const uint8_t *)a.x + (long long)min(token, a.tokens - 1) * a.x_stride * (BF16 ? 2 : 4) + eighth * (BF16 ? 2 : 4);
    }
    // (tokens behind the last are the last one again, or zeros: their results are not stored)
    const auto put = [&](const Eight<BF16> &x, int i, int buffer) {
        bf16x8 pieces[P];
        x.pieces(pieces);
#pragma unroll
        for (int n = 0; n < P; ++n) s_x[(buffer * P + n) * kPlane + (wave * MT + i) * 64 + lane] = __builtin_bit_cast(qt_u32x4, pieces[n]);
    };
    const auto put_rest = [&](int first, int buffer) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            Eight<BF16> x;
            x.load(from[i >> 2], first + 32 * (i & 3), valid[i >> 2] - eighth);
            put(x, i, buffer);
        }
    };
    const auto load_tokens = [&](int block, int buffer) {
        const int first = block * kLinearInputs;
        if constexpr (!BF16) {
#pragma unroll
            for (int i = 0; i < MT; ++i) raw[i].load(from[i >> 2], first + 32 * (i & 3), valid[i >> 2] - eighth);
        } else if constexpr (STAGED) {
            // (nothing but whole blocks, so that they are waited for where they are used)
            if (first + kLinearInputs <= a.inputs) {
#pragma unroll
                for (int i = 0; i < MT; ++i) raw[i].load(from[i >> 2], first + 32 * (i & 3));
            }
        } else if (first + kLinearInputs <= a.inputs) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
                __builtin_amdgcn_global_load_lds((const QT_GLOBAL void *)(from[i >> 2] + 2 * (first + 32 * (i & 3))), (QT_LDS void *)(s_x + buffer * kPlane + (wave * MT + i) * 64),
                                                 16, 0, 0);
        } else {
            put_rest(first, buffer);
        }
    };
    const auto put_tokens = [&](int block, int buffer) {
        if constexpr (BF16 && STAGED) {
            const int first = block * kLinearInputs;
            if (first + kLinearInputs <= a.inputs) {
#pragma unroll
                for (int i = 0; i < MT; ++i) put(raw[i], i, buffer);
            } else {
                put_rest(first, buffer);
            }
        }
        if constexpr (!BF16) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                put(raw[i], i, buffer);
                __builtin_amdgcn_sched_barrier(0);          // (one at a time: registers)
            }
        }
    };
    fp4_f32x4 sum[MT][N];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < N; ++n) sum[m][n] = (fp4_f32x4){0.f, 0.f, 0.f, 0.f};
    if (turn < a.blocks) {
        load_tokens(turn, 0);
        load_weights(turn);
        put_tokens(turn, 0);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int first = 0; first < a.blocks; first += SPLIT) {
        const int block = first + turn, buffer = BF16 ? (first / SPLIT) & 1 : 0;
        qt_u32x4 now[N];
        float by[N][GROUPS];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            now[n] = word[n];
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) by[n][g] = scale[n][g];
        }
        const bool more = block + SPLIT < a.blocks;
        if (more) {
            load_tokens(block + SPLIT, BF16 ? buffer ^ 1 : 0);
            load_weights(block + SPLIT);
        }
        // (of an odd number of blocks the last is one of the first waves')
        const bool mine_too = SPLIT == 1 || block < a.blocks;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            if (!mine_too) break;
            bf16x8 numbers[N][J];
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int j = 0; j < J; ++j) numbers[n][j] = fp4_to_bf16(now[n][g * J + j]);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                fp4_f32x4 part[N];
#pragma unroll
                for (int n = 0; n < N; ++n) part[n] = (fp4_f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    bf16x8 x[P];
#pragma unroll
                    for (int p = 0; p < P; ++p) x[p] = __builtin_bit_cast(bf16x8, s_x[(buffer * P + p) * kPlane + (m * 4 + g * J + j) * 64 + mine]);
#pragma unroll
                    for (int n = 0; n < N; ++n) part[n] = multiply_pieces<P>(x, numbers[n][j], part[n]);
                }
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[m][n][i] = __builtin_fmaf(by[n][g], part[n][i], sum[m][n][i]);
            }
        }
        if constexpr (!BF16) {
            __syncthreads();
        }
        if (more) put_tokens(block + SPLIT, BF16 ? buffer ^ 1 : 0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
    if constexpr (SPLIT > 1) {
        static_assert(SPLIT == 2 && MT * N <= kBuffers * P * kPlane / kManyThreads, "room for the sums of one half");
        fp4_f32x4 *const s_sum = (fp4_f32x4 *)s_all[1];
        if (turn == 1) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < N; ++n) s_sum[((wave * MT + m) * N + n) * 64 + lane] = sum[m][n];
        }
        __syncthreads();
        if (turn == 1) return;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < N; ++n) sum[m][n] += s_sum[((wave * MT + m) * N + n) * 64 + lane];
    }
    if ((first_tile + N) * kLinearOutputs <= a.outputs) {
        // sixteen tokens at a time through LDS, so that a lane stores sixteen bytes of a token
        typedef typename std::conditional<BF16, uint16_t, float>::type Number;
        typedef typename std::conditional<BF16, Unaligned16, Unaligned16of4>::type Store;
        constexpr int kEach = BF16 ? 8 : 4, kRow = 16 * N + kEach, kLanes = 16 * N / kEach;
        Number *const s_out = (Number *)s_all[0] + wave * 16 * kRow;
        float bias[N];
#pragma unroll
        for (int n = 0; n < N; ++n) bias[n] = linear_bias(a, (first_tile + n) * kLinearOutputs + (lane & 15));
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y = sum[m][n][i] + bias[n];
                    if constexpr (BF16) s_out[(4 * quarter + i) * kRow + 16 * n + (lane & 15)] = float_to_bf16_bits(y);
                    else s_out[(4 * quarter + i) * kRow + 16 * n + (lane & 15)] = y;
                }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int k = 0; k < 16 * kLanes / 64; ++k) {
                const int at = 64 * k + lane, token = first_token + 16 * m + at / kLanes, column = at % kLanes * kEach;
                const qt_u32x4 y = *(const qt_u32x4 *)(s_out + at / kLanes * kRow + column);
                if (token < a.tokens) ((Store *)((Number *)a.out + token * a.out_stride + first_tile * kLinearOutputs + column))->v = y;
            }
            asm volatile("" ::: "memory");
        }
        return;
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int output = (first_tile + n) * kLinearOutputs + (lane & 15);
        if (output >= a.outputs) continue;
        const float bias = linear_bias(a, output);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int token = first_token + 16 * m + 4 * quarter + i;
                if (token < a.tokens) linear_store<BF16>(a, token, output, sum[m][n][i] + bias);
            }
    }
}

bool linear_aligned(const LinearArgs &a) { return is_aligned(a.x, 16) && a.x_stride % 8 == 0; }

template <bool BF16, int MT, int N, int SPLIT, bool STAGED>
void launch_many(const LinearArgs &a, int scales_of_block, hipStream_t stream) {
    const ManyGrid grid = {(a.tokens + 16 * MT - 1) / (16 * MT), (a.outputs + 64 * N - 1) / (64 * N), 8};
    const long long all = (long long)grid.rows * grid.columns, blocks = (all + kXcds - 1) / kXcds * kXcds;
    if (blocks >= kMostThreads / (SPLIT * kManyThreads)) { set_error(kBadArgument, "linear_product: too many tokens and outputs (%d, %d)", a.tokens, a.outputs); return; }
    const int shift = scales_of_block == 2 ? 0 : 1 + a.scales_shift;
    hipLaunchKernelGGL((linear_many_kernel<BF16, MT, N, SPLIT, STAGED>), dim3((unsigned)blocks), dim3(SPLIT * kManyThreads), 0, stream, a, grid, shift);
}

}  // namespace

long long linear_many_workgroups(const LinearArgs &a) { return (long long)((a.tokens + 63) / 64) * ((a.outputs + 127) / 128); }

// Large tiles use what they read more often, but two of them fill a unit, and the last ones leave it half idle: from one and a half a unit on, in fp32 from three and a
// half.  4096 inputs in bf16, 128 x 256 against 64 x 128, 1024 tokens and 11008 outputs (344 large) 104.8 and 100.5 us, 14336 (448) 112.4 and 120.9, 4096 and 4096 (512) 119 and
// 137, 2048 and 11008 (688) 179 and 184.5; in fp32 64 x 192 against 64 x 128, 1024 and 4096 (352) 120 and 102, 8192 (688) 204 and 199.5, 11008 (928) 251 and 287.5.
// With no more than one workgroup a unit, eight waves of it cover each other's loads: 512 tokens and 4096 outputs (256 workgroups) 23.1 us, of four waves 26.6, in fp32 56
// and 72; 256 and 14336 (448) in fp32 108 and 95, as a unit's LDS holds one of them, in bf16 37 and 38.
// Rows that are not aligned are STAGED, and take the smaller tile: 6000 tokens of 4100 inputs, 11008 outputs 605 us (aligned 460; put into LDS as they come 60 more, by the larger tile 150),
// 898 of 3140, 2202 outputs 33 us (3136 29).
void launch_linear_many(const LinearArgs &a, bool bf16, int scales_of_block, hipStream_t stream) {
    const long long large = bf16 ? (long long)((a.tokens + 127) / 128) * ((a.outputs + 255) / 256) : (long long)((a.tokens + 63) / 64) * ((a.outputs + 191) / 192);
    const bool aligned = linear_aligned(a);
    if (2 * large >= (bf16 ? 3LL : 7LL) * compute_units() && (!bf16 || aligned)) {
        if (bf16) launch_many<true, 8, 4, 1, false>(a, scales_of_block, stream);
        else launch_many<false, 4, 3, 1, false>(a, scales_of_block, stream);
    } else if (linear_many_workgroups(a) > compute_units()) {
        if (!bf16) launch_many<false, 4, 2, 1, false>(a, scales_of_block, stream);
        else if (aligned) launch_many<true, 4, 2, 1, false>(a, scales_of_block, stream);
        else launch_many<true, 4, 2, 1, true>(a, scales_of_block, stream);
    } else {
        if (!bf16) launch_many<false, 4, 2, 2, false>(a, scales_of_block, stream);
        else if (aligned) launch_many<true, 4, 2, 2, false>(a, scales_of_block, stream);
        else launch_many<true, 4, 2, 2, true>(a, scales_of_block, stream);
    }
}

}  // namespace qt
