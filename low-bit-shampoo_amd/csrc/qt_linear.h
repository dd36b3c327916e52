// Weights of a projection held in 4 bits, and their products with tokens.
//
// A row of weights (the inputs of one output) is cut into segments of `blocksize`, each an fp32 scale and 4-bit floating numbers as in
// the attention cache (qt_cache.h).  Numbers lie as the matrix instructions take them: 16 outputs x 128 inputs are 1024 bytes, 16
// for each lane of a wave -- lane l has output l % 16, its byte 4 j + i the inputs 32 j + 8 (l / 16) + 2 i (low nibble) and the next one
// -- so that a wave's load is 1 KB without a gap and needs no exchange.  Blocks of 128 inputs follow one another, then the next 16
// outputs.  Scales: [ceil(outputs / 16)][segments][16].  What is behind the last input or output is zero.
#pragma once

#include "qt_common.h"
#include "qt_fp4.h"
#include "qtensor_hip.h"

namespace qt {

constexpr int kLinearInputs = 128;      // of a block
constexpr int kLinearOutputs = 16;

struct LinearArgs {
    const uint8_t *codes;
    const float *scales;
    const void *x, *bias;
    void *out;
    long long x_stride, out_stride;     // elements between tokens
    int tokens, inputs, outputs;
    int blocks, segments;               // of 128 inputs; scales of an output
    int scales_shift;                   // 1 where two blocks share a scale
    bool bias_bf16;
};

// The product for many tokens (qt_linear_many.hip), and of how many workgroups it is at least.
long long linear_many_workgroups(const LinearArgs &a);
void launch_linear_many(const LinearArgs &a, bool bf16, int scales_of_block, hipStream_t stream);

#if defined(__HIPCC__)
__device__ __forceinline__ float linear_bias(const LinearArgs &a, int output) {
    if (!a.bias) return 0.0f;
    return a.bias_bf16 ? bf16_bits_to_float(((const uint16_t *)a.bias)[output]) : ((const float *)a.bias)[output];
}
template <bool BF16>
__device__ __forceinline__ void linear_store(const LinearArgs &a, int token, int output, float y) {
    const long long at = token * a.out_stride + output;
    if (BF16) ((uint16_t *)a.out)[at] = float_to_bf16_bits(y);
    else ((float *)a.out)[at] = y;
}
#endif
}  // namespace qt
