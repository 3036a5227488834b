// Launchers of the operators between two decoding steps (one translation unit per group); arguments have been checked.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/mkb200_sequences.h"

namespace mkbs {

using bf16 = __nv_bfloat16;

constexpr int kSms = 148;  // what grids and splits are sized by

// Total order of floats as whole numbers; 0 is below all of them.  Minus zero counts as zero.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t order) { return __uint_as_float(order ^ ((order >> 31) ? 0x80000000u : 0xffffffffu)); }

// Rows that sequence `b` holds.
__device__ __forceinline__ int length_of(const int32_t* lengths, int length, int positions, int b) {
    return min(max(lengths != nullptr ? __ldg(lengths + b) : length, 0), positions);
}

cudaError_t beam_launch(const MkbsBeams& b, cudaStream_t s);
size_t beam_bytes(const MkbsBeams& b);
cudaError_t reorder_launch(const MkbsReorder& r, cudaStream_t s);
cudaError_t select_launch(const MkbsSelect& a, cudaStream_t s);
cudaError_t move_launch(const MkbsMove& m, cudaStream_t s);
cudaError_t key_weights_launch(const MkbsKeyWeights& w, cudaStream_t s);
size_t key_weights_bytes(const MkbsKeyWeights& w);

}  // namespace mkbs
