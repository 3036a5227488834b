// Launchers of the operators between two decoding steps (one translation unit per group); arguments have been checked.
#pragma once
#include <algorithm>
#include <atomic>
#include <initializer_list>
#include <memory>
#include <new>
#include <utility>

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/mkb200_sequences.h"

namespace mkbs {

using bf16 = __nv_bfloat16;

constexpr int kSms = 148;  // what grids and splits are sized by
constexpr int kStaticShared = 16 * 1024;  // most that a kernel has besides

// Total order of floats as whole numbers; 0 is below all of them.  Minus zero counts as zero.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t order) { return __uint_as_float(order ^ ((order >> 31) ? 0x80000000u : 0xffffffffu)); }

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Rows that sequence `b` holds.
__device__ __forceinline__ int length_of(const int32_t* lengths, int length, int positions, int b) {
    return min(max(lengths != nullptr ? __ldg(lengths + b) : length, 0), positions);
}

// Lets `kernel` have all of an SM's shared memory, once per device.
template <auto kernel>
inline cudaError_t allow_shared_memory() {
    static std::atomic<bool> set[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || set[dev & 63].load(std::memory_order_relaxed)) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - kStaticShared);
    if (e == cudaSuccess) set[dev & 63].store(dev < 64, std::memory_order_relaxed);
    return e;
}

// Whether blocks of `size` are apart that begin at i s[0] + j s[1] + k s[2], i below n[0] and so on (s, of a dimension of one: anything).
inline bool apart(int64_t size, std::initializer_list<std::pair<int64_t, int64_t>> dims) {
    std::pair<int64_t, int64_t> d[3];  // (stride, count)
    int m = 0;
    int64_t blocks = 1;
    for (const auto& [n, s] : dims) {
        if (n < 2) continue;
        if (s < size) return false;
        d[m++] = {s, n};
        blocks *= n;
    }
    std::sort(d, d + m);
    int64_t extent = size;
    bool nested = true;  // each stride steps over all that the smaller ones reach: the usual case
    for (int i = 0; i < m; ++i) {
        nested = nested && d[i].first >= extent;
        extent += d[i].first * (d[i].second - 1);
    }
    if (nested || m < 2) return nested;
    if (blocks > 1 << 24) return false;  // (interleaved: every block is looked at)
    const std::unique_ptr<int64_t[]> at(new (std::nothrow) int64_t[blocks]);
    if (!at) return false;
    int64_t have = 1;
    at[0] = 0;
    for (int i = 0; i < m; ++i) {
        for (int64_t j = have; j < have * d[i].second; ++j) at[j] = at[j - have] + d[i].first;
        have *= d[i].second;
    }
    std::sort(at.get(), at.get() + blocks);
    for (int64_t j = 1; j < blocks; ++j)
        if (at[j] - at[j - 1] < size) return false;
    return true;
}

cudaError_t beam_launch(const MkbsBeams& b, cudaStream_t s);
size_t beam_bytes(const MkbsBeams& b);
cudaError_t reorder_launch(const MkbsReorder& r, cudaStream_t s);
cudaError_t select_launch(const MkbsSelect& a, cudaStream_t s);
cudaError_t move_launch(const MkbsMove& m, cudaStream_t s);
cudaError_t key_weights_launch(const MkbsKeyWeights& w, cudaStream_t s);
size_t key_weights_bytes(const MkbsKeyWeights& w);

}  // namespace mkbs
