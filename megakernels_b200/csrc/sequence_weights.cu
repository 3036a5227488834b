// The softmax weight that a run of queries gives each cached key, summed over the queries and the heads that share the key:
//   w[j] += sum_r exp(z_rj - log sum_i exp z_ri),  z = scale q k,  r = (query, head of the group).
// Three launches: maxima and sums of every row over tiles of keys; a row's log sum from its tiles'; the scores again, for
// the sum over a key's rows.  FMA in 32 bits.
#include "hybrid_common.cuh"
#include "sequence_kernels.h"

namespace mkbs {
namespace {

constexpr int kTile = 64, kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

struct WeightArgs {
    MkbsKeyWeights w;
    int per, rows, tiles;  // query heads of a key, rows of a key/value head, tiles of keys
    float2* parts;         // [item][row][tile]: maximum, sum (logarithms to base 2)
    float* log_sums;       // [item][row]
};

// Scores of rows r0.. and keys j0.. in base 2: thread (ty, tx) has rows ty + 16 i and keys tx + 16 k.
template <int D>
__device__ __forceinline__ void tile_scores(const WeightArgs& a, int layer, int b, int g, int r0, int j0, float (*q)[D + 1], float (*k)[D + 1], float (&z)[4][4]) {
    const bf16* const qs = static_cast<const bf16*>(a.w.q) + layer * a.w.q_layer + b * a.w.q_sequence;
    const bf16* const ks = static_cast<const bf16*>(a.w.k) + layer * a.w.k_layer + b * a.w.k_sequence;
    __syncthreads();
    for (int i = threadIdx.x; i < kTile * D; i += kThreads) {
        const int n = i / D, d = i % D, r = r0 + n, j = j0 + n;
        q[n][d] = r < a.rows ? __bfloat162float(qs[((int64_t)(r / a.per) * a.w.heads + g * a.per + r % a.per) * D + d]) : 0.f;
        k[n][d] = j < a.w.positions ? __bfloat162float(ks[((int64_t)j * a.w.kv_heads + g) * D + d]) : 0.f;
    }
    __syncthreads();
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) z[i][c] = 0.f;
    for (int d = 0; d < D; ++d) {
        float x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = q[ty + 16 * i][d], y[i] = k[tx + 16 * i][d];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) z[i][c] = fmaf(x[i], y[c], z[i][c]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) z[i][c] *= a.w.scale * kLog2e;
}

template <int D>
__global__ void __launch_bounds__(kThreads) stats_kernel(const WeightArgs a) {
    extern __shared__ float smem[];
    auto q = reinterpret_cast<float (*)[D + 1]>(smem), k = q + kTile;
    const int item = blockIdx.z, g = item % a.w.kv_heads, b = item / a.w.kv_heads % a.w.sequences, layer = item / a.w.kv_heads / a.w.sequences;
    const int n = length_of(a.w.lengths, a.w.length, a.w.positions, b), r0 = blockIdx.y * kTile, j0 = blockIdx.x * kTile;
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    float z[4][4];
    if (j0 < n) tile_scores<D>(a, layer, b, g, r0, j0, q, k, z);
    for (int i = 0; i < 4; ++i) {
        const int r = r0 + ty + 16 * i, last = n - a.w.queries + r / a.per;
        float top = -INFINITY, sum = 0.f;
        if (j0 < n) {
            for (int c = 0; c < 4; ++c)
                if (j0 + tx + 16 * c <= last) top = fmaxf(top, z[i][c]);
            for (int o = 8; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            for (int c = 0; c < 4; ++c)
                if (j0 + tx + 16 * c <= last) sum += exp2f(z[i][c] - top);
            for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        if (tx == 0 && r < a.rows) a.parts[((int64_t)item * a.rows + r) * a.tiles + blockIdx.x] = make_float2(top, sum);
    }
}

__global__ void __launch_bounds__(kThreads) log_sum_kernel(const WeightArgs a) {
    const int64_t row = (int64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
    if (row >= (int64_t)a.w.layers * a.w.sequences * a.w.kv_heads * a.rows) return;
    const float2* const parts = a.parts + row * a.tiles;
    float top = -INFINITY, sum = 0.f;
    for (int i = threadIdx.x % 32; i < a.tiles; i += 32) top = fmaxf(top, parts[i].x);
    top = mkbh::warp_max(top);
    for (int i = threadIdx.x % 32; i < a.tiles; i += 32)
        if (parts[i].x > -INFINITY) sum += parts[i].y * exp2f(parts[i].x - top);
    sum = mkbh::warp_sum(sum);
    if (threadIdx.x % 32 == 0) a.log_sums[row] = sum > 0.f ? top + log2f(sum) : INFINITY;  // (a row that sees no key)
}

template <int D>
__global__ void __launch_bounds__(kThreads) weights_kernel(const WeightArgs a) {
    extern __shared__ float smem[];
    auto q = reinterpret_cast<float (*)[D + 1]>(smem), k = q + kTile;
    const int item = blockIdx.y, g = item % a.w.kv_heads, b = item / a.w.kv_heads % a.w.sequences, layer = item / a.w.kv_heads / a.w.sequences;
    const int n = length_of(a.w.lengths, a.w.length, a.w.positions, b), j0 = blockIdx.x * kTile;
    if (j0 >= n) return;
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int r0 = 0; r0 < a.rows; r0 += kTile) {
        float z[4][4];
        tile_scores<D>(a, layer, b, g, r0, j0, q, k, z);
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + ty + 16 * i, last = n - a.w.queries + r / a.per;
            if (r >= a.rows) continue;
            const float off = a.log_sums[(int64_t)item * a.rows + r];
            for (int c = 0; c < 4; ++c)
                if (j0 + tx + 16 * c <= last) sum[c] += exp2f(z[i][c] - off);
        }
    }
    __syncthreads();
    for (int c = 0; c < 4; ++c) smem[ty * kTile + tx + 16 * c] = sum[c];
    __syncthreads();
    const int j = j0 + threadIdx.x;
    if (threadIdx.x >= kTile || j >= n) return;
    float total = 0.f;
    for (int i = 0; i < 16; ++i) total += smem[i * kTile + threadIdx.x];
    a.w.weights[layer * a.w.w_layer + b * a.w.w_sequence + g * a.w.w_head + j] += total;
}

WeightArgs plan(const MkbsKeyWeights& w, size_t* bytes) {
    const int per = w.heads / w.kv_heads, rows = w.queries * per, tiles = (w.positions + kTile - 1) / kTile;
    const size_t all = (size_t)w.layers * w.sequences * w.kv_heads * rows;
    *bytes = all * tiles * 8 + all * 4;
    char* const base = static_cast<char*>(w.workspace);
    return {w, per, rows, tiles, reinterpret_cast<float2*>(base), reinterpret_cast<float*>(base + all * tiles * 8)};
}

template <int D>
cudaError_t launch(const WeightArgs& a, cudaStream_t s) {
    const int items = a.w.layers * a.w.sequences * a.w.kv_heads, smem = 2 * kTile * (D + 1) * 4;
    cudaError_t e;
    if ((e = cudaFuncSetAttribute(stats_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return e;
    if ((e = cudaFuncSetAttribute(weights_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return e;
    stats_kernel<D><<<dim3(a.tiles, (a.rows + kTile - 1) / kTile, items), kThreads, smem, s>>>(a);
    log_sum_kernel<<<(unsigned)(((int64_t)items * a.rows + kThreads / 32 - 1) / (kThreads / 32)), kThreads, 0, s>>>(a);
    weights_kernel<D><<<dim3(a.tiles, items), kThreads, smem, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

size_t key_weights_bytes(const MkbsKeyWeights& w) {
    size_t bytes;
    plan(w, &bytes);
    return bytes;
}

cudaError_t key_weights_launch(const MkbsKeyWeights& w, cudaStream_t s) {
    size_t bytes;
    const WeightArgs a = plan(w, &bytes);
    return w.dim == 64 ? launch<64>(a, s) : launch<128>(a, s);
}

}  // namespace mkbs
