// Cache rows and states of sequences, moved in place: slots that take another slot's, and a cache cut to the rows that stay.
#include "hybrid_common.cuh"
#include "sequence_kernels.h"

namespace mkbs {
namespace {

// ---- x[slot] <- x[parents[slot]] ---------------------------------------------------------- //
// A block takes one run of bytes of all slots at once: it reads what other slots take into shared memory, each source once
// however many take it, and writes it when all of it is there.  Runs do not overlap, so no slot loses what another still needs.
constexpr int kReorderThreads = 512, kReorderBytes = 96 * 1024;

struct ReorderArgs {
    int slots, num_regions, first;
    const int32_t *parents, *lengths;
    MkbsRegion regions[MKBS_MAX_REGIONS];
};

template <typename V>
__global__ void __launch_bounds__(kReorderThreads) reorder_kernel(const __grid_constant__ ReorderArgs a) {
    extern __shared__ uint4 raw[];
    __shared__ int parent[MKBS_MAX_SLOTS], length[MKBS_MAX_SLOTS], place[MKBS_MAX_SLOTS], source[MKBS_MAX_SLOTS], sources, longest;
    const int t = threadIdx.x;
    V* const kept = reinterpret_cast<V*>(raw);
    if (t == 0) sources = longest = 0;
    for (int s = t; s < a.slots; s += kReorderThreads) {
        const int p = a.parents[s];
        parent[s] = p >= 0 && p < a.slots ? p : s;
        length[s] = a.lengths != nullptr ? max(a.lengths[s], 0) : 1 << 30;
        place[s] = -1;
    }
    __syncthreads();
    for (int s = t; s < a.slots; s += kReorderThreads) {
        if (parent[s] == s || length[parent[s]] <= a.first) continue;
        place[parent[s]] = 0;  // (several write the same)
    }
    __syncthreads();
    for (int s = t; s < a.slots; s += kReorderThreads) {
        if (place[s] < 0) continue;
        place[s] = atomicAdd(&sources, 1);
        source[place[s]] = s;
        atomicMax(&longest, length[s]);
    }
    __syncthreads();
    if (sources == 0) return;
    const int run = kReorderBytes / sources / 128 * 128;  // bytes of a slot in a step
    int64_t step = blockIdx.x;
    for (int r = 0; r < a.num_regions; ++r) {
        const MkbsRegion& g = a.regions[r];
        const int64_t from = (int64_t)a.first * g.row_bytes, to = (int64_t)min(longest, g.rows) * g.row_bytes;
        const int64_t runs = to > from ? (to - from + run - 1) / run : 0;
        for (; step < runs * g.outer; step += gridDim.x) {
            char* const base = static_cast<char*>(g.base) + step / runs * g.outer_stride;
            const int64_t begin = from + step % runs * run;
            auto units = [&](int slot) {  // of the run that the slot holds
                const int64_t end = (int64_t)min(length[slot], g.rows) * g.row_bytes;
                return (int)(max((int64_t)0, min((int64_t)run, end - begin)) / (int64_t)sizeof(V));
            };
            const int per = run / (int)sizeof(V);
            for (int i = t; i < sources * per; i += kReorderThreads) {
                const int n = i / per, u = i - n * per;
                if (u < units(source[n])) kept[i] = reinterpret_cast<const V*>(base + source[n] * g.slot_stride + begin)[u];
            }
            __syncthreads();
            for (int s = 0; s < a.slots; ++s) {
                const int p = parent[s];
                if (p == s || place[p] < 0) continue;
                const int n = units(p);
                V* const out = reinterpret_cast<V*>(base + s * g.slot_stride + begin);
                for (int u = t; u < n; u += kReorderThreads) out[u] = kept[place[p] * per + u];
            }
            __syncthreads();
        }
        step -= runs * g.outer;
    }
}

// ---- which rows stay ------------------------------------------------------------------------ //
// A block per layer, sequence and head.  The weight of the last row that stays is found digit by digit (11, 11 and 10 bits
// of its order) by counting; rows of that very weight stay in the order of their places.
constexpr int kSelectThreads = 1024, kDigits = 2048;


__device__ __forceinline__ int block_scan(int v, int* warps, int* total) {  // exclusive; kSelectThreads threads
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += n;
    }
    if (lane == 31) warps[warp] = sum;
    __syncthreads();
    if (warp == 0) {
        int w = warps[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int n = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += n;
        }
        warps[lane] = w;
    }
    __syncthreads();
    *total = warps[31];
    const int before = (warp ? warps[warp - 1] : 0) + sum - v;
    __syncthreads();
    return before;
}

__global__ void __launch_bounds__(kSelectThreads) select_kernel(const MkbsSelect s) {
    __shared__ int count[kDigits], warps[32], found[2];
    const int t = threadIdx.x, head = blockIdx.x, b = blockIdx.y, layer = blockIdx.z;
    const int n = length_of(s.lengths, s.length, s.positions, b), kept = min(n, s.keep);
    const int64_t at = layer * s.w_layer + b * s.w_sequence + head * s.w_head;
    const float* const w = s.weights + at;
    float* const kept_w = s.kept != nullptr ? s.kept + at : nullptr;
    int32_t* const rows = s.rows + (((int64_t)layer * s.sequences + b) * s.kv_heads + head) * s.keep;
    for (int r = kept + t; r < s.keep; r += kSelectThreads) rows[r] = -1;
    // not a number: the order of minus infinity
    auto order = [&](int j) { return order_of(fmaxf(w[j], -INFINITY)); };
    const int lo = n > s.keep ? s.sinks : n, hi = n > s.keep ? n - s.recent : n;  // rows that compete
    int need = s.keep - s.sinks - s.recent;
    uint32_t limit = 0;
    int shift = 32;
    if (n > s.keep && need > 0) {
        for (const int bits : {11, 11, 10}) {
            shift -= bits;
            for (int d = t; d < kDigits; d += kSelectThreads) count[d] = 0;
            __syncthreads();
            const uint32_t above = shift + bits == 32 ? 0 : limit >> (shift + bits);
            for (int j = lo + t; j < hi; j += kSelectThreads) {
                const uint32_t o = order(j);
                if (shift + bits == 32 || o >> (shift + bits) == above) atomicAdd(&count[o >> shift & ((1 << bits) - 1)], 1);
            }
            __syncthreads();
            // digits from the largest down: two per thread
            const int d = kDigits - 1 - 2 * t, c0 = count[d], c1 = count[d - 1];
            int total;
            const int before = block_scan(c0 + c1, warps, &total);
            if (before < need && need <= before + c0) found[0] = d, found[1] = before;
            if (before + c0 < need && need <= before + c0 + c1) found[0] = d - 1, found[1] = before + c0;
            __syncthreads();
            limit |= (uint32_t)found[0] << shift;
            need -= found[1];  // of this weight's digits so far
            __syncthreads();
        }
    }
    // rows above the limit, and the first `need` rows at it
    int out = 0, ties = 0;
    for (int j0 = 0; j0 < n; j0 += kSelectThreads) {
        const int j = j0 + t;
        const bool there = j < n, competes = j >= lo && j < hi;
        const float x = there ? w[j] : 0.f;
        const uint32_t o = order_of(fmaxf(x, -INFINITY));
        const bool tie = there && competes && o == limit;
        int tied, total;
        const int tie_rank = ties + block_scan(tie, warps, &tied);
        const bool stays = there && (!competes || (need > 0 && (o > limit || (tie && tie_rank < need))));
        const int to = out + block_scan(stays, warps, &total);  // (all of this step's weights have been read)
        if (stays) {
            rows[to] = j;
            if (kept_w != nullptr) kept_w[to] = x;
        }
        out += total;
        ties += tied;
    }
}

// ---- rows that stay, to the front ------------------------------------------------------------ //
// A block takes one head's rows of one cache in their order, some at a time: all of them are in registers before the first is
// written, and later rows come from behind what has been written.
constexpr int kMoveThreads = 256, kMoveAhead = 4;

__global__ void __launch_bounds__(kMoveThreads) move_kernel(const MkbsMove m) {
    const int lanes = m.head_bytes / 16, head = blockIdx.x / 2, which = blockIdx.x & 1, b = blockIdx.y, layer = blockIdx.z;
    if (m.caches[which] == nullptr) return;
    const int n = length_of(m.lengths, m.length, m.positions, b), kept = min(n, m.keep);
    const int32_t* const rows = m.rows + (((int64_t)layer * m.sequences + b) * m.kv_heads + head) * m.keep;
    const int per = kMoveThreads / lanes, mine = threadIdx.x / lanes, u = threadIdx.x - mine * lanes;
    const int64_t row_bytes = (int64_t)m.kv_heads * m.head_bytes;
    char* const base = static_cast<char*>(m.caches[which]) + layer * m.c_layer + b * m.c_sequence + (int64_t)head * m.head_bytes + u * 16;
    for (int r0 = 0; r0 < kept; r0 += per * kMoveAhead) {
        uint4 x[kMoveAhead];
        bool moves[kMoveAhead];
#pragma unroll
        for (int i = 0; i < kMoveAhead; ++i) {
            const int r = r0 + i * per + mine, from = mine < per && r < kept ? rows[r] : -1;
            moves[i] = from >= 0 && from < n && from != r;
            if (moves[i]) x[i] = *reinterpret_cast<const uint4*>(base + from * row_bytes);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kMoveAhead; ++i)
            if (moves[i]) *reinterpret_cast<uint4*>(base + (r0 + i * per + mine) * row_bytes) = x[i];
        __syncthreads();
    }
}

template <typename V>
cudaError_t reorder(const ReorderArgs& a, cudaStream_t s) {
    if (const cudaError_t e = allow_shared_memory<reorder_kernel<V>>(); e != cudaSuccess) return e;
    reorder_kernel<V><<<2 * kSms, kReorderThreads, kReorderBytes, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t reorder_launch(const MkbsReorder& r, cudaStream_t s) {
    ReorderArgs a{r.slots, r.num_regions, r.first, r.parents, r.lengths, {}};
    uintptr_t bits = 0;  // what every address and size is a multiple of
    for (int i = 0; i < r.num_regions; ++i) {
        const MkbsRegion& g = a.regions[i] = r.regions[i];
        bits |= reinterpret_cast<uintptr_t>(g.base) | (uintptr_t)g.outer_stride | (uintptr_t)g.slot_stride | (uintptr_t)g.row_bytes;
    }
    return bits % 16 == 0 ? reorder<uint4>(a, s) : bits % 4 == 0 ? reorder<uint32_t>(a, s) : reorder<uint8_t>(a, s);
}

cudaError_t select_launch(const MkbsSelect& a, cudaStream_t s) {
    select_kernel<<<dim3(a.kv_heads, a.sequences, a.layers), kSelectThreads, 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t move_launch(const MkbsMove& m, cudaStream_t s) {
    move_kernel<<<dim3(2 * m.kv_heads, m.sequences, m.layers), kMoveThreads, 0, s>>>(m);
    return cudaGetLastError();
}

}  // namespace mkbs
