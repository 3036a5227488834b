// Beam search's selection: the k best of a group's beams * vocab continuations.
//
// The score of continuation (b, v) is c_b + (l_bv - top_b) - log sum_v exp(l_bv - top_b); within a beam it grows with
// the logit.  So the order of whole segments of a beam's vocabulary by their largest logit says which of them can hold
// one of the k best: a segment behind k others has k better continuations before it.  That gives two launches:
//   scan   reads every logit once: the maximum of every segment, and per warp the maximum and sum of exponentials of a
//          run of segments;
//   merge  a block per group: the log sums, the k best segments of all beams, and of their elements (still in L2)
//          the k best.
// Both selections are knock-outs: candidates fall into a few hundred groups by thread, the groups' best ones are ranked by
// counting, the members of the k best groups go into the next round.  A candidate is a 64-bit key and its index, which are
// never equal (what is no candidate has the key 0 and comes last), so every round is exact, ties included.
#include "hybrid_common.cuh"
#include "sequence_kernels.h"

namespace mkbs {
namespace {

constexpr int kBlockElems = 256;  // elements that a warp reads at a time
constexpr int kScanWarps = 8;
constexpr int kMergeThreads = 1024;
constexpr float kLog2e = 1.4426950408889634f;

struct BeamPlan {
    int rows, segment, segments, per_warp, parts;  // elements per segment; segments, segments per warp and warps of a row
    int level1, level2;                            // candidates: all segments, the elements of k of them
    int groups_ranked, list_a, list_b;             // groups per round, entries of the two lists
    size_t part_offset, bytes;
    explicit BeamPlan(const MkbsBeams& b) {
        rows = b.groups * b.beams;
        const int64_t span = b.vocab + 15;  // (a row may start anywhere in 16 bytes)
        // as many segments as the chosen ones have elements, at least 256
        for (segment = kBlockElems; (int64_t)b.beams * ((span + segment - 1) / segment) > 2 * (int64_t)b.k * segment; segment *= 2) {
        }
        segments = (int)((span + segment - 1) / segment);
        // two blocks' worth of warps per SM before a warp takes a second segment
        per_warp = (int)(((int64_t)rows * segments + kSms * 16 - 1) / (kSms * 16));
        parts = (segments + per_warp - 1) / per_warp;
        level1 = b.beams * segments;
        level2 = (level1 < b.k ? level1 : b.k) * segment;
        for (groups_ranked = 64; groups_ranked < 4 * b.k; groups_ranked *= 2) {
        }
        const int most = level1 > level2 ? level1 : level2;
        list_a = next(most, b.k);
        list_b = next(list_a, b.k);
        part_offset = ((size_t)rows * segments * 4 + 255) / 256 * 256;
        bytes = part_offset + (size_t)rows * parts * 8;
    }
    int next(int m, int k) const {  // entries of the next round
        if (m <= groups_ranked) return 0;
        return k * (m <= kMergeThreads ? (m + groups_ranked - 1) / groups_ranked : (m + kMergeThreads - 1) / kMergeThreads * (kMergeThreads / groups_ranked));
    }
    size_t merge_smem() const { return (size_t)(list_a + list_b + groups_ranked) * 12 + (size_t)groups_ranked * 4 + MKBS_MAX_BEST * 4 + MKBS_MAX_BEAMS * 24 + 16; }
};

struct BeamArgs {
    int beams, vocab, k, segment, segments, per_warp, parts, groups_ranked, list_a, list_b;
    int64_t row_stride;
    const void* logits;
    const float* scores;
    const uint8_t* done;
    int eos;
    uint32_t* tops;  // [rows][segments]: order_of of the largest logit
    float2* sums;    // [rows][parts]: maximum, sum of exponentials
    float* out_scores;
    int32_t *out_parents, *out_tokens;
    uint8_t* out_done;
};

// Elements between the 16-byte boundary before a row and the row.
template <typename T>
__device__ __forceinline__ int shift_of(const T* row) { return (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T)); }

__device__ __forceinline__ bool is_live(float c) { return c > -INFINITY && c < INFINITY; }

// The lane's elements of a block: a lane holds 8 bf16 or twice 4 floats next to each other.  Not a number and what lies
// outside the row is minus infinity.
template <typename T>
__device__ __forceinline__ void load_elems(const T* base, int p, int shift, int end, float (&x)[8]) {
    constexpr int n = 16 / sizeof(T);
#pragma unroll
    for (int v = 0; v < 8 / n; ++v) {
        const int at = p + v * kBlockElems / 2;
        if (at >= shift && at + n <= end) {
            const uint4 w = mkb::ld_nc_v4(base + at);
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 2) {
                    x[2 * i] = mkb::bf16_lo(words[i]);
                    x[2 * i + 1] = mkb::bf16_hi(words[i]);
                } else {
                    x[4 * v + i] = __uint_as_float(words[i]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < n; ++i) x[n * v + i] = at + i >= shift && at + i < end ? mkbh::to_f<T>(base[at + i]) : -INFINITY;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaxf(x[i], -INFINITY);
}

template <typename T>
__global__ void __launch_bounds__(32 * kScanWarps) beam_scan_kernel(const BeamArgs a) {
    mkbh::let_next();
    constexpr int kAhead = 4;  // blocks whose loads are under way together
    const int lane = threadIdx.x & 31, row = blockIdx.y, part = blockIdx.x * kScanWarps + (threadIdx.x >> 5);
    if (part >= a.parts) return;
    // beams whose continuations' scores do not depend on their logits
    if ((a.done != nullptr && a.done[row]) || (a.scores != nullptr && !is_live(a.scores[row]))) return;
    const T* const begin = static_cast<const T*>(a.logits) + row * a.row_stride;
    const int shift = shift_of(begin), end = shift + a.vocab, blocks = a.segment / kBlockElems;
    const T* const base = begin - shift;
    const int first = part * a.per_warp * blocks, last = min(first + a.per_warp * blocks, a.segments * blocks);
    constexpr int n = 16 / sizeof(T);
    float top = -INFINITY, sum = 0.f, best = -INFINITY;
    for (int at = first; at < last; at += kAhead) {
        float x[kAhead][8], high[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int p = at + u < last ? (at + u) * kBlockElems + lane * n : end;
            load_elems(base, p, shift, end, x[u]);
        }
        float most = top;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            high[u] = x[u][0];
#pragma unroll
            for (int i = 1; i < 8; ++i) high[u] = fmaxf(high[u], x[u][i]);
            most = fmaxf(most, high[u]);
        }
        if (most == INFINITY) {  // infinite logits count, the others are nothing beside them
            if (top < INFINITY) sum = 0.f;
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += x[u][i] == INFINITY ? 1.f : 0.f;
        } else if (most > -INFINITY) {
            sum *= exp2f((top - most) * kLog2e);  // (0 from minus infinity)
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                float part_sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) part_sum += exp2f((x[u][i] - most) * kLog2e);
                sum += part_sum;
            }
        }
        top = most;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (at + u >= last) break;
            best = fmaxf(best, high[u]);
            if ((at + u + 1) % blocks == 0) {
                const uint32_t order = __reduce_max_sync(0xffffffffu, order_of(best));
                if (lane == 0) a.tops[(size_t)row * a.segments + (at + u) / blocks] = order;
                best = -INFINITY;
            }
        }
    }
    const float most = value_of(__reduce_max_sync(0xffffffffu, order_of(top)));
    const float factor = top == most ? 1.f : exp2f((top - most) * kLog2e);
    sum = mkbh::warp_sum(top > -INFINITY ? sum * factor : 0.f);
    if (lane == 0) a.sums[(size_t)row * a.parts + part] = make_float2(most, sum);
}

__device__ __forceinline__ uint64_t order64(double x) {
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
    return b ^ ((b >> 63) ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double value64(uint64_t order) { return __longlong_as_double((long long)(order ^ ((order >> 63) ? 1ull << 63 : ~0ull))); }

struct Candidate {
    uint64_t key;  // 0: none
    uint32_t at;
    __device__ __forceinline__ bool before(const Candidate& o) const { return key > o.key || (key == o.key && at < o.at); }
};

struct MergeSmem {
    uint64_t *key_a, *key_b, *group_key;
    double *log_sum, *start;
    uint32_t *at_a, *at_b, *group_at;
    int *rank, *chosen;
    float* top;
    __device__ MergeSmem(void* raw, int list_a, int list_b, int groups) {
        key_a = static_cast<uint64_t*>(raw);
        key_b = key_a + list_a;
        group_key = key_b + list_b;
        log_sum = reinterpret_cast<double*>(group_key + groups);
        start = log_sum + MKBS_MAX_BEAMS;
        at_a = reinterpret_cast<uint32_t*>(start + MKBS_MAX_BEAMS);
        at_b = at_a + list_a;
        group_at = at_b + list_b;
        rank = reinterpret_cast<int*>(group_at + groups);
        chosen = rank + groups;
        top = reinterpret_cast<float*>(chosen + MKBS_MAX_BEST);
    }
};

// The k first of candidates 0 .. count - 1; `take(rank, candidate)` is called for each of them by some thread.
template <typename Get, typename Take>
__device__ __forceinline__ void knock_out(const MergeSmem& sm, int count, int k, int groups, Get get, Take take) {
    const int t = threadIdx.x, lanes = kMergeThreads / groups, group = t / lanes;
    auto rank_groups = [&]() {  // (group_key, group_at) -> rank
        for (int g = t; g < groups; g += kMergeThreads) sm.rank[g] = 0;
        __syncthreads();
        const int mine = t % groups, share = groups / lanes, from = t / groups * share;
        const Candidate own{sm.group_key[mine], sm.group_at[mine]};
        int before = 0;
#pragma unroll 4
        for (int j = from; j < from + share; ++j) before += Candidate{sm.group_key[j], sm.group_at[j]}.before(own);
        if (before) atomicAdd(&sm.rank[mine], before);
        __syncthreads();
    };
    bool in_a = false, listed = false;
    auto candidate = [&](int i) {
        if (!listed) return get(i);
        return in_a ? Candidate{sm.key_a[i], sm.at_a[i]} : Candidate{sm.key_b[i], sm.at_b[i]};
    };
    while (count > groups) {
        // Candidates of a thread: t, t + 1024, ...; of few candidates one that leaves no group empty
        const bool few = count <= kMergeThreads;
        const int turns = few ? 1 : (count + kMergeThreads - 1) / kMergeThreads, members = few ? (count + groups - 1) / groups : turns * lanes;
        const int first = few ? t % lanes * groups + group : t;
        Candidate best{0, 0x80000000u};
        for (int i = first; i < count; i += kMergeThreads) {
            const Candidate c = candidate(i);
            if (c.before(best)) best = c;
        }
        for (int o = lanes / 2; o; o >>= 1) {
            const Candidate c{__shfl_xor_sync(0xffffffffu, best.key, o), __shfl_xor_sync(0xffffffffu, best.at, o)};
            if (c.before(best)) best = c;
        }
        if (t % lanes == 0) sm.group_key[group] = best.key, sm.group_at[group] = best.key ? best.at : 0x80000000u + group;
        __syncthreads();
        rank_groups();
        const int place = sm.rank[group];
        uint64_t* const key = in_a ? sm.key_b : sm.key_a;
        uint32_t* const at = in_a ? sm.at_b : sm.at_a;
        if (place < k) {
            for (int n = 0; n < turns; ++n) {
                const int i = first + n * kMergeThreads, member = n * lanes + t % lanes;
                if (member >= members) continue;
                const Candidate c = i < count ? candidate(i) : Candidate{0, 0};
                key[place * members + member] = c.key;
                at[place * members + member] = c.at;
            }
        }
        count = k * members;
        in_a = !in_a;
        listed = true;
        __syncthreads();
    }
    if (t < groups) {
        const Candidate c = t < count ? candidate(t) : Candidate{0, 0x80000000u + t};
        sm.group_key[t] = c.key;
        sm.group_at[t] = c.key ? c.at : 0x80000000u + t;  // (what is none is behind all others, and no two alike)
    }
    __syncthreads();
    rank_groups();
    if (t < groups && sm.rank[t] < k) take(sm.rank[t], Candidate{sm.group_key[t], sm.group_at[t]});
    __syncthreads();
}

enum Kind { kLive = 0, kDone = 1, kDead = 2 };  // kDead: every continuation has score minus infinity

template <typename T>
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const BeamArgs a) {
    extern __shared__ uint64_t raw[];
    const MergeSmem sm(raw, a.list_a, a.list_b, a.groups_ranked);
    __shared__ int kind[MKBS_MAX_BEAMS];
    const int group = blockIdx.x, row0 = group * a.beams, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    mkbh::after_previous();
    for (int b = warp; b < a.beams; b += kMergeThreads / 32) {
        const int row = row0 + b;
        const float c = a.scores != nullptr ? a.scores[row] : 0.f;
        int what = !is_live(c) ? kDead : a.done != nullptr && a.done[row] ? kDone : kLive;
        if (what == kLive) {
            const float2* const sums = a.sums + (size_t)row * a.parts;
            float top = -INFINITY;
            for (int i = lane; i < a.parts; i += 32) top = fmaxf(top, sums[i].x);
            top = mkbh::warp_max(top);
            double sum = 0.0;
            for (int i = lane; i < a.parts; i += 32) {
                const float2 part = sums[i];
                if (part.x == top) sum += part.y;
                else if (part.x > -INFINITY) sum += part.y * exp((double)part.x - (double)top);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (top == -INFINITY) what = kDead;
            if (lane == 0) sm.top[b] = top, sm.log_sum[b] = log(sum);
        }
        if (lane == 0) kind[b] = what, sm.start[b] = c;
    }
    __syncthreads();
    const uint64_t lowest = order64(-(double)INFINITY);
    auto key_of = [&](int b, float x) {
        const double d = x == sm.top[b] ? 0.0 : (double)x - (double)sm.top[b];
        return x == -INFINITY ? lowest : order64(sm.start[b] + (d - sm.log_sum[b]));
    };
    auto row_of = [&](int b) { return static_cast<const T*>(a.logits) + (row0 + b) * a.row_stride; };
    const int segments = a.segments, count = a.beams * segments;
    knock_out(sm, count, a.k, a.groups_ranked, [&](int i) {
        const int b = i / segments, s = i - b * segments, shift = shift_of(row_of(b));
        if (s * a.segment >= shift + a.vocab) return Candidate{0, (uint32_t)i};
        if (kind[b] == kLive) return Candidate{key_of(b, value_of(a.tops[(size_t)(row0 + b) * segments + s])), (uint32_t)i};
        const bool ends = kind[b] == kDone && (a.eos + shift) / a.segment == s;
        return Candidate{ends ? order64(sm.start[b]) : lowest, (uint32_t)i};
    }, [&](int rank, const Candidate& c) { sm.chosen[rank] = c.key ? (int)c.at : -1; });
    const int chosen = min(a.k, count);
    knock_out(sm, chosen * a.segment, a.k, a.groups_ranked, [&](int i) {
        const int at = sm.chosen[i / a.segment];
        if (at < 0) return Candidate{0, 0};
        const int b = at / segments, s = at - b * segments;
        const T* const row = row_of(b);
        const int v = s * a.segment + i % a.segment - shift_of(row);
        if (v < 0 || v >= a.vocab) return Candidate{0, 0};
        const uint32_t flat = (uint32_t)b * a.vocab + v;
        if (kind[b] == kLive) return Candidate{key_of(b, fmaxf(mkbh::to_f<T>(row[v]), -INFINITY)), flat};
        return Candidate{kind[b] == kDone && v == a.eos ? order64(sm.start[b]) : lowest, flat};
    }, [&](int rank, const Candidate& c) {
        const int b = c.at / a.vocab, v = c.at - b * a.vocab, to = group * a.k + rank;
        a.out_scores[to] = (float)value64(c.key);
        a.out_parents[to] = row0 + b;
        a.out_tokens[to] = v;
        if (a.out_done != nullptr) a.out_done[to] = v == a.eos || (a.done != nullptr && a.done[row0 + b]);
    });
}

template <typename T>
cudaError_t launch(const BeamPlan& p, const MkbsBeams& b, const BeamArgs& a, cudaStream_t s) {
    const size_t smem = p.merge_smem();
    if (smem > 48 * 1024) {
        const cudaError_t e = allow_shared_memory<beam_merge_kernel<T>>();
        if (e != cudaSuccess) return e;
    }
    beam_scan_kernel<T><<<dim3((p.parts + kScanWarps - 1) / kScanWarps, p.rows), 32 * kScanWarps, 0, s>>>(a);
    if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(b.groups);
    c.blockDim = dim3(kMergeThreads);
    c.dynamicSmemBytes = smem;
    c.stream = s;
    cudaLaunchAttribute early = mkbh::may_begin_early();
    c.attrs = &early;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, beam_merge_kernel<T>, a);
}

}  // namespace

size_t beam_bytes(const MkbsBeams& b) { return BeamPlan(b).bytes; }

cudaError_t beam_launch(const MkbsBeams& b, cudaStream_t s) {
    const BeamPlan p(b);
    char* const work = static_cast<char*>(b.workspace);
    const BeamArgs a{b.beams, b.vocab, b.k, p.segment, p.segments, p.per_warp, p.parts, p.groups_ranked, p.list_a, p.list_b, b.row_stride, b.logits, b.scores,
                     b.done, b.eos, reinterpret_cast<uint32_t*>(work), reinterpret_cast<float2*>(work + p.part_offset), b.out_scores, b.out_parents,
                     b.out_tokens, b.out_done};
    return b.dtype == MKBS_F32 ? launch<float>(p, b, a, s) : launch<bf16>(p, b, a, s);
}

}  // namespace mkbs
