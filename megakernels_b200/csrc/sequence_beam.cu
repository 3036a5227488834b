// Beam search's selection: the k best of a group's beams * vocab continuations.
//
// The score of continuation (b, v) is c_b + (l_bv - top_b) - log sum_v exp(l_bv - top_b); within a beam it grows with
// the logit.  So the order of whole segments of a beam's vocabulary by their largest logit says which of them can hold
// one of the k best: a segment behind k others has k better continuations before it.  That gives two launches:
//   scan   reads every logit once: the maximum of every segment, and per block the maximum and sum of exponentials of a
//          run of segments;
//   merge  a block per group: the log sums, the k best segments of all beams, and of their elements (still in L2)
//          the k best.
// Both selections go through the candidates' scores in fp32 first: a lower bound of the k-th best is the k-th best of the segments' maxima
// over groups of threads, and what may lie above it is listed, of segments and of their elements mostly little more than k.  The listed elements'
// 64-bit scores are ranked by counting.  Where the list is too short for the elements that may lie above, they get a bound of their own; where it still is
// (equal logits, fewer than k finite scores), the selection is a knock-out: candidates fall into groups by thread, the groups' best ones are ranked by counting, the members of the k best
// groups go into the next round.  A candidate is a 64-bit key and its index, which are never equal (what is no candidate has the
// key 0 and comes last), so both are exact, ties included.
// Measured, replayed as a graph: 4 rows of 128256 bf16 8.8 us (1 MB, 0.2 at memory's rate: two dependent launches and the merge's chain
// of a dozen meetings of a block bound it), 8 groups of 8 with k = 16 17.5 us (16 MB, 2.5; the scan 8 - 9 of them, 2 TB/s).  With a second bound, for the
// elements, and one element a load 10.8 and 24.4; with segments of 256 elements there too, 9.8 and 20.6; with neighbouring segments in one group of the bound
// 16 instead of 8.8 where one of 11 beams of 5814 has most of the best (the list overflows).
#include "hybrid_common.cuh"
#include "sequence_kernels.h"

namespace mkbs {
namespace {

constexpr int kBlockElems = 256;  // elements that a warp reads at a time
constexpr int kScanWarps = 8, kAhead = 4;  // (kAhead: blocks whose loads are under way together)
constexpr int kMergeThreads = 512, kStaged = 8192, kListed = kMergeThreads;  // (kStaged: candidates whose bounds lie in shared memory)
constexpr int kCandidateBytes = 12;
constexpr size_t kMostShared = 227 * 1024 - kStaticShared;
constexpr float kLog2e = 1.4426950408889634f;

struct BeamPlan {
    int rows, segment, segments, per_warp, parts;  // elements per segment; segments of a row and of a warp, blocks of a row
    int groups, list_a, list_b, staged;            // of the merge: groups per round, entries of the two lists, bounds in shared memory
    int chosen;                                    // segments whose elements are candidates, at most
    size_t part_offset, bytes;
    explicit BeamPlan(const MkbsBeams& b) {
        lay_out(b, true);
        if (merge_smem() > kMostShared) lay_out(b, false);
    }
    // Ample: room for segments that tie, and segments so long that there are not many more of them than 16-byte loads of the chosen ones.  (Where
    // the knock-out's lists have no room beside that, as many segments as elements.)
    void lay_out(const MkbsBeams& b, bool ample) {
        rows = b.groups * b.beams;
        const int64_t span = b.vocab + 15;  // (a row may start anywhere in 16 bytes)
        chosen = ample ? b.k + b.k / 2 + 16 : b.k + b.k / 4 + 8;
        for (segment = kBlockElems; (int64_t)b.beams * ((span + segment - 1) / segment) > (int64_t)chosen * segment * 2 / (ample ? 8 : 1); segment *= 2) {
        }
        segments = (int)((span + segment - 1) / segment);
        // as few segments per warp as let all blocks run at once, three on an SM (groups of 8 rows of 128256, 8, 12 and
        // 24 of them, k = 8: with 1 block 17.1, 25.6, 30.8 us, 2 14.9, 17.6, 30.9, 3 15.3, 17.5, 25.1, 4 16.4, 19.6, 25.8)
        for (per_warp = 1; parts = (segments + per_warp * kScanWarps - 1) / (per_warp * kScanWarps), parts > 1 && (int64_t)rows * parts > 3 * kSms; ++per_warp) {
        }
        // candidates: all segments, then the elements of k of them, or of those that may be among the k
        const int level1 = b.beams * segments, level2 = (level1 < chosen ? level1 : chosen) * segment, most = level1 > level2 ? level1 : level2;
        staged = most < kStaged ? (most + 1) / 2 * 2 : kStaged;
        // (the more groups, the shorter the lists, and the longer a round's ranking)
        for (groups = 64;; groups *= 2) {
            list_a = next(most, b.k) < kListed ? kListed : (next(most, b.k) + 3) / 4 * 4;  // (16-byte numbers follow)
            list_b = (next(list_a, b.k) + 3) / 4 * 4;
            if (groups >= kMergeThreads || (groups >= 4 * b.k && merge_smem() <= kMostShared)) break;
        }
        part_offset = ((size_t)rows * segments * 4 + 255) / 256 * 256;
        bytes = part_offset + (size_t)rows * parts * 8;
    }
    int next(int m, int k) const {  // entries of the next round
        if (m <= groups) return 0;
        return k * (m <= kMergeThreads ? (m + groups - 1) / groups : (m + kMergeThreads - 1) / kMergeThreads * (kMergeThreads / groups));
    }
    size_t merge_smem() const {  // (bounds and lists take turns)
        const size_t lists = (size_t)(list_a + list_b) * kCandidateBytes, bounds = (size_t)staged * 4;
        return (lists > bounds ? lists : bounds) + (size_t)groups * (kCandidateBytes + 4) + (size_t)chosen * 16 + MKBS_MAX_BEAMS * 28 + kListed * 4;
    }
};

struct BeamArgs {
    int beams, vocab, k, segment, segments, per_warp, parts, groups, list_a, list_b, staged, chosen;
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

// 16 bytes of a row from element `at` on; what lies outside the row is minus infinity.  (Out of line: a launch fetches its code
// anew, and few vectors lie at a row's ends.)
template <typename T>
__device__ __noinline__ uint4 edge_vector(const T* base, int at, int shift, int end) {
    uint32_t words[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            words[i] = at + i >= shift && at + i < end ? __float_as_uint(base[at + i]) : 0xff800000u;
        } else {
            const uint16_t* const bits = reinterpret_cast<const uint16_t*>(base);
            const int k = at + 2 * i;
            const uint32_t low = k >= shift && k < end ? bits[k] : 0xff80u, high = k + 1 >= shift && k + 1 < end ? bits[k + 1] : 0xff80u;
            words[i] = low | high << 16;
        }
    }
    return make_uint4(words[0], words[1], words[2], words[3]);
}

// 16 bytes of minus infinity
template <typename T>
__device__ __forceinline__ uint4 none_of() {
    constexpr uint32_t word = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
    return make_uint4(word, word, word, word);
}

// The lane's elements of a block: a lane holds 8 bf16 or twice 4 floats next to each other.
template <typename T>
struct Elems {
    static constexpr int kVector = 16 / sizeof(T), kVectors = 8 / kVector;
    uint4 w[kVectors];
    __device__ __forceinline__ void load(const T* base, int block, int lane, int shift, int end) {
        const int p = block * kBlockElems + lane * kVector;
        const bool inside = block * kBlockElems >= shift && (block + 1) * kBlockElems <= end;  // (for the whole warp)
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            const int at = p + v * kBlockElems / 2;
            w[v] = inside ? mkb::ld_nc_v4(base + at) : edge_vector(base, at, shift, end);
        }
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            const uint32_t words[4] = {w[v].x, w[v].y, w[v].z, w[v].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 2) {
                    x[2 * i] = mkb::bf16_lo(words[i]);
                    x[2 * i + 1] = mkb::bf16_hi(words[i]);
                } else {
                    x[4 * v + i] = __uint_as_float(words[i]);
                }
            }
        }
    }
    // the largest; not a number is minus infinity
    __device__ __forceinline__ float most() const {
        if constexpr (sizeof(T) == 2) {
            auto pair = [](uint32_t u) { return *reinterpret_cast<const __nv_bfloat162*>(&u); };
            const __nv_bfloat162 m = __hmax2(__hmax2(pair(w[0].x), pair(w[0].y)), __hmax2(pair(w[0].z), pair(w[0].w)));
            return fmaxf(fmaxf(__low2float(m), __high2float(m)), -INFINITY);
        } else {
            float x[8];
            floats(x);
            return fmaxf(fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))), -INFINITY);
        }
    }
};

// A sum of exponentials goes with the largest logit `top` of what it sums: it is that of exp(l - top), so that the largest term is
// exactly 1, and a beam with one continuation gives it the whole probability.  What such a sum is multiplied with to go with
// `high`, which is not less:
__device__ __forceinline__ float to_top(float top, float high) { return top == high ? 1.f : fast_exp2((top - high) * kLog2e); }

// A lane's sum of elements first .. last - 1 in the general way, for logits that are infinite or no numbers.
template <typename T>
__device__ __noinline__ float general_sum(const T* base, int first, int last, int lane, float top) {
    float sum = 0.f;
#pragma unroll 4
    for (int i = first + lane; i < last; i += 32) {
        const float x = fmaxf(mkbh::to_f<T>(base[i]), -INFINITY);
        sum += x == -INFINITY ? 0.f : to_top(x, top);
    }
    return sum;
}

template <typename T>
__global__ void __launch_bounds__(32 * kScanWarps) beam_scan_kernel(const BeamArgs a) {
    __shared__ float2 shared[kScanWarps];
    mkbh::let_next();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.y;
    // beams whose continuations' scores do not depend on their logits
    if ((a.done != nullptr && a.done[row]) || (a.scores != nullptr && !is_live(a.scores[row]))) return;
    const T* const begin = static_cast<const T*>(a.logits) + row * a.row_stride;
    const int shift = shift_of(begin), end = shift + a.vocab, blocks = a.segment / kBlockElems;
    const T* const base = begin - shift;
    const int first = (blockIdx.x * kScanWarps + warp) * a.per_warp * blocks, last = min(first + a.per_warp * blocks, a.segments * blocks);
    float top = -INFINITY, sum = 0.f, best = -INFINITY;
    Elems<T> ahead[kAhead];
    auto load = [&](int at) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (at + u < last) ahead[u].load(base, at + u, lane, shift, end);
    };
    load(first);
    for (int at = first; at < last; at += kAhead) {
        Elems<T> now[kAhead];
        float most = top;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) now[u] = ahead[u];
        load(at + kAhead);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (at + u >= last) break;
            const float high = now[u].most();
            most = fmaxf(most, high);
            best = fmaxf(best, high);
            if ((at + u + 1) % blocks == 0) {
                const uint32_t order = __reduce_max_sync(0xffffffffu, order_of(best));
                if (lane == 0) a.tops[(size_t)row * a.segments + (at + u) / blocks] = order;
                best = -INFINITY;
            }
        }
        const float off = most == -INFINITY ? 0.f : most;
        sum *= fast_exp2((top - off) * kLog2e);  // (0 from minus infinity)
        top = most;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (at + u >= last) break;
            float x[8], y[2] = {0.f, 0.f};
            now[u].floats(x);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i & 1] += fast_exp2((x[i] - off) * kLog2e);
            sum += y[0] + y[1];
        }
    }
    // the lanes' and the warps' sums; a part without a finite logit has the sum 0
    const float high = value_of(__reduce_max_sync(0xffffffffu, order_of(top)));
    if (__any_sync(0xffffffffu, !(sum < INFINITY))) sum = general_sum(base, max(first * kBlockElems, shift), min(last * kBlockElems, end), lane, high);
    else if (sum > 0.f) sum *= to_top(top, high);
    sum = mkbh::warp_sum(sum);
    if (lane == 0) shared[warp] = make_float2(high, sum);
    __syncthreads();
    if (threadIdx.x == 0) {
        float most = shared[0].x, all = 0.f;
#pragma unroll
        for (int i = 1; i < kScanWarps; ++i) most = fmaxf(most, shared[i].x);
#pragma unroll 1
        for (int i = 0; i < kScanWarps; ++i) all += shared[i].y > 0.f ? shared[i].y * to_top(shared[i].x, most) : 0.f;
        a.sums[(size_t)row * a.parts + blockIdx.x] = make_float2(most, all);
    }
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
    const void** chosen_row;
    uint32_t *at_a, *at_b, *group_at, *staged, *listed;
    int *rank, *chosen_beam, *chosen_first, *kind;  // chosen_first: what the segment's first element continues its beam with
    float *top, *offset;
    __device__ MergeSmem(void* raw, const BeamArgs& a) {
        group_at = static_cast<uint32_t*>(raw);  // (read 16 bytes at a time)
        listed = group_at + a.groups;
        staged = listed + kListed;
        key_a = reinterpret_cast<uint64_t*>(staged);
        key_b = key_a + a.list_a;
        at_a = reinterpret_cast<uint32_t*>(key_b + a.list_b);
        at_b = at_a + a.list_a;
        uint32_t *const lists_end = at_b + a.list_b, *const bounds_end = staged + a.staged;
        group_key = reinterpret_cast<uint64_t*>(lists_end > bounds_end ? lists_end : bounds_end);
        chosen_row = reinterpret_cast<const void**>(group_key + a.groups);
        log_sum = reinterpret_cast<double*>(chosen_row + a.chosen);
        start = log_sum + MKBS_MAX_BEAMS;
        rank = reinterpret_cast<int*>(start + MKBS_MAX_BEAMS);
        chosen_beam = rank + a.groups;
        chosen_first = chosen_beam + a.chosen;
        kind = chosen_first + a.chosen;
        top = reinterpret_cast<float*>(kind + MKBS_MAX_BEAMS);
        offset = top + MKBS_MAX_BEAMS;
    }
};

enum Kind { kLive = 0, kDone = 1, kDead = 2 };  // kDead: every continuation has score minus infinity

// Segments, then elements, go through the same code, loops are hardly unrolled, and there are not more threads than there is work
// for: a block runs through this once, fetching and issuing instructions is what takes the time.
template <typename T>
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const BeamArgs a) {
    extern __shared__ __align__(16) uint64_t raw[];
    const MergeSmem sm(raw, a);
    __shared__ int listed, listed_soon;
    __shared__ uint32_t bound;
    const int t = threadIdx.x, group_of = blockIdx.x, row0 = group_of * a.beams, warp = t >> 5, lane = t & 31;
    const int segments = a.segments, groups = a.groups, k = a.k, shift_segment = __ffs(a.segment) - 1;
    constexpr int threads = kMergeThreads;
    const int lanes = threads / groups, group = t / lanes;
    const float per_segments = 1.f / segments;  // (exact quotients: candidates are fewer than 2^17)
    const uint32_t* const tops = a.tops + (size_t)row0 * segments;
    const uint64_t lowest = order64(-(double)INFINITY);
    auto row_of = [&](int b) { return static_cast<const T*>(a.logits) + (row0 + b) * a.row_stride; };
    auto beam_of = [&](int i) { return (int)((i + 0.5f) * per_segments); };
    if (t == 0) listed_soon = 0;
    for (int b = t; b < a.beams; b += threads) {
        const float c = a.scores != nullptr ? a.scores[row0 + b] : 0.f;
        const bool over = a.done != nullptr && a.done[row0 + b];
        sm.start[b] = c;
        sm.kind[b] = !is_live(c) ? kDead : over ? kDone : kLive;
    }
    __syncthreads();
    mkbh::after_previous();
    int chosen = 0, infinite = 0;  // (infinite: some logit is; the bounds below hold for finite ones)
    float known = -INFINITY;       // a lower bound of the k-th best from the segments
#pragma unroll 1
    for (int stage = 0; stage < 2; ++stage) {
        int count = stage == 0 ? a.beams * segments : chosen << shift_segment;
        // element i: of which beam, and where in its row; -1: none
        auto place = [&](int i, int& v) {
            v = sm.chosen_first[i >> shift_segment] + (i & (a.segment - 1));
            return v >= 0 && v < a.vocab ? sm.chosen_beam[i >> shift_segment] : -1;
        };
        // a segment's largest logit, or an element, as order_of; 0: there is none (not set for a beam that has none, or has ended)
        auto fetch = [&](int i) {
            if (stage == 0) return tops[i];
            int v = 0;
            const int b = place(i, v);  // (read in any case, so that reads do not wait for one another)
            const float x = mkbh::to_f<T>(static_cast<const T*>(sm.chosen_row[i >> shift_segment])[min(max(v, 0), a.vocab - 1)]);
            return b >= 0 && sm.kind[b] == kLive ? order_of(fmaxf(x, -INFINITY)) : 0u;
        };
        auto stage_all = [&] {
#pragma unroll 8
            for (int i = t; i < count; i += threads) sm.staged[i] = fetch(i);
        };
        auto choose = [&](int n, int b, int s) {  // segment s of beam b, as the n-th; b below 0: none
            const T* const row = row_of(max(b, 0));
            sm.chosen_beam[n] = b;
            sm.chosen_first[n] = (s << shift_segment) - shift_of(row);
            sm.chosen_row[n] = row;
        };
        const bool staged = count <= a.staged;
        if (staged && known == -INFINITY) stage_all();
        if (stage == 0) {
#pragma unroll 1
            for (int b = warp; b < a.beams; b += threads / 32) {  // the beams' sums
                float top = -INFINITY;
                double sum = 0.0;
                if (sm.kind[b] == kLive) {
                    const float2* const sums = a.sums + (size_t)(row0 + b) * a.parts;
                    float2 part = make_float2(-INFINITY, 0.f);  // of the lane's parts together, the first 32 at once
                    for (int i = lane; i < a.parts; i += 32) {
                        const float2 next = sums[i];
                        const float high = fmaxf(part.x, next.x);
                        part.y = (part.y > 0.f ? part.y * to_top(part.x, high) : 0.f) + (next.y > 0.f ? next.y * to_top(next.x, high) : 0.f);
                        part.x = high;
                    }
                    top = mkbh::warp_max(part.x);
                    if (part.y > 0.f) sum = part.y * to_top(part.x, top);
#pragma unroll
                    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    infinite |= top == INFINITY;
                }
                if (lane == 0 && sm.kind[b] == kLive) {
                    const double log_sum = log(sum);
                    sm.top[b] = top;
                    sm.log_sum[b] = log_sum;
                    sm.offset[b] = (float)(sm.start[b] - (double)top - log_sum);
                    if (top == -INFINITY) sm.kind[b] = kDead;
                }
                __syncwarp();
                if (lane == 0 && sm.kind[b] != kLive) sm.offset[b] = -INFINITY;
            }
        }
        if (t == 0) listed = 0;
        infinite = __syncthreads_or(infinite);
        auto candidate = [&](int i) {
            const uint32_t order = fetch(i);
            int b, v = 0;
            bool there, ends;
            uint32_t at = i;
            if (stage == 0) {
                b = beam_of(i);
                const int s = i - b * segments, shift = shift_of(row_of(b));
                there = (s << shift_segment) < shift + a.vocab;
                ends = (a.eos + shift) >> shift_segment == s;
            } else {
                b = place(i, v);
                there = b >= 0;
                b = max(b, 0);
                ends = v == a.eos;
                at = (uint32_t)b * a.vocab + v;
            }
            if (!there) return Candidate{0, at};
            uint64_t key = lowest;
            if (sm.kind[b] == kLive) {
                const float x = value_of(order), top = sm.top[b];
                if (x > -INFINITY) key = order64(sm.start[b] + ((x == top ? 0.0 : (double)x - (double)top) - sm.log_sum[b]));
            } else if (sm.kind[b] == kDone && ends) {
                key = order64(sm.start[b]);
            }
            return Candidate{key, at};
        };
        auto take = [&](int rank, const Candidate& c) {
            if (stage == 0) {
                const int b = c.key ? beam_of(c.at) : -1;
                choose(rank, b, c.at - b * segments);
            } else {
                const int b = c.at / a.vocab, v = c.at - b * a.vocab, to = group_of * k + rank;
                a.out_scores[to] = (float)value64(c.key);
                a.out_parents[to] = row0 + b;
                a.out_tokens[to] = v;
                if (a.out_done != nullptr) a.out_done[to] = v == a.eos || (a.done != nullptr && a.done[row0 + b]);
            }
        };
        // A score in fp32, and by how much it may be off
        auto score = [&](int i, uint32_t order, float& off) {
            const int b = stage == 0 ? beam_of(i) : max(sm.chosen_beam[i >> shift_segment], 0);
            const float x = order ? value_of(order) : -INFINITY, y = sm.offset[b];
            off = (fabsf(x) + fabsf(y)) * 0x1p-21f;  // (infinite with the score; then the bounds are not numbers, and pass no comparison)
            return x + y;
        };
        // Listed elements are ranked in 64 bits
        auto rank_listed = [&](int some) {
            Candidate own{0, 0};
            if (t < some) own = candidate(sm.listed[t]);
            sm.key_a[t] = own.key;
            sm.at_a[t] = own.at;
            __syncthreads();
#pragma unroll 1
            for (int c = warp; c < some; c += threads / 32) {  // (a warp ranks a candidate)
                const Candidate it{sm.key_a[c], sm.at_a[c]};
                int rank = 0;
                for (int j = lane; j - lane < some; j += 32) rank += __popc(__ballot_sync(0xffffffffu, j < some && Candidate{sm.key_a[j], sm.at_a[j]}.before(it)));
                if (lane == 0 && rank < k) take(rank, it);
            }
        };
        // the one continuation of beams that have ended
        auto list_ended = [&](auto list) {
            if (a.done == nullptr || t >= (stage == 0 ? a.beams : chosen)) return;
            const int b = stage == 0 ? t : sm.chosen_beam[t];
            if (b < 0 || sm.kind[b] != kDone) return;
            const int at = stage == 0 ? 0 : a.eos - sm.chosen_first[t];
            if (stage == 0) list(0, b, (a.eos + shift_of(row_of(b))) >> shift_segment);
            else if (at >= 0 && at < a.segment) list((t << shift_segment) + at, 0, 0);
        };
        if (known > -INFINITY) {  // elements that the segments' bound lets pass: mostly few
            auto list = [&](int i, int, int) {
                const int n = atomicAdd(&listed_soon, 1);
                if (n < kListed) sm.listed[n] = i;
            };
            // 16 bytes at a time, as a segment begins at a multiple of them
            constexpr int kVector = 16 / sizeof(T), kShift = sizeof(T) == 2 ? 3 : 2, kTogether = 2;
            const int vectors = count >> kShift, of_segment = a.segment >> kShift;
#pragma unroll 1
            for (int q0 = t; q0 < vectors; q0 += kTogether * threads) {
                uint4 w[kTogether];
#pragma unroll
                for (int u = 0; u < kTogether; ++u) {
                    const int q = q0 + u * threads, c = q >> (shift_segment - kShift), b = q < vectors ? sm.chosen_beam[c] : -1;
                    w[u] = none_of<T>();
                    if (b < 0 || sm.kind[b] != kLive) continue;
                    const int v = sm.chosen_first[c] + (q & (of_segment - 1)) * kVector;
                    const T* const row = static_cast<const T*>(sm.chosen_row[c]);
                    if (v >= 0 && v + kVector <= a.vocab) w[u] = mkb::ld_nc_v4(row + v);
                    else w[u] = edge_vector(row - shift_of(row), v + shift_of(row), shift_of(row), shift_of(row) + a.vocab);
                }
#pragma unroll
                for (int u = 0; u < kTogether; ++u) {
                    const int q = q0 + u * threads;
                    if (q >= vectors) break;
                    const float y = sm.offset[max(sm.chosen_beam[q >> (shift_segment - kShift)], 0)];
                    const uint32_t words[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
                    for (int e = 0; e < kVector; ++e) {
                        const float x = sizeof(T) == 4 ? __uint_as_float(words[e & 3]) : e & 1 ? mkb::bf16_hi(words[e / 2]) : mkb::bf16_lo(words[e / 2]);
                        const float off = (fabsf(x) + fabsf(y)) * 0x1p-21f;  // (as in `score`; what is no number passes no comparison)
                        if (x + y + off >= known) list(q * kVector + e, 0, 0);
                    }
                }
            }
            list_ended(list);
            __syncthreads();
            const int some = listed_soon;
            if (some >= min(k, count) && some <= kListed) {
                rank_listed(some);
                break;
            }
            if (staged) stage_all();
            __syncthreads();
        }
        float best_score = -INFINITY;
#pragma unroll 2
        for (int i = t; i < count; i += threads) {
            float off;
            const float x = score(i, staged ? sm.staged[i] : fetch(i), off);
            best_score = fmaxf(best_score, x - off);
            if (staged) sm.staged[i] = __float_as_uint(x + off);
        }
        // (neighbours fall into different groups: often one beam, or one run of tokens, has most of the best)
        sm.listed[t] = order_of(best_score);
        __syncthreads();
        if (t < groups) {
            uint32_t most = sm.listed[t];
            for (int j = t + groups; j < threads; j += groups) most = max(most, sm.listed[j]);
            sm.group_at[t] = most;
            sm.rank[t] = 0;
        }
        __syncthreads();
        // ranks of the groups' maxima: a thread compares one of them with a share of the others
        const int mine = t % groups, share = groups / lanes, first = t / groups * share;
        {
            const uint32_t own = sm.group_at[mine];
            int before = 0;
#pragma unroll 4
            for (int j = first; j < first + share; j += 4) {
                const uint4 o = *reinterpret_cast<const uint4*>(sm.group_at + j);
                before += (o.x > own || (o.x == own && j < mine)) + (o.y > own || (o.y == own && j + 1 < mine)) + (o.z > own || (o.z == own && j + 2 < mine)) +
                          (o.w > own || (o.w == own && j + 3 < mine));
            }
            if (before) atomicAdd(&sm.rank[mine], before);
        }
        __syncthreads();
        if (t < groups && sm.rank[t] == k - 1) bound = sm.group_at[t];
        __syncthreads();
        const float least = value_of(bound);
        // What may be among the k best: of the segments all are chosen, in any order, of the elements the k best
        const int most = stage == 0 ? a.chosen : kListed;
        auto list = [&](int i, int b, int segment_of) {
            const int n = atomicAdd(&listed, 1);
            if (n >= most) return;
            if (stage == 0) choose(n, b, segment_of);
            else sm.listed[n] = i;
        };
        if (least > -INFINITY && !infinite) {
#pragma unroll 4
            for (int i = t; i < count; i += threads) {
                float high;
                if (staged) {
                    high = __uint_as_float(sm.staged[i]);
                } else {
                    float off;
                    high = score(i, fetch(i), off);
                    high += off;
                }
                if (high >= least) list(i, stage == 0 ? beam_of(i) : 0, stage == 0 ? i - beam_of(i) * segments : 0);
            }
            list_ended(list);
        }
        __syncthreads();
        const int some = listed;
        const bool few_listed = some >= min(k, count) && some <= most && least > -INFINITY;
        if (stage == 0 && few_listed) {
            chosen = some;
            known = least;
        } else if (few_listed) {
            rank_listed(some);
        } else {
            // Rounds: into groups by thread, the groups' best ranked, the members of the first k into a list
            int from_list = 0;  // 0: candidate(i), 1: list a, 2: list b
            auto get = [&](int i) {
                if (from_list == 0) return candidate(i);
                return from_list == 1 ? Candidate{sm.key_a[i], sm.at_a[i]} : Candidate{sm.key_b[i], sm.at_b[i]};
            };
#pragma unroll 1
            for (bool last = false;;) {
                last = count <= groups;
                // Candidates of a thread: t, t + threads, ...; of few candidates one that leaves no group empty; in the end a group is a candidate
                const bool few = count <= threads;
                const int turns = few ? 1 : (count + threads - 1) / threads, members = few ? (count + groups - 1) / groups : turns * lanes;
                const int from = last ? (t % lanes ? count : group) : few ? t % lanes * groups + group : t;
                Candidate best{0, 0};
#pragma unroll 1
                for (int i = from; i < count; i += threads) {
                    const Candidate c = get(i);
                    if (c.before(best)) best = c;
                }
                for (int o = lanes / 2; o; o >>= 1) {
                    const Candidate c{__shfl_xor_sync(0xffffffffu, best.key, o), __shfl_xor_sync(0xffffffffu, best.at, o)};
                    if (c.before(best)) best = c;
                }
                if (t % lanes == 0) {
                    sm.group_key[group] = best.key;
                    sm.group_at[group] = best.key ? best.at : 0x80000000u + group;  // (what is none is behind all others, and no two alike)
                    sm.rank[group] = 0;
                }
                __syncthreads();
                const Candidate own{sm.group_key[mine], sm.group_at[mine]};
                int before = 0;
                for (int j = first; j < first + share; ++j) before += Candidate{sm.group_key[j], sm.group_at[j]}.before(own);
                if (before) atomicAdd(&sm.rank[mine], before);
                __syncthreads();
                const int rank = sm.rank[group];
                if (last) {
                    if (t % lanes == 0 && rank < k) take(rank, best);
                    break;
                }
                uint64_t* const key = from_list == 1 ? sm.key_b : sm.key_a;
                uint32_t* const at = from_list == 1 ? sm.at_b : sm.at_a;
                if (rank < k) {
#pragma unroll 1
                    for (int n = 0; n < turns; ++n) {
                        const int i = from + n * threads, member = n * lanes + t % lanes;
                        if (member >= members) continue;
                        const Candidate c = i < count ? get(i) : Candidate{0, 0};
                        key[rank * members + member] = c.key;
                        at[rank * members + member] = c.at;
                    }
                }
                count = k * members;
                from_list = from_list == 1 ? 2 : 1;
                __syncthreads();
            }
        }
        if (stage == 0 && !few_listed) chosen = min(k, a.beams * segments);
        __syncthreads();
    }
}

template <typename T>
cudaError_t launch(const BeamPlan& p, const MkbsBeams& b, const BeamArgs& a, cudaStream_t s) {
    // (in any case: what a kernel may have without asking counts its static words too)
    if (const cudaError_t e = allow_shared_memory<beam_merge_kernel<T>>(); e != cudaSuccess) return e;
    beam_scan_kernel<T><<<dim3(p.parts, p.rows), 32 * kScanWarps, 0, s>>>(a);
    if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(b.groups);
    c.blockDim = dim3(kMergeThreads);
    c.dynamicSmemBytes = p.merge_smem();
    c.stream = s;
    cudaLaunchAttribute early = mkbh::may_begin_early();
    c.attrs = &early;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, beam_merge_kernel<T>, a);
}

}  // namespace

size_t beam_bytes(const MkbsBeams& b) {
    const BeamPlan p(b);
    return p.merge_smem() <= kMostShared ? p.bytes : 0;
}

cudaError_t beam_launch(const MkbsBeams& b, cudaStream_t s) {
    const BeamPlan p(b);
    char* const work = static_cast<char*>(b.workspace);
    const BeamArgs a{b.beams, b.vocab, b.k, p.segment, p.segments, p.per_warp, p.parts, p.groups, p.list_a, p.list_b, p.staged, p.chosen, b.row_stride, b.logits, b.scores,
                     b.done, b.eos, reinterpret_cast<uint32_t*>(work), reinterpret_cast<float2*>(work + p.part_offset), b.out_scores, b.out_parents,
                     b.out_tokens, b.out_done};
    return b.dtype == MKBS_F32 ? launch<float>(p, b, a, s) : launch<bf16>(p, b, a, s);
}

}  // namespace mkbs
