// Cache rows and states of sequences, moved in place: slots that take another slot's, and a cache cut to the rows that stay.
#include <type_traits>

#include "hybrid_common.cuh"
#include "sequence_kernels.h"

namespace mkbs {
namespace {

// ---- x[slot] <- x[parents[slot]] ---------------------------------------------------------- //
// A block takes one run of bytes of all slots that depend on each other at once: it reads what other slots take into shared
// memory, each source once however many take it, and writes it when all of it is there.  Runs do not overlap, so no slot loses
// what another still needs.  Slots that depend on each other are the components of the graph of parents (a beam search's
// groups): the fewer sources a run has, the longer its copies are.
// Memory bounds it: 8 groups of 8 slots, 1024 rows of 2 KB in 16 caches take 385 us at 6.46 TB/s; 4 slots, 101 rows of 1 KB in 32 caches
// 8.8 us at 2.0 TB/s, a launch and a round trip of copies.
constexpr int kReorderThreads = MKBS_MAX_SLOTS, kReorderBytes = 96 * 1024;  // (bytes: of the plain kernel)
constexpr int kStages = 4, kStageBytes = 52 * 1024, kShortRun = 2048;

struct ReorderArgs {
    int slots, num_regions, first;
    const int32_t *parents, *lengths;
    int32_t* status;
    MkbsRegion regions[MKBS_MAX_REGIONS];
};

struct Components {
    int parent[MKBS_MAX_SLOTS], length[MKBS_MAX_SLOTS], label[MKBS_MAX_SLOTS], place[MKBS_MAX_SLOTS];
    int source[MKBS_MAX_SLOTS], target[MKBS_MAX_SLOTS];  // sources, and slots that take one, by component
    int source_begin[MKBS_MAX_SLOTS + 1], target_begin[MKBS_MAX_SLOTS + 1], run[MKBS_MAX_SLOTS], longest[MKBS_MAX_SLOTS];
    int count, changed;
    unsigned long long bytes;  // that all sources hold

    __device__ __forceinline__ bool moves(int s, int first) const { return parent[s] != s && length[parent[s]] > first; }

    // By all threads of a block, of which there is one per slot.
    __device__ void find(const ReorderArgs& a) {
        const int s = threadIdx.x, n = a.slots;
        if (s < n) {
            const int p = a.parents[s];
            parent[s] = p >= 0 && p < n ? p : s;
            length[s] = a.lengths != nullptr ? max(a.lengths[s], 0) : 1 << 30;
            label[s] = s;
            place[s] = 0;
        }
        if (s == 0) count = 0, bytes = 0;
        __syncthreads();
        const bool taken = s < n && moves(s, a.first);
        if (taken) place[parent[s]] = 1;
        do {  // every slot learns the lowest slot that it is connected with
            __syncthreads();
            if (s == 0) changed = 0;
            __syncthreads();
            if (taken) {
                const int mine = label[s], its = label[parent[s]], low = min(mine, its);
                if (mine > low) atomicMin(&label[s], low), changed = 1;
                if (its > low) atomicMin(&label[parent[s]], low), changed = 1;
            }
            __syncthreads();
        } while (changed);
        // sources and targets in the order of their components, components in the order of their lowest slots
        const bool source_here = s < n && place[s];
        int sources = 0, targets = 0, before = 0, own_sources = 0, own_targets = 0, most = 0;
        if (s < n) {
            for (int i = 0; i < n; ++i) {
                const bool first_of = label[i] < label[s] || (label[i] == label[s] && i < s), takes = moves(i, a.first);
                sources += place[i] && first_of;
                targets += takes && first_of;
                if (label[i] == s) {
                    own_sources += place[i];
                    own_targets += takes;
                    if (place[i]) most = max(most, length[i]);
                }
            }
            run[s] = own_sources > 0;  // a component's lowest slot
        }
        __syncthreads();
        if (s < n) {
            for (int i = 0; i < s; ++i) before += run[i];
            if (source_here) source[sources] = s, place[s] = sources;
            if (taken) target[targets] = s;
            if (own_sources > 0) {
                longest[before] = most;
                source_begin[before + 1] = own_sources;
                target_begin[before + 1] = own_targets;
                atomicMax(&count, before + 1);
            }
        }
        __syncthreads();
        if (s == 0) {
            source_begin[0] = target_begin[0] = 0;
            for (int c = 0; c < count; ++c) {
                source_begin[c + 1] += source_begin[c];
                target_begin[c + 1] += target_begin[c];
            }
        }
        __syncthreads();
        if (s < count) {
            unsigned long long all = 0;
            for (int r = 0; r < a.num_regions; ++r) all += (unsigned long long)(max(min(longest[s], a.regions[r].rows) - a.first, 0) * a.regions[r].row_bytes) * a.regions[r].outer;
            atomicAdd(&bytes, all * (source_begin[s + 1] - source_begin[s]));
        }
        __syncthreads();
        if (s < count) {
            // two steps and more for every block, as far as copies do not get short (a step costs the warp nearly a microsecond: six states
            // of 5 MB with 1, 2, 3, 4, 8 steps 14.9, 14.9, 15.9, 16.0, 20.5 us)
            const int sources_here = source_begin[s + 1] - source_begin[s], longest_run = kStageBytes / sources_here / 128 * 128;
            const int64_t share = (int64_t)(bytes / (2 * kSms) / sources_here + 127) / 128 * 128;
            run[s] = (int)min((int64_t)longest_run, max((int64_t)kShortRun, share));
        }
        __syncthreads();
    }
};

// A step: one run of the bytes of a component's slots, in one layer of one region.
struct Step {
    int c, r;
    int at, runs;   // step of this component and region, and how many runs a layer has there (memory ends before 2^31 runs)
    int64_t begin;  // of the run, from a slot's first byte on
    char* base;     // of the run in slot 0
    __device__ __forceinline__ void count(const ReorderArgs& a, const Components& k) {
        const MkbsRegion& g = a.regions[r];
        const int64_t bytes = (min(k.longest[c], g.rows) - a.first) * g.row_bytes;
        runs = bytes > 0 ? (int)((bytes + k.run[c] - 1) / k.run[c]) : 0;
    }
    __device__ __forceinline__ bool settle(const ReorderArgs& a, const Components& k) {  // false: there are no more
        while (c < k.count && at >= runs * a.regions[r].outer) {
            at -= runs * a.regions[r].outer;
            if (++r == a.num_regions) r = 0, ++c;
            if (c < k.count) count(a, k);
        }
        if (c >= k.count) return false;
        const int layer = at / runs;
        begin = a.first * a.regions[r].row_bytes + (int64_t)(at - layer * runs) * k.run[c];
        base = static_cast<char*>(a.regions[r].base) + layer * a.regions[r].outer_stride + begin;
        return true;
    }
    __device__ __forceinline__ Step(const ReorderArgs& a, const Components& k) : c(0), r(0), at(blockIdx.x), runs(0) {
        if (k.count > 0) count(a, k);
    }
    // bytes of the run that a slot holds
    __device__ __forceinline__ int held(const ReorderArgs& a, const Components& k, int slot) const {
        const MkbsRegion& g = a.regions[r];
        return (int)max((int64_t)0, min((int64_t)k.run[c], min(k.length[slot], g.rows) * g.row_bytes - begin));
    }
};

// Everything a multiple of 16 bytes: one warp keeps bulk copies under way, a lane per slot.
__global__ void __launch_bounds__(kReorderThreads, 1) reorder_bulk_kernel(const __grid_constant__ ReorderArgs a) {
    extern __shared__ uint4 raw[];
    __shared__ Components k;
    __shared__ uint64_t bars[kStages];
    k.find(a);
    if (threadIdx.x >= 32) return;
    const int lane = threadIdx.x;
    const uint32_t bar0 = mkb::smem_u32(bars), data = (mkb::smem_u32(raw) + 127u) & ~127u;
    if (lane == 0) {
        for (int i = 0; i < kStages; ++i) mkb::mbar_init(bar0 + i * 8, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    Step load(a, k), store = load;
    int issued = 0;
    auto arrived = [&](int step, unsigned long long limit_ns) {
        unsigned long long began = 0;
        while (!mkb::mbar_try_wait(bar0 + step % kStages * 8, (uint32_t)(step / kStages) & 1u)) {
            const unsigned long long now = mkb::globaltimer_ns();
            if (began == 0) began = now;
            if (now - began > limit_ns) return false;
        }
        return true;
    };
    auto issue = [&]() {
        const int st = issued % kStages, from = k.source_begin[load.c], to = k.source_begin[load.c + 1], run = k.run[load.c];
        int bytes = 0;
        for (int i = from + lane; i < to; i += 32) bytes += load.held(a, k, k.source[i]);
        bytes = __reduce_add_sync(0xffffffffu, bytes);
        if (lane == 0) mkb::mbar_expect_tx(bar0 + st * 8, bytes);
        __syncwarp();
        for (int i = from + lane; i < to; i += 32) {
            const int n = load.held(a, k, k.source[i]);
            if (n > 0)
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(data + st * kStageBytes + (i - from) * run),
                             "l"(load.base + k.source[i] * a.regions[load.r].slot_stride), "r"(n), "r"(bar0 + st * 8)
                             : "memory");
        }
        ++issued;
        load.at += gridDim.x;
    };
    while (issued < kStages && load.settle(a, k)) issue();
    for (int done = 0; store.settle(a, k); ++done, store.at += gridDim.x) {
        const int st = done % kStages, source0 = k.source_begin[store.c], run = k.run[store.c];
        if (!__all_sync(0xffffffffu, arrived(done, 2000000000ull))) {  // (every lane reads what has arrived)
            if (lane == 0 && a.status != nullptr && atomicCAS(a.status, 0, (int)MKBS_ERR_DEVICE_TIMEOUT) == 0) a.status[1] = blockIdx.x;
            for (int i = done; i < issued; ++i) arrived(i, 200000000ull);  // (before shared memory goes away)
            break;
        }
        for (int i = k.target_begin[store.c] + lane; i < k.target_begin[store.c + 1]; i += 32) {
            const int s = k.target[i], p = k.parent[s], n = store.held(a, k, p);
            if (n > 0)
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(store.base + s * a.regions[store.r].slot_stride),
                             "r"(data + st * kStageBytes + (k.place[p] - source0) * run), "r"(n)
                             : "memory");
        }
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        if (done > 0 && load.settle(a, k)) {  // the stage before this one is free when its copies have been read
            asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            __syncwarp();
            issue();
        }
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// Any sizes and alignments.
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
// of its order) by counting, until few rows share its digits: those are listed, and the rest of the digits is found among them.  Rows
// of that very weight stay in the order of their places.  The weights are read from memory once: their orders lie in shared memory, as
// far as they fit, for the passes that follow: digits (seldom), list, write.  A warp has a run of the rows in shared memory and one
// of those behind; it counts those that stay, and with the counts of the runs before it writes them.
// Instructions and what a pass begins and ends with bound it, not memory: 128 blocks of 65001 rows take 30 us (the weights at 1.1 TB/s;
// with every digit found by a pass over all rows and no list 39), 448 of 4096 rows 10 (24, with 1024 threads each), 32 of 1500 5.4 (7.7).
constexpr int kDigits = 2048, kSelectAhead = 8, kAtOnce = 4, kFewRows = 1536, kRanked = 256;
constexpr int kMostOrders = (227 * 1024 - kStaticShared) / 16 * 4;

__device__ __forceinline__ uint32_t inclusive_scan(uint32_t v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t m = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += m;
    }
    return v;
}

template <int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) select_kernel(const MkbsSelect s, const int fit) {
    constexpr int kEach = kDigits / kThreads;
    extern __shared__ uint4 orders[];  // (a multiple of four of them)
    __shared__ __align__(16) int count[kDigits];
    __shared__ int sums[32], found[3], few[kFewRows], listed;
    __shared__ int above[2][32], ties[2][32];  // rows of the runs in shared memory, and behind: above the limit, at it
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, head = blockIdx.x, b = blockIdx.y, layer = blockIdx.z;
    const int n = length_of(s.lengths, s.length, s.positions, b), kept = min(n, s.keep);
    const int64_t at = layer * s.w_layer + b * s.w_sequence + head * s.w_head;
    const float* const w = s.weights + at;
    int32_t* const rows = s.rows + (((int64_t)layer * s.sequences + b) * s.kv_heads + head) * s.keep;
    for (int r = kept + t; r < s.keep; r += kThreads) rows[r] = -1;
    if (n <= s.keep) {
        for (int r = t; r < n; r += kThreads) rows[r] = r;
        float* const out = s.kept != nullptr ? s.kept + at : nullptr;
        if (out != nullptr && out != w)
            for (int r = t; r < n; r += kThreads) out[r] = w[r];
        return;
    }
    const int rivals = n - s.sinks - s.recent, quads = (rivals + 3) / 4;  // rows that compete, from row `sinks` on
    const float* const of_rivals = w + s.sinks;
    int need = s.keep - s.sinks - s.recent;  // of them stay
    const bool some = need > 0;
    // order_of, not a number as minus infinity; what fills the last four up is below everything
    auto from_memory = [&](int i) { return i < rivals ? order_of(fmaxf(of_rivals[i], -INFINITY)) : 0u; };
    const int near = min(quads, fit / 4);  // in shared memory
    auto run_of = [&](int part, int& from, int& to) {  // the warp's, whole turns of 32 lanes
        const int all = part ? quads - near : near, run = (all + kThreads - 1) / kThreads * 32, first = part ? near : 0;
        from = first + warp * run;
        to = min(from + run, first + all);
    };
    auto load = [&](int part, int q0, int to, uint4 (&o)[kAtOnce]) {  // four rows of a lane, and those of the next turns
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const int q = q0 + 32 * u + lane;
            o[u] = make_uint4(0, 0, 0, 0);
            if (q >= to) continue;
            if (part == 0) o[u] = orders[q];
            else o[u] = make_uint4(from_memory(4 * q), from_memory(4 * q + 1), from_memory(4 * q + 2), from_memory(4 * q + 3));
        }
    };
    auto clear = [&] {
#pragma unroll
        for (int i = 0; i < kEach; i += 2) reinterpret_cast<int2*>(count)[i / 2 * kThreads + t] = make_int2(0, 0);
    };
    uint32_t limit = 0;
    int shift = 32, size = rivals;  // rows that begin with the digits so far
    // The digit from the counts, from the largest down, kEach per thread: how many rows lie above a digit
    auto decide = [&] {
        __syncthreads();
        const int d0 = kDigits - kEach * (t + 1);
        int c[kEach], mine = 0;
#pragma unroll
        for (int i = 0; i < kEach; i += 2) {
            const int2 two = *reinterpret_cast<const int2*>(count + d0 + i);
            c[i] = two.x, c[i + 1] = two.y;
            mine += two.x + two.y;
        }
        int before = inclusive_scan(mine, lane);
        if (lane == 31) sums[warp] = before;
        __syncthreads();
        before += __reduce_add_sync(0xffffffffu, lane < warp ? sums[lane] : 0) - mine;
#pragma unroll
        for (int i = kEach - 1; i >= 0; --i) {
            if (before < need && need <= before + c[i]) found[0] = d0 + i, found[1] = before, found[2] = c[i];
            before += c[i];
        }
        clear();  // (all have read)
        __syncthreads();
        limit |= (uint32_t)found[0] << shift;
        need -= found[1];
        size = found[2];
    };
    auto next_digit = [&] {
        const int bits = shift > 10 ? 11 : 10;
        shift -= bits;
        return 1u << bits;
    };
    clear();
    if (t < 64) (&above[0][0])[t] = (&ties[0][0])[t] = 0;
    if (t == 0) listed = 0;
    __syncthreads();
    next_digit();
    {
        uint32_t* const kept_orders = reinterpret_cast<uint32_t*>(orders);
        int i0 = t;
        for (const int all = min(rivals, fit) - (kSelectAhead - 1) * kThreads; i0 < all; i0 += kSelectAhead * kThreads) {
            float x[kSelectAhead];
#pragma unroll
            for (int u = 0; u < kSelectAhead; ++u) x[u] = of_rivals[i0 + u * kThreads];
#pragma unroll
            for (int u = 0; u < kSelectAhead; ++u) {
                const uint32_t o = order_of(fmaxf(x[u], -INFINITY));
                kept_orders[i0 + u * kThreads] = o;
                atomicAdd(&count[o >> shift], 1);
            }
        }
        for (; i0 < 4 * quads; i0 += kSelectAhead * kThreads) {
            uint32_t o[kSelectAhead];
#pragma unroll
            for (int u = 0; u < kSelectAhead; ++u) o[u] = from_memory(i0 + u * kThreads);
#pragma unroll
            for (int u = 0; u < kSelectAhead; ++u) {
                const int i = i0 + u * kThreads;
                if (i < 4 * near) kept_orders[i] = o[u];
                if (i < rivals) atomicAdd(&count[o[u] >> shift], 1);
            }
        }
    }
    if (some) {
        decide();
        while (shift > 0 && size > kFewRows) {
            const uint32_t digits = next_digit();
#pragma unroll 1
            for (int part = 0; part < 2; ++part) {
                int from, to;
                run_of(part, from, to);
#pragma unroll 1
                for (int q0 = from; q0 < to; q0 += 32 * kAtOnce) {
                    uint4 o[kAtOnce];
                    load(part, q0, to, o);
#pragma unroll
                    for (int u = 0; u < kAtOnce; ++u) {
                        const uint32_t each[4] = {o[u].x, o[u].y, o[u].z, o[u].w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {  // (what does not begin with the digits so far is beyond the last one: orders end at 0xff800000)
                            const uint32_t digit = (each[i] - limit) >> shift;
                            if (digit < digits) atomicAdd(&count[digit], 1);
                        }
                    }
                }
            }
            decide();
        }
        // Rows above all that begin with the digits, of each run, and a list of those that do, or how many they are when no digit is left
        const uint32_t span = shift > 0 ? (1u << shift) - 1 : 0;
#pragma unroll 1
        for (int part = 0; part < 2; ++part) {
            int from, to, up = 0, at_it = 0;
            run_of(part, from, to);
#pragma unroll 1
            for (int q0 = from; q0 < to; q0 += 32 * kAtOnce) {
                uint4 o[kAtOnce];
                load(part, q0, to, o);
                uint32_t within = 0;  // a bit for each row
#pragma unroll
                for (int u = 0; u < kAtOnce; ++u) {
                    const uint32_t each[4] = {o[u].x, o[u].y, o[u].z, o[u].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        up += each[i] > limit + span;
                        within |= each[i] - limit <= span ? 1u << (4 * u + i) : 0u;
                    }
                }
                const int have = __popc(within);
                at_it += have;
                if (have && shift > 0) {
                    for (int to_list = atomicAdd(&listed, have); within; within &= within - 1) {  // (`size` of them in all)
                        const int bit = __ffs(within) - 1;
                        few[to_list++] = 4 * (q0 + 32 * (bit / 4) + lane) + bit % 4;
                    }
                }
            }
            up = __reduce_add_sync(0xffffffffu, up);
            if (shift == 0) at_it = __reduce_add_sync(0xffffffffu, at_it);
            if (lane == 0) {
                above[part][warp] = up;
                if (shift == 0) ties[part][warp] = at_it;
            }
        }
        if (shift > 0) {
            __syncthreads();
            constexpr int kMine = (kFewRows + kThreads - 1) / kThreads;
            const int all = size;
            int place[kMine];
            uint32_t own[kMine];
#pragma unroll
            for (int u = 0; u < kMine; ++u) {
                const int e = t + u * kThreads;
                place[u] = e < all ? few[e] : -1;
                own[u] = e >= all ? 0u : place[u] < 4 * near ? reinterpret_cast<const uint32_t*>(orders)[place[u]] : from_memory(place[u]);
            }
            if (size <= kRanked) {  // ranked by counting
                if (t < kRanked) reinterpret_cast<uint32_t*>(count)[t] = own[0];  // (0 behind the list)
                __syncthreads();
                if (t < size) {
                    int before = 0, alike = 0;
#pragma unroll 4
                    for (int e = 0; e < size; e += 4) {
                        const uint4 o = *reinterpret_cast<const uint4*>(count + e);
                        before += (o.x > own[0]) + (o.y > own[0]) + (o.z > own[0]) + (o.w > own[0]);
                        alike += (o.x == own[0]) + (o.y == own[0]) + (o.z == own[0]) + (o.w == own[0]);
                    }
                    if (before < need && need <= before + alike) found[0] = (int)own[0], found[1] = before;  // (all that are alike write the same)
                }
                __syncthreads();
                limit = (uint32_t)found[0];
                need -= found[1];
                shift = 0;
            }
            while (shift > 0) {
                const uint32_t digits = next_digit();
#pragma unroll
                for (int u = 0; u < kMine; ++u) {
                    const uint32_t digit = (own[u] - limit) >> shift;
                    if (place[u] >= 0 && digit < digits) atomicAdd(&count[digit], 1);
                }
                decide();
            }
#pragma unroll
            for (int u = 0; u < kMine; ++u)
                if (place[u] >= 0 && own[u] >= limit) {
                    const bool far = place[u] / 4 >= near;
                    const int of = far ? quads - near : near, run = (of + kThreads - 1) / kThreads * 32;
                    atomicAdd(own[u] > limit ? &above[far][(place[u] / 4 - (far ? near : 0)) / run] : &ties[far][(place[u] / 4 - (far ? near : 0)) / run], 1);
                }
        }
        __syncthreads();
        // Rows above the limit stay, and the first `need` at it: mostly all of those
        auto in_runs = [&](const int (&of)[2][32], int part) {  // before the warp's run of that part
            return __reduce_add_sync(0xffffffffu, (part || lane < warp ? of[0][lane] : 0) + (part && lane < warp ? of[1][lane] : 0));
        };
        auto write = [&](auto all_stay) {
            constexpr bool kAllStay = decltype(all_stay)::value;
            auto stays = [&](uint32_t order) { return kAllStay ? order >= limit : order > limit; };
#pragma unroll 1
            for (int part = 0; part < 2; ++part) {
                int from, to;
                run_of(part, from, to);
                if (from >= to) continue;
                const int ties_before = in_runs(ties, part);
                int out = s.sinks + in_runs(above, part) + (kAllStay ? ties_before : 0), tied = ties_before;
#pragma unroll 1
                for (int q0 = from; q0 < to; q0 += 32 * kAtOnce) {
                    uint4 o[kAtOnce];
                    load(part, q0, to, o);
                    uint32_t ups = 0, ats = 0;          // how many of a turn, a byte for each (up to 128 rows of one)
                    uint32_t up_bits = 0, at_bits = 0;  // which of the lane's
#pragma unroll
                    for (int u = 0; u < kAtOnce; ++u) {
                        const uint32_t each[4] = {o[u].x, o[u].y, o[u].z, o[u].w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (stays(each[i])) up_bits |= 1u << (4 * u + i);
                            if (!kAllStay && each[i] == limit) at_bits |= 1u << (4 * u + i);
                        }
                        ups |= (uint32_t)__popc(up_bits >> 4 * u & 15) << 8 * u;
                        if (!kAllStay) ats |= (uint32_t)__popc(at_bits >> 4 * u & 15) << 8 * u;
                    }
                    const uint32_t ups_upto = inclusive_scan(ups, lane), ups_all = __shfl_sync(0xffffffffu, ups_upto, 31);
                    uint32_t ats_upto = 0, ats_all = 0;
                    if (!kAllStay) {
                        ats_upto = inclusive_scan(ats, lane);
                        ats_all = __shfl_sync(0xffffffffu, ats_upto, 31);
                    }
#pragma unroll
                    for (int u = 0; u < kAtOnce; ++u) {
                        uint32_t stay = up_bits >> 4 * u & 15;
                        int place = out + ((ups_upto - ups) >> 8 * u & 255);
                        if (!kAllStay) {
                            const int tie = tied + ((ats_upto - ats) >> 8 * u & 255);
                            uint32_t at_it = at_bits >> 4 * u & 15;
                            while (__popc(at_it) > max(need - tie, 0)) at_it &= ~(1u << (31 - __clz(at_it)));  // (the first ones stay)
                            stay |= at_it;
                            place += min(tie, need);
                        }
                        int32_t* put = rows + place;
                        const int first = s.sinks + 4 * (q0 + 32 * u + lane);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (stay >> i & 1) *put++ = first + i;
                        out += ups_all >> 8 * u & 255;
                        tied += ats_all >> 8 * u & 255;
                    }
                }
            }
        };
        if (__reduce_add_sync(0xffffffffu, ties[0][lane] + ties[1][lane]) == need) write(std::true_type());
        else write(std::false_type());
    }
    for (int r = t; r < s.sinks; r += kThreads) rows[r] = r;
    for (int r = t; r < s.recent; r += kThreads) rows[s.keep - s.recent + r] = n - s.recent + r;
    if (s.kept == nullptr) return;
    // In their order: weights to come lie behind those that have been written
    float* const put = s.kept + at;
    for (int r0 = 0; r0 < s.keep; r0 += kSelectAhead * kThreads) {
        float x[kSelectAhead];
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kSelectAhead; ++u) {
            const int r = r0 + u * kThreads + t;
            x[u] = r < s.keep ? w[rows[r]] : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kSelectAhead; ++u) {
            const int r = r0 + u * kThreads + t;
            if (r < s.keep) put[r] = x[u];
        }
    }
}

// ---- rows that stay, to the front ------------------------------------------------------------ //
// A block takes one head's rows of one cache, or a part of their columns, in their order, some at a time: all of them have been
// read before the first is written.  Later rows come from behind what is written, so the next ones are on their way meanwhile:
// copies into shared memory, of which each thread writes what it has fetched itself.  Where rows come from travels the same way,
// some steps further ahead.
// Memory bounds it, at 6.0 TB/s in pieces of 256 bytes (448 heads, 1024 rows of each cache: 80 us) and 5.0 in pieces of 128, a kilobyte apart
// (128 heads, 8192 rows: 108 us).
constexpr int kMoveThreads = 256, kMoveRows = 4, kMoveStages = 4, kMoveFrom = 8, kMoveBytes = kMoveStages * kMoveRows * kMoveThreads * 16;

__global__ void __launch_bounds__(kMoveThreads) move_kernel(const MkbsMove m, const int parts) {
    extern __shared__ uint4 fetched[];  // [stage][row][thread], then the places that rows come from
    const int lanes = m.head_bytes / 16 / parts, part = blockIdx.x % parts, which = blockIdx.x / parts % 2, head = blockIdx.x / parts / 2;
    const int b = blockIdx.y, layer = blockIdx.z;
    char* const cache = static_cast<char*>(which ? m.caches[1] : m.caches[0]);
    if (cache == nullptr) return;
    const int n = length_of(m.lengths, m.length, m.positions, b), kept = min(n, m.keep);
    const int32_t* const rows = m.rows + (((int64_t)layer * m.sequences + b) * m.kv_heads + head) * m.keep;
    const int per = kMoveThreads / lanes, mine = threadIdx.x / lanes, u = threadIdx.x - mine * lanes, step = per * kMoveRows, steps = (kept + step - 1) / step;
    const int64_t row_bytes = (int64_t)m.kv_heads * m.head_bytes;
    char* const base = cache + layer * m.c_layer + b * m.c_sequence + (int64_t)head * m.head_bytes + (part * lanes + u) * 16;
    int32_t* const from = reinterpret_cast<int32_t*>(reinterpret_cast<char*>(fetched) + kMoveBytes);  // [step % kMoveFrom][row]
    auto look_up = [&](int i) {
        for (int r = threadIdx.x; r < step && i * step + r < kept; r += kMoveThreads)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(mkb::smem_u32(from + i % kMoveFrom * step + r)), "l"(rows + i * step + r) : "memory");
    };
    uint32_t moving = 0;  // four bits a step, the one fetched last lowest
    auto fetch = [&](int i) {
        moving <<= kMoveRows;
#pragma unroll
        for (int k = 0; k < kMoveRows; ++k) {
            const int r = i * step + k * per + mine;
            if (mine >= per || r >= kept) continue;
            const int source = from[i % kMoveFrom * step + k * per + mine];
            if (source <= r || source >= n) continue;  // (it stays: rows before r may have been written)
            moving |= 1u << k;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mkb::smem_u32(fetched + (i % kMoveStages * kMoveRows + k) * kMoveThreads + threadIdx.x)),
                         "l"(base + source * row_bytes)
                         : "memory");
        }
    };
    auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    for (int i = 0; i < kMoveFrom - 1; ++i) look_up(i);
    commit();
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    for (int i = 0; i < kMoveStages - 1; ++i) {
        fetch(i);
        commit();
    }
    for (int i = 0; i < steps; ++i) {
        fetch(i + kMoveStages - 1);
        look_up(i + kMoveFrom - 1);
        commit();
        asm volatile("cp.async.wait_group %0;" ::"n"(kMoveStages - 1) : "memory");
        __syncthreads();  // everybody has fetched step i and looked step i + 4 up, which is fetched next
        const uint32_t moves = moving >> kMoveRows * (kMoveStages - 1);
#pragma unroll
        for (int k = 0; k < kMoveRows; ++k)
            if (moves >> k & 1)
                *reinterpret_cast<uint4*>(base + (int64_t)(i * step + k * per + mine) * row_bytes) = fetched[(i % kMoveStages * kMoveRows + k) * kMoveThreads + threadIdx.x];
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}
static_assert(kMoveRows * kMoveStages <= 32, "bits of `moving`");
static_assert(kMoveFrom >= 2 * kMoveStages, "a step is looked up and the block has met before it is fetched");

template <typename V>
cudaError_t reorder(const ReorderArgs& a, cudaStream_t s) {
    if (const cudaError_t e = allow_shared_memory<reorder_kernel<V>>(); e != cudaSuccess) return e;
    reorder_kernel<V><<<2 * kSms, kReorderThreads, kReorderBytes, s>>>(a);
    return cudaGetLastError();
}

template <int kThreads>
cudaError_t select(const MkbsSelect& a, int fit, cudaStream_t s) {
    if (const cudaError_t e = allow_shared_memory<select_kernel<kThreads>>(); e != cudaSuccess) return e;
    select_kernel<kThreads><<<dim3(a.kv_heads, a.sequences, a.layers), kThreads, fit * 4, s>>>(a, fit);
    return cudaGetLastError();
}

}  // namespace

cudaError_t reorder_launch(const MkbsReorder& r, cudaStream_t s) {
    ReorderArgs a{r.slots, r.num_regions, r.first, r.parents, r.lengths, r.status, {}};
    uintptr_t bits = 0;  // what every address and size is a multiple of
    for (int i = 0; i < r.num_regions; ++i) {
        const MkbsRegion& g = a.regions[i] = r.regions[i];
        bits |= reinterpret_cast<uintptr_t>(g.base) | (uintptr_t)g.outer_stride | (uintptr_t)g.slot_stride | (uintptr_t)g.row_bytes;
    }
    if (bits % 16 != 0) return bits % 4 == 0 ? reorder<uint32_t>(a, s) : reorder<uint8_t>(a, s);
    if (const cudaError_t e = allow_shared_memory<reorder_bulk_kernel>(); e != cudaSuccess) return e;
    reorder_bulk_kernel<<<kSms, r.slots <= 32 ? 32 : kReorderThreads, kStages * kStageBytes + 128, s>>>(a);
    return cudaGetLastError();
}

cudaError_t select_launch(const MkbsSelect& a, cudaStream_t s) {
    const int longest = a.lengths != nullptr ? a.positions : a.length, fit = longest <= a.keep ? 0 : longest < kMostOrders ? (longest + 3) / 4 * 4 : kMostOrders;
    // Few warps for few rows: 512 blocks of 4096 rows take 11.8, 17.4, 31.8 us with 256, 512 and 1024 threads, 8 blocks 6.7, 6.7, 8.9; of 16384
    // rows 31, 30, 37 and 11.8, 10.9, 9.8; of 32768 rows 73, 56, 52 and 18.6, 14.6, 14.2
    return fit <= 8192 ? select<256>(a, fit, s) : fit <= 16384 ? select<512>(a, fit, s) : select<1024>(a, fit, s);
}

cudaError_t move_launch(const MkbsMove& m, cudaStream_t s) {
    // A block and more for every SM, none with less than 32 bytes of a row, a sector (64 blocks of 256-byte rows, 512 of 1500 kept: with
    // 1, 2, 4 parts 14.4, 11.9, 11.4 us with the selection as it was then; 256 blocks of 128-byte rows, 8192 of 65001: 152, 157, 160)
    int parts = 1;
    while (m.kv_heads * 2 * m.sequences * m.layers * parts < kSms && m.head_bytes % (64 * parts) == 0) parts *= 2;
    if (const cudaError_t e = allow_shared_memory<move_kernel>(); e != cudaSuccess) return e;
    move_kernel<<<dim3(2 * m.kv_heads * parts, m.sequences, m.layers), kMoveThreads, kMoveBytes + kMoveFrom * 4 * kMoveRows * (kMoveThreads / (m.head_bytes / 16 / parts)), s>>>(m, parts);
    return cudaGetLastError();
}

}  // namespace mkbs
