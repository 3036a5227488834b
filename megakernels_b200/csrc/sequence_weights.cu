// The softmax weight that a run of queries gives each cached key, summed over the queries and the heads that share the key:
//   w[j] += sum_r exp2(z_rj - log2 sum_i exp2 z_ri),  z = scale log2(e) q k,  r = (query, head of the group).
// Two passes over the scores, since a row's sum has to be known before its share of a key's weight is.
//
// More than 16 rows: scores on tcgen05.mma, both passes, in one kernel of a block per SM that goes from unit to unit of work.
//   rows   a unit is 128 rows of queries (M) and a run of keys, 128 at a time: a thread has a row and a quarter of its keys, and keeps their
//          sum; where there are few rows their keys are several units, and a small launch joins the parts;
//   keys   a unit is 128 keys (M) and a run of rows, 128 at a time: a thread has a key and a quarter of the rows, so that a key's weight is a
//          sum in registers; where there are few keys their rows are several units, and a small launch adds the parts.
// The exponentials bound both (16 a clock and SM: 0.54 us for 128 x 128 scores at 1.9 GHz, products 0.07 - 0.13).  Sums of a row refer to a
// maximum that is looked for in a row's first keys only, and again where a sum gets too large.  Measured: 39.1 us for 1501 queries on 1501
// keys (32 heads of 64, exponentials of the causal half 16 us; a cluster per tile instead 59), 57.6 us for 64 queries on 32768 keys (32 heads
// of 128, exponentials 30 us).  A step of 128 x 128 takes 1,400 cycles: the warps that sum 1,050 of exponentials and 250 of waits and loads, the warp
// that issues products 580 (64 for each of eight: both operands come from shared memory) and 400 of waits, so that either is near the other's time.
// Steps: warps of a scheduler need not meet at a unit's end (-5 us), one warp finds the units (-2), chosen lanes of whole warps issue (-0.5).
// No gain: twice the columns a thread (57 and 78 us then), a polynomial for every fourth exponential, halves of a step's columns loaded while the
// others are summed (59.5), waits that poll (64).
// Up to 16 rows (a token's heads): the keys' traffic bounds it.  They are read once, straight into mma.sync fragments; the products go
// through memory (4 bytes a row where a key has 128 or 256), not yet scaled: with scaled scores, rounded before a row's logarithm was taken
// from them, large scores lost a weight's last digits (1.4e-3 of it at scores of 2^15; 20.4 us instead of 20.7 for 4 rows, 33.5 instead of 33.0 for 15).  One query on 65001 keys (32 heads of 64, 8 of keys): 21.7 us, 3.3 TB/s.  Blocks
// that all fit the SMs at once: 26.6 -> 22.9 us against four per SM, of which three fit; the sum's loads issued together and before the
// statistics: 21.3; heads of the same keys in neighbouring blocks: 21.0.  Twice the loads of a warp, or two batches in turn: 24.
#include <cfloat>

#include "hybrid_kernels.h"
#include "hybrid_tcgen05.cuh"
#include "sequence_kernels.h"

namespace mkbs {
namespace {

using namespace mkbh;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 128, kSlab = kTile * 128;  // a slab: 128 rows of 64 bf16
constexpr int kWarps = 16, kShares = kWarps / 4, kCols = kTile / kShares, kThreads = 64 + 32 * kWarps;  // softmax warps, columns of a thread
constexpr int kBuffers = 4;                      // of 128 columns of tensor memory
constexpr int kFew = 16;                         // rows of a fragment

struct WeightArgs {
    int sequences, queries, heads, kv_heads, positions, length, per, rows;
    int row_tiles, key_tiles, splits;   // key_tiles: of the longest sequence that there may be; units of a row tile
    int chunk, parts, items;            // row tiles of a unit, units of a key tile
    float scale;  // to base 2
    const int32_t* lengths;
    const bf16 *q, *k;
    int64_t q_layer, q_sequence, k_layer, k_sequence;
    float* weights;
    int64_t w_layer, w_sequence, w_head;
    float2* stats;  // [item][row tile][split][128]: maximum and sum;  few rows: [item][split][16]
    float* offs;    // [item][row tile][128]: log2 of a row's sum, infinite where a row sees no key or there is no row
    float* sums;    // [item][part][key tile][128]: weights, where there are parts
    float* scores;  // few rows: products, [item][position][row], rows rounded up to 4, 8 or 16
    float hidden;   // the product of a key that a row does not see: minus infinity when scaled
    int* status;
    unsigned long long timeout_ns;
};
struct Item {
    int g, b, layer, n;
    __device__ __forceinline__ Item(const WeightArgs& a, int item)
        : g(item), b(0), layer(0) {
        if (a.items != a.kv_heads) {
            b = item / a.kv_heads;
            g = item - b * a.kv_heads;
            layer = b / a.sequences;
            b -= layer * a.sequences;
        }
        n = length_of(a.lengths, a.length, a.positions, b);
    }
    __device__ __forceinline__ float* weights(const WeightArgs& a) const { return a.weights + layer * a.w_layer + b * a.w_sequence + g * a.w_head; }
};

// (not a number stays that)
__device__ __forceinline__ float off_of(float top, float sum) { return sum == 0.f ? INFINITY : top + log2f(sum); }
// (maximum, sum) of two parts
__device__ __forceinline__ float2 join(float2 a, float2 b) {
    const float top = fmaxf(a.x, b.x);
    if (top == -INFINITY) return make_float2(top, 0.f);
    return make_float2(top, a.y * fast_exp2(a.x - top) + b.y * fast_exp2(b.x - top));
}

// ---- scores on tcgen05 ----------------------------------------------------------------------- //
struct WeightMaps {
    CUtensorMap q, k;  // [dim, heads, queries, sequences, layers], [kv_heads * dim, positions, sequences, layers]
};
__device__ __forceinline__ void load_keys(uint32_t dst, const CUtensorMap* map, const Item& it, int dim, int row, uint32_t bar) {
    for (int i = 0; i < dim / 64; ++i)
        asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst + i * kSlab),
                     "l"(map), "r"(it.g * dim + i * 64), "r"(row), "r"(it.b), "r"(it.layer), "r"(bar)
                     : "memory");
}
// (rows of 64 columns, heads of a query next to each other)
__device__ __forceinline__ void load_queries(uint32_t dst, const CUtensorMap* map, const Item& it, int dim, int per, int query, uint32_t bar) {
    for (int i = 0; i < dim / 64; ++i)
        asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst + i * kSlab),
                     "l"(map), "r"(i * 64), "r"(it.g * per), "r"(query), "r"(it.b), "r"(it.layer), "r"(bar)
                     : "memory");
}

constexpr int kUnits = 8;  // that are described ahead.  Two operands are held, and scores wait in kBuffers buffers, so no warp is further behind
static_assert(kUnits >= kBuffers + 3, "units between the copies and the last warp that sums");
// Shared memory: two operands of units, a ring of operands of their steps with 512 bytes each, units.
template <int kDim>
struct Smem {
    static constexpr int kOperand = kDim / 64 * kSlab, kExtra = 512, kHeld = 2;
    static constexpr int stages = kDim == 64 ? 6 : 4;
    static constexpr int ring = kHeld * kOperand, extra = ring + stages * kOperand, cross = extra + stages * kExtra;
    static constexpr int units = cross + 2 * kShares * kTile * 8, bars = units + kUnits * 32;
    static constexpr int ctl = bars + (2 * kHeld + 2 * stages + 2 * kBuffers + 4 + kUnits) * 8, total = ctl + 16 + 1024;
    static_assert(total <= 227 * 1024 - kStaticShared, "shared memory of a block");
};

// A unit of work: a tile held, and tiles of the other operand, first .. first + count - 1.
template <bool kKeys>
struct Unit {
    int item, tile, part, first, count;
    static __host__ __device__ uint32_t all(const WeightArgs& a) { return (uint32_t)a.items * (kKeys ? a.key_tiles * a.parts : a.row_tiles * a.splits); }
    // A block's `turn`-th unit: the longest come first and are dealt out to and fro; none: the turn is over
    __device__ __forceinline__ bool find(const WeightArgs& a, uint32_t turn) {
        uint32_t u = turn * gridDim.x + (turn & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        if (turn * gridDim.x >= all(a)) return false;
        count = 0, first = -1;  // (no unit)
        if (u >= all(a)) return true;
        const uint32_t parts = kKeys ? a.parts : a.splits, rest = u / a.items;
        item = (int)(u - rest * a.items);
        tile = parts == 1 ? rest : rest / parts;
        part = (int)(rest - tile * parts);
        const int of_tile = kTile / a.per, before = Item(a, item).n - a.queries;  // (query t sees rows 0 .. before + t)
        if (kKeys) {  // the first tile has the most rows
            first = part * a.chunk;
            if (tile * kTile > before) first += (tile * kTile - before) / of_tile;
            if (tile * kTile < before + a.queries) count = max(min(a.chunk, a.row_tiles - first), 0);
        } else {  // the last tile has the most keys
            tile = a.row_tiles - 1 - tile;
            const int tiles = (max(before + min((tile + 1) * of_tile, a.queries), 0) + kTile - 1) / kTile;
            first = parts == 1 ? 0 : (int)((uint64_t)tiles * part / parts);
            count = (parts == 1 ? tiles : (int)((uint64_t)tiles * (part + 1) / parts)) - first;
        }
        return true;
    }
};

template <int kDim, bool kKeys>
__global__ void __launch_bounds__(kThreads, 1) weights_kernel(const __grid_constant__ WeightMaps maps, const WeightArgs a) {
    extern __shared__ uint8_t raw[];
    using S = Smem<kDim>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t raw32 = mkb::smem_u32(raw), base = (raw32 + 1023u) & ~1023u;
    char* const at = reinterpret_cast<char*>(raw) + (base - raw32);
    volatile int* const ctl = reinterpret_cast<volatile int*>(at + S::ctl);  // [0] dead, [1] tensor memory
    auto bar = [&](int i) { return base + S::bars + i * 8; };
    auto held_full = [&](int i) { return bar(i & 1); };
    auto held_empty = [&](int i) { return bar(2 + (i & 1)); };
    auto full = [&](int t) { return bar(4 + t % S::stages); };
    auto empty = [&](int t) { return bar(4 + S::stages + t % S::stages); };
    auto scored = [&](int t) { return bar(4 + 2 * S::stages + t % kBuffers); };
    auto read = [&](int t) { return bar(4 + 2 * S::stages + kBuffers + t % kBuffers); };
    auto meeting = [&](int i) { return bar(4 + 2 * S::stages + 2 * kBuffers + i); };
    auto described = [&](int u) { return bar(4 + 2 * S::stages + 2 * kBuffers + 4 + u % kUnits); };
    auto held = [&](int i) { return base + (i & 1) * S::kOperand; };
    auto stage = [&](int t) { return base + S::ring + t % S::stages * S::kOperand; };
    auto wait = [&](uint32_t b, int turn, int role) { return tc_wait(b, (uint32_t)turn & 1u, ctl, a.timeout_ns, a.status, role); };
    auto wait_all = [&](uint32_t b, int turn) { return __all_sync(0xffffffffu, wait(b, turn, 2)); };

    if (threadIdx.x < 2) asm volatile("prefetch.tensormap [%0];" ::"l"(threadIdx.x ? &maps.k : &maps.q) : "memory");
    if (kTile % a.per != 0) {  // rows that the copies leave out are finite
        for (int i = threadIdx.x; i < S::extra / 16; i += kThreads) reinterpret_cast<uint4*>(at)[i] = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) mkb::mbar_init(held_full(i), 1), mkb::mbar_init(held_empty(i), 1);
        for (int i = 0; i < S::stages; ++i) mkb::mbar_init(full(i), 1), mkb::mbar_init(empty(i), kKeys ? 1 + kWarps : 1);
        for (int i = 0; i < kBuffers; ++i) mkb::mbar_init(scored(i), 1), mkb::mbar_init(read(i), kWarps);
        for (int i = 0; i < 4; ++i) mkb::mbar_init(meeting(i), kShares);
        for (int i = 0; i < kUnits; ++i) mkb::mbar_init(described(i), 1);
        ctl[0] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    // (the copies begin while the others get the tensor memory)
    uint32_t tmem = 0;
    if (warp > 0) {
        if (warp == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + S::ctl + 4), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
        tc_before_sync();
        asm volatile("bar.sync 1, %0;" ::"n"(kThreads - 32) : "memory");
        tc_after_sync();
        tmem = (uint32_t)ctl[1];
        let_next();  // (not before: a block of the next launch that held tensor memory would wait for this one, and this one for the memory)
        if (kKeys) after_previous();  // (the limit of waits is not for the launch before this one)
    }

    const int of_tile = kTile / a.per, box_bytes = kDim / 64 * of_tile * a.per * 128;
    // (Both roles run as whole warps with a chosen lane: on one lane of a diverged warp every operand of an instruction of this kind is
    // first moved to a uniform register.)
    auto wait_whole = [&](uint32_t b, int turn, int role) { return __all_sync(0xffffffffu, wait(b, turn, role)); };
    if (warp == 0) {
        const bool chosen = tc_elect();
        bool ok = true;
        int t = 0, u = 0;
        Unit<kKeys> unit = {};
        auto describe = [&] {  // unit u, for the other warps; (what the place held before has been read, as held_empty says)
            if (chosen) {
                int4* const to = reinterpret_cast<int4*>(at + S::units + u % kUnits * 32);
                to[0] = make_int4(unit.item, unit.tile, unit.part, unit.first);
                to[1].x = unit.count;
                mkb::mbar_arrive(described(u));
            }
            __syncwarp();
        };
        for (uint32_t turn = 0; ok && unit.find(a, turn); ++turn) {
            if (unit.count == 0) {
                if (!kKeys && unit.first >= 0) {  // rows without a key here
                    const int64_t row_tile = (int64_t)unit.item * a.row_tiles + unit.tile;
                    for (int i = lane; i < kTile; i += 32)
                        if (a.splits > 1) a.stats[(row_tile * a.splits + unit.part) * kTile + i] = make_float2(-INFINITY, 0.f);
                        else a.offs[row_tile * kTile + i] = INFINITY;
                }
                continue;
            }
            const Item it(a, unit.item);
            ok = wait_whole(held_empty(u), (u >> 1) ^ 1, 0);
            if (!ok) break;
            describe();
            if (chosen) {
                mkb::mbar_expect_tx(held_full(u), kKeys ? S::kOperand : box_bytes);
                if (kKeys) load_keys(held(u), &maps.k, it, kDim, unit.tile * kTile, held_full(u));
                else load_queries(held(u), &maps.q, it, kDim, a.per, unit.tile * of_tile, held_full(u));
            }
            __syncwarp();
            ++u;
            auto rows = [&](int step, int n) {
                mkb::mbar_expect_tx(full(step), box_bytes + S::kExtra);
                load_queries(stage(step), &maps.q, it, kDim, a.per, n * of_tile, full(step));
            };
            int begun = 0;
            if (kKeys && u == 1) {  // keys and queries are there; the offsets are the launch before's
                begun = min(unit.count, S::stages);
                if (chosen)
                    for (int i = 0; i < begun; ++i) rows(i, unit.first + i);
                __syncwarp();
                after_previous();
            }
            for (int i = 0; i < unit.count; ++i, ++t) {
                const int n = unit.first + i;
                if (i >= begun) ok = wait_whole(empty(t), t / S::stages ^ 1, 0);
                if (!ok) break;
                if (chosen && kKeys) {
                    if (i >= begun) rows(t, n);
                    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                     base + S::extra + t % S::stages * S::kExtra),
                                 "l"(a.offs + ((int64_t)unit.item * a.row_tiles + n) * kTile), "r"(S::kExtra), "r"(full(t))
                                 : "memory");
                } else if (chosen) {
                    mkb::mbar_expect_tx(full(t), S::kOperand);
                    load_keys(stage(t), &maps.k, it, kDim, n * kTile, full(t));
                }
                __syncwarp();
            }
        }
        if (kKeys && u == 0) after_previous();  // (a launch does not end before the one before it)
        ok = ok && wait_whole(held_empty(u), (u >> 1) ^ 1, 0);
        unit.count = 0;  // (no more)
        if (ok) describe();
        // no copy may be in flight when the block's shared memory goes away
        for (int i = max(u - 2, 0); i < u; ++i) tc_wait(held_full(i), (uint32_t)(i >> 1) & 1u, nullptr, a.timeout_ns, a.status, 0);
        for (int i = max(t - S::stages, 0); i < t; ++i) tc_wait(full(i), (uint32_t)(i / S::stages) & 1u, nullptr, a.timeout_ns, a.status, 0);
    } else if (warp == 1) {
        const bool chosen = tc_elect();
        const uint32_t desc = tc_idesc(kTile, kTile);
        bool ok = true;
        int t = 0, u = 0;
        for (;;) {
            ok = wait_whole(described(u), u / kUnits, 1);
            const int count = ok ? *reinterpret_cast<const volatile int*>(at + S::units + u % kUnits * 32 + 16) : 0;
            if (count == 0) break;
            ok = wait_whole(held_full(u), u >> 1, 1);
            for (int n = 0; n < count && ok; ++n, ++t) {
                ok = wait_whole(full(t), t / S::stages, 1) && wait_whole(read(t), t / kBuffers ^ 1, 1);
                if (!ok) break;
                tc_after_sync();
                if (chosen) {
                    const uint64_t of_held = tc_desc(held(u)), of_stage = tc_desc(stage(t));
#pragma unroll
                    for (int slab = 0; slab < kDim / 64; ++slab)
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)  // (32 bytes on: the address is in units of 16, and does not carry beyond its field)
                            tc_mma(tmem + t % kBuffers * kTile, of_held + (slab * kSlab + kk * 32) / 16, of_stage + (slab * kSlab + kk * 32) / 16, desc,
                                   (uint32_t)((slab | kk) != 0));
                    tc_commit(empty(t));
                    if (n == count - 1) tc_commit(held_empty(u));
                    tc_commit(scored(t));
                }
                __syncwarp();
            }
            if (!ok) break;
            ++u;
        }
    } else if (warp >= 2) {
        const int quarter = warp & 3, share = (warp - 2) >> 2, lanes = quarter * 32 + lane;  // (a warp may touch 32 lanes of tensor memory)
        bool ok = true;
        int t = 0, u = 0;
        auto scores = [&](uint32_t (&x)[kCols]) {  // the thread's, of step t
            static_assert(kCols == 32, "one load of 32 columns");
            tc_load32(tmem + ((uint32_t)(quarter * 32) << 16) + t % kBuffers * kTile + share * kCols, x);
            tc_before_sync();
            __syncwarp();
            if (lane == 0) mkb::mbar_arrive(read(t));
        };
        Unit<kKeys> unit, last_unit = {};
        auto cross = [&](int i) { return reinterpret_cast<float2*>(at + S::cross) + (i & 1) * kShares * kTile + lanes; };
        auto join_last = [&] {  // of unit u - 1
            if (u == 0) return true;
            if (!wait_all(meeting(quarter), u - 1)) return false;
            if (share != (u & (kShares - 1))) return true;  // (in turn)
            const float2* const from = cross(u - 1);
            const Item it(a, last_unit.item);
            if constexpr (kKeys) {
                float sum = from[0].y;
#pragma unroll
                for (int c = 1; c < kShares; ++c) sum += from[c * kTile].y;
                const int j = last_unit.tile * kTile + lanes;
                if (a.parts > 1) a.sums[(((int64_t)last_unit.item * a.parts + last_unit.part) * a.key_tiles + last_unit.tile) * kTile + lanes] = sum;
                else if (j < it.n) atomicAdd(it.weights(a) + j, sum);  // (nothing else adds to it: an addition that nobody waits for)
            } else {
                const bool there = lanes < of_tile * a.per && last_unit.tile * of_tile * a.per + lanes < a.rows;
                float2 all = make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int c = 0; c < kShares; ++c)
                    if (there) all = join(all, from[c * kTile]);
                const int64_t row_tile = (int64_t)last_unit.item * a.row_tiles + last_unit.tile;
                if (a.splits > 1) a.stats[(row_tile * a.splits + last_unit.part) * kTile + lanes] = all;
                else a.offs[row_tile * kTile + lanes] = off_of(all.x, all.y);
            }
            return true;
        };
        for (;;) {
            ok = wait_all(described(u), u / kUnits);
            if (!ok) break;
            {
                const volatile int* const from = reinterpret_cast<const volatile int*>(at + S::units + u % kUnits * 32);
                unit.item = from[0], unit.tile = from[1], unit.part = from[2], unit.first = from[3], unit.count = from[4];
            }
            if (unit.count == 0) break;
            const Item it(a, unit.item);
            const int before = it.n - a.queries;
            float2 mine = make_float2(-INFINITY, 0.f);  // rows: maximum and sum; keys: x is not used
            if constexpr (kKeys) {
                const int j = unit.tile * kTile + lanes;
                const int first_row = max(unit.tile * kTile + quarter * 32 - before, 0) * a.per, own_row = max(j - before, 0) * a.per, last_row = max(unit.tile * kTile + quarter * 32 + 31 - before, 0) * a.per;  // the first that sees it
                float s4[4] = {0.f, 0.f, 0.f, 0.f};
                for (int n = 0; n < unit.count; ++n, ++t) {
                    const int r0 = (unit.first + n) * of_tile * a.per + share * kCols;
                    ok = wait_all(scored(t), t / kBuffers) && wait_all(full(t), t / S::stages);
                    if (!ok) break;
                    tc_after_sync();
                    uint32_t x[kCols];
                    scores(x);
                    const float4* const off = reinterpret_cast<const float4*>(at + S::extra + t % S::stages * S::kExtra) + share * (kCols / 4);
                    if (last_row <= r0) {
#pragma unroll
                        for (int c = 0; c < kCols / 4; ++c) {
                            const float4 o = off[c];
                            s4[0] += fast_exp2(fmaf(__uint_as_float(x[4 * c]), a.scale, -o.x));
                            s4[1] += fast_exp2(fmaf(__uint_as_float(x[4 * c + 1]), a.scale, -o.y));
                            s4[2] += fast_exp2(fmaf(__uint_as_float(x[4 * c + 2]), a.scale, -o.z));
                            s4[3] += fast_exp2(fmaf(__uint_as_float(x[4 * c + 3]), a.scale, -o.w));
                        }
                    } else if (first_row < r0 + kCols) {
                        const int hidden = own_row - r0;  // columns before that do not see the key
#pragma unroll
                        for (int c = 0; c < kCols / 4; ++c) {
                            const float4 o = off[c];
                            const float p[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float y = fast_exp2(fmaf(__uint_as_float(x[4 * c + e]), a.scale, -p[e]));
                                s4[e] += 4 * c + e >= hidden ? y : 0.f;
                            }
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mkb::mbar_arrive(empty(t));
                }
                mine.y = (s4[0] + s4[1]) + (s4[2] + s4[3]);
            } else {
                const int r0 = unit.tile * of_tile * a.per, have = min(of_tile * a.per, a.rows - r0), warp_row = quarter * 32;
                const int last = before + (r0 + lanes) / a.per, warp_last = before + (r0 + warp_row) / a.per, warp_end = before + (r0 + warp_row + 31) / a.per;
                for (int n = 0; n < unit.count; ++n, ++t) {
                    ok = wait_all(scored(t), t / kBuffers);
                    if (!ok) break;
                    tc_after_sync();
                    uint32_t x[kCols];
                    scores(x);
                    const int j0 = (unit.first + n) * kTile + share * kCols;
                    if (warp_row >= have || j0 > warp_end) continue;  // no row sees any of these keys
                    const bool whole = j0 + kCols - 1 <= warp_last;  // every row sees all of these keys
                    if (whole && __all_sync(0xffffffffu, mine.x > -INFINITY)) {
                        float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int c = 0; c < kCols; ++c) s4[c & 3] += fast_exp2(fmaf(__uint_as_float(x[c]), a.scale, -mine.x));
                        const float sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
                        if (__all_sync(0xffffffffu, sum < 0x1p100f)) {
                            mine.y += sum;
                            continue;
                        }
                    }
                    float top = mine.x, sum = 0.f;
#pragma unroll
                    for (int c = 0; c < kCols; ++c) {
                        const float z = j0 + c <= last ? __uint_as_float(x[c]) * a.scale : -INFINITY;
                        top = fmaxf(top, z);
                        x[c] = __float_as_uint(z);
                    }
                    if (top > -INFINITY) {
#pragma unroll
                        for (int c = 0; c < kCols; ++c) sum += fast_exp2(__uint_as_float(x[c]) - top);
                        mine = make_float2(top, fmaf(mine.y, fast_exp2(mine.x - top), sum));  // (0 from minus infinity)
                    }
                }
            }
            if (!ok) break;
            // The threads of a row or key: their parts are joined a unit later, so that the warps need not meet
            ok = join_last();
            if (!ok) break;
            cross(u)[share * kTile] = mine;
            __syncwarp();
            if (lane == 0) mkb::mbar_arrive(meeting(quarter));
            last_unit = unit;
            ++u;
        }
        if (ok) join_last();
    }
    tc_before_sync();
    __syncthreads();
    if (*ctl) tc_settle();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// A row's parts to the logarithm of its sum.
__global__ void __launch_bounds__(kTile) weights_join_kernel(const WeightArgs a) {
    let_next();
    after_previous();
    const float2* const parts = a.stats + (int64_t)blockIdx.x * a.splits * kTile + threadIdx.x;
    float top = -INFINITY, sum = 0.f;
    for (int i = 0; i < a.splits; ++i) top = fmaxf(top, parts[i * kTile].x);
    for (int i = 0; i < a.splits; ++i) {
        const float2 p = parts[i * kTile];
        if (p.x > -INFINITY) sum += p.y * fast_exp2(p.x - top);
    }
    a.offs[(int64_t)blockIdx.x * kTile + threadIdx.x] = off_of(top, sum);
}

// A key's parts to its weight.
__global__ void __launch_bounds__(kTile) weights_add_kernel(const WeightArgs a) {
    const Item it(a, blockIdx.y);
    const int j = blockIdx.x * kTile + threadIdx.x, of_tile = kTile / a.per;
    const int first = max((int)blockIdx.x * kTile - (it.n - a.queries), 0) / of_tile, parts = (max(a.row_tiles - first, 0) + a.chunk - 1) / a.chunk;
    after_previous();
    if (j >= it.n) return;
    float sum = 0.f;
    for (int i = 0; i < parts; ++i) sum += a.sums[(((int64_t)blockIdx.y * a.parts + i) * a.key_tiles + blockIdx.x) * kTile + threadIdx.x];
    it.weights(a)[j] += sum;
}

// ---- up to 16 rows ------------------------------------------------------------------------------ //
constexpr int kFewThreads = 256, kFewWarps = kFewThreads / 32, kAhead = 4;  // groups of 8 keys whose loads a warp has under way
constexpr int few_blocks(int dim) { return dim == 64 ? 3 : 2; }  // per SM, by their registers

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Rows are the M side, 8 keys the N side.  The contraction's order is free: lane (n, c) of a warp, n = lane / 4 and c = lane % 4, holds the
// neighbours 8 c + 32 i .. + 7 of key n, two products' worth, so a key is read in 16-byte pieces straight into fragments.
template <int kDim, int kRowsPad>
__global__ void __launch_bounds__(kFewThreads, few_blocks(kDim)) weights_few_kernel(const WeightArgs a) {
    let_next();
    constexpr int kPieces = kDim / 32;
    __shared__ float2 shared[kFewWarps][kFew];
    const Item it(a, blockIdx.x);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane / 4, c = lane % 4, before = it.n - a.queries;
    const bf16* const keys = a.k + it.layer * a.k_layer + it.b * a.k_sequence + it.g * kDim + c * 8;
    const int64_t key_row = (int64_t)a.kv_heads * kDim;
    float* const scores = a.scores + (int64_t)blockIdx.x * a.positions * kRowsPad;
    uint32_t q[kPieces][2][4];  // rows n and n + 8
    int last[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = n + 8 * h;
        last[h] = r < a.rows ? before + r / a.per : -1;
        const bf16* const row = a.q + it.layer * a.q_layer + it.b * a.q_sequence + ((int64_t)(r / a.per) * a.heads + it.g * a.per + r % a.per) * kDim + c * 8;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const uint4 w = r < a.rows ? *reinterpret_cast<const uint4*>(row + 32 * i) : make_uint4(0, 0, 0, 0);
            q[i][0][h] = w.x;
            q[i][0][2 + h] = w.y;
            q[i][1][h] = w.z;
            q[i][1][2 + h] = w.w;
        }
    }
    const int groups = (it.n + 7) / 8, total = (int)gridDim.y * kFewWarps, me = (int)blockIdx.y * kFewWarps + warp;
    const int first = (int)((int64_t)groups * me / total), end = (int)((int64_t)groups * (me + 1) / total);
    float2 stats[2] = {make_float2(-INFINITY, 0.f), make_float2(-INFINITY, 0.f)};
    for (int g0 = first; g0 < end; g0 += kAhead) {
        uint4 w[kAhead][kPieces];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int j = (g0 + u) * 8 + n;
            const bool there = g0 + u < end && j < it.n;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) w[u][i] = there ? mkb::ld_nc_v4(keys + j * key_row + 32 * i) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (g0 + u >= end) break;
            float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                mma_bf16(d, q[i][0], w[u][i].x, w[u][i].y);
                mma_bf16(d, q[i][1], w[u][i].z, w[u][i].w);
            }
            // d[0], d[1]: row n, keys 2 c and 2 c + 1;  d[2], d[3]: row n + 8
            const int j = (g0 + u) * 8 + 2 * c;
#pragma unroll
            for (int h = 0; h < kRowsPad / 8 + (kRowsPad == 4); ++h) {
                // (products, not scores, are kept: scaled and taken from a reference in one operation they are rounded once, near the result)
                const float x0 = j <= last[h] ? d[2 * h] : a.hidden, x1 = j + 1 <= last[h] ? d[2 * h + 1] : a.hidden;
                const float top = fmaxf(fmaxf(x0 * a.scale, x1 * a.scale), stats[h].x);
                if (n + 8 * h < kRowsPad) {
                    if (j < it.n) scores[(int64_t)j * kRowsPad + n + 8 * h] = x0;
                    if (j + 1 < it.n) scores[(int64_t)(j + 1) * kRowsPad + n + 8 * h] = x1;
                }
                if (top > -INFINITY)
                    stats[h] = make_float2(top, stats[h].y * fast_exp2(stats[h].x - top) + fast_exp2(fmaf(x0, a.scale, -top)) + fast_exp2(fmaf(x1, a.scale, -top)));
            }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int o = 1; o < 4; o <<= 1)
            stats[h] = join(stats[h], make_float2(__shfl_xor_sync(0xffffffffu, stats[h].x, o), __shfl_xor_sync(0xffffffffu, stats[h].y, o)));
        if (c == 0) shared[warp][n + 8 * h] = stats[h];
    }
    __syncthreads();
    if (threadIdx.x < kFew) {
        float2 all = shared[0][threadIdx.x];
        for (int i = 1; i < kFewWarps; ++i) all = join(all, shared[i][threadIdx.x]);
        a.stats[((int64_t)blockIdx.x * gridDim.y + blockIdx.y) * kFew + threadIdx.x] = all;
    }
}

template <int kRowsPad>
__global__ void __launch_bounds__(kFewThreads) weights_sum_kernel(const WeightArgs a) {
    __shared__ float2 of_row[kFew];  // its largest score, one over its sum
    const Item it(a, blockIdx.y);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float* const scores = a.scores + (int64_t)blockIdx.y * a.positions * kRowsPad;
    float* const weights = it.weights(a);
    constexpr int kBatch = 4;  // keys of a thread whose loads are under way
    const int step = gridDim.x * kFewThreads;
    float4 z[kBatch][kRowsPad / 4];
    float w[kBatch];
    auto load = [&](int64_t j) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (j + (int64_t)i * step < it.n) {
                w[i] = weights[j + i * step];
#pragma unroll
                for (int r = 0; r < kRowsPad / 4; ++r) z[i][r] = *reinterpret_cast<const float4*>(scores + (j + i * step) * kRowsPad + 4 * r);
            }
    };
    int64_t j = (int64_t)blockIdx.x * kFewThreads + threadIdx.x;
    after_previous();
    load(j);
    for (int r = warp; r < kRowsPad; r += kFewWarps) {
        const float2* const parts = a.stats + (int64_t)blockIdx.y * a.splits * kFew + r;
        float2 all = make_float2(-INFINITY, 0.f);
        for (int i = lane; i < a.splits; i += 32) all = join(all, parts[i * kFew]);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) all = join(all, make_float2(__shfl_xor_sync(0xffffffffu, all.x, o), __shfl_xor_sync(0xffffffffu, all.y, o)));
        if (lane == 0) of_row[r] = all.x == -INFINITY ? make_float2(0.f, 0.f) : make_float2(all.x, 1.f / all.y);  // (one that sees no key: no weights)
    }
    __syncthreads();
    float2 row[kRowsPad];
#pragma unroll
    for (int r = 0; r < kRowsPad; ++r) row[r] = of_row[r];
    auto add = [&](float& sum, int r, float x) { sum = fmaf(fast_exp2(fmaf(x, a.scale, -row[r].x)), row[r].y, sum); };
    while (j < it.n) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (j + (int64_t)i * step < it.n) {
                float two[2] = {0.f, 0.f};
#pragma unroll
                for (int r = 0; r < kRowsPad; r += 4) {
                    const float4 x = z[i][r / 4];
                    add(two[0], r, x.x), add(two[1], r + 1, x.y), add(two[0], r + 2, x.z), add(two[1], r + 3, x.w);
                }
                weights[j + i * step] = w[i] + (two[0] + two[1]);
            }
        j += (int64_t)kBatch * step;
        if (j < it.n) load(j);
    }
}

// ---- host ------------------------------------------------------------------------------------------ //
struct Plan {
    WeightArgs a;
    int rows_pad;
    bool few;
    size_t bytes;
    explicit Plan(const MkbsKeyWeights& w) {
        auto up = [](int n, int of) { return (n + of - 1) / of; };
        auto take = [&](size_t n) {  // bytes of the workspace
            char* const at = static_cast<char*>(w.workspace) + bytes;
            bytes += (n + 255) / 256 * 256;
            return at;
        };
        bytes = 0;
        a = {};
        a.sequences = w.sequences;
        a.queries = w.queries;
        a.heads = w.heads;
        a.kv_heads = w.kv_heads;
        a.positions = w.positions;
        a.length = w.length;
        a.lengths = w.lengths;
        a.per = w.heads / w.kv_heads;
        a.rows = w.queries * a.per;
        a.items = w.layers * w.sequences * w.kv_heads;
        a.scale = w.scale * kLog2e;
        if (a.scale == 0.f) a.scale = FLT_MIN;  // (what is hidden stays so; products below 2^100 all have the same weight)
        a.hidden = a.scale > 0.f ? -INFINITY : INFINITY;
        a.q = static_cast<const bf16*>(w.q);
        a.k = static_cast<const bf16*>(w.k);
        a.q_layer = w.q_layer, a.q_sequence = w.q_sequence, a.k_layer = w.k_layer, a.k_sequence = w.k_sequence;
        a.weights = w.weights;
        a.w_layer = w.w_layer, a.w_sequence = w.w_sequence, a.w_head = w.w_head;
        a.status = w.status;
        a.timeout_ns = w.wait_timeout_ms ? w.wait_timeout_ms * 1000000ull : kWaitNs;
        const int longest = w.lengths != nullptr ? w.positions : w.length;
        few = a.rows <= kFew;
        if (few) {
            rows_pad = a.rows <= 4 ? 4 : a.rows <= 8 ? 8 : 16;
            // blocks that fit the SMs at once, none with less than 64 keys a warp
            a.splits = few_blocks(w.dim) * kSms / a.items;
            if (a.splits > up(longest, 64 * kFewWarps)) a.splits = up(longest, 64 * kFewWarps);
            if (a.splits < 1) a.splits = 1;
            a.scores = reinterpret_cast<float*>(take((size_t)a.items * w.positions * rows_pad * 4));
            a.stats = reinterpret_cast<float2*>(take((size_t)a.items * a.splits * kFew * 8));
            return;
        }
        a.row_tiles = up(w.queries, kTile / a.per);
        a.key_tiles = longest > kTile ? up(longest, kTile) : 1;
        // as many units of rows as SMs
        a.splits = kSms / (a.items * a.row_tiles);
        a.splits = a.splits < 1 ? 1 : a.splits > a.key_tiles ? a.key_tiles : a.splits;
        // four units of keys and more for every SM, none of less than four row tiles
        a.chunk = a.row_tiles;
        while (a.chunk > 4 && (int64_t)a.items * a.key_tiles * up(a.row_tiles, a.chunk) < 4 * kSms) a.chunk = up(a.chunk, 2);
        a.parts = up(a.row_tiles, a.chunk);
        a.offs = reinterpret_cast<float*>(take((size_t)a.items * a.row_tiles * kTile * 4));
        if (a.splits > 1) a.stats = reinterpret_cast<float2*>(take((size_t)a.items * a.row_tiles * a.splits * kTile * 8));
        if (a.parts > 1) a.sums = reinterpret_cast<float*>(take((size_t)a.items * a.parts * a.key_tiles * kTile * 4));
    }
};

// 4 or 5 dimensions of bf16 with the 128-byte swizzle; what lies outside reads as zero
cudaError_t encode(CUtensorMap* map, const bf16* ptr, int dims, const cuuint64_t* size, const cuuint64_t* stride_bytes, const cuuint32_t* box) {
    EncodeFn fn = nullptr;
    if (const cudaError_t e = tc_encoder(&fn); e != cudaSuccess) return e;
    const cuuint32_t one[5] = {1, 1, 1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dims, const_cast<bf16*>(ptr), size, stride_bytes, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <int kDim>
cudaError_t launch(const MkbsKeyWeights& w, const Plan& p, cudaStream_t s) {
    const WeightArgs& a = p.a;
    WeightMaps maps;
    cudaError_t e;
    // (a dimension of one has any stride)
    const cuuint64_t q_row = (cuuint64_t)w.heads * kDim * 2, k_row = (cuuint64_t)w.kv_heads * kDim * 2;
    const cuuint64_t q_sequence = w.sequences > 1 ? w.q_sequence * 2 : q_row, q_layer = w.layers > 1 ? w.q_layer * 2 : q_row;
    const cuuint64_t k_sequence = w.sequences > 1 ? w.k_sequence * 2 : k_row, k_layer = w.layers > 1 ? w.k_layer * 2 : k_row;
    const cuuint64_t q_size[5] = {kDim, (cuuint64_t)w.heads, (cuuint64_t)w.queries, (cuuint64_t)w.sequences, (cuuint64_t)w.layers};
    const cuuint64_t q_stride[4] = {kDim * 2, q_row, q_sequence, q_layer};
    const cuuint32_t q_box[5] = {64, (cuuint32_t)a.per, (cuuint32_t)(kTile / a.per), 1, 1};
    if ((e = encode(&maps.q, a.q, 5, q_size, q_stride, q_box)) != cudaSuccess) return e;
    const cuuint64_t k_size[4] = {(cuuint64_t)w.kv_heads * kDim, (cuuint64_t)w.positions, (cuuint64_t)w.sequences, (cuuint64_t)w.layers};
    const cuuint64_t k_stride[3] = {k_row, k_sequence, k_layer};
    const cuuint32_t k_box[4] = {64, kTile, 1, 1};
    if ((e = encode(&maps.k, a.k, 4, k_size, k_stride, k_box)) != cudaSuccess) return e;
    if ((e = allow_shared_memory<weights_kernel<kDim, false>>()) != cudaSuccess) return e;
    if ((e = allow_shared_memory<weights_kernel<kDim, true>>()) != cudaSuccess) return e;
    auto blocks = [](uint32_t units) { return dim3(units < kSms ? units : kSms); };
    weights_kernel<kDim, false><<<blocks(Unit<false>::all(a)), kThreads, Smem<kDim>::total, s>>>(maps, a);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    if (a.splits > 1 && (e = launch_early(weights_join_kernel, dim3(a.items * a.row_tiles), dim3(kTile), 0, s, a)) != cudaSuccess) return e;
    e = launch_early(weights_kernel<kDim, true>, blocks(Unit<true>::all(a)), dim3(kThreads), Smem<kDim>::total, s, maps, a);
    if (e != cudaSuccess || a.parts == 1) return e;
    return launch_early(weights_add_kernel, dim3(a.key_tiles, a.items), dim3(kTile), 0, s, a);
}

template <int kDim, int kRowsPad>
cudaError_t launch_few(const Plan& p, cudaStream_t s) {
    weights_few_kernel<kDim, kRowsPad><<<dim3(p.a.items, p.a.splits), kFewThreads, 0, s>>>(p.a);
    if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
    return launch_early(weights_sum_kernel<kRowsPad>, dim3(p.a.splits, p.a.items), dim3(kFewThreads), 0, s, p.a);
}
template <int kDim>
cudaError_t choose(const MkbsKeyWeights& w, const Plan& p, cudaStream_t s) {
    if (!p.few) return launch<kDim>(w, p, s);
    return p.rows_pad == 4 ? launch_few<kDim, 4>(p, s) : p.rows_pad == 8 ? launch_few<kDim, 8>(p, s) : launch_few<kDim, 16>(p, s);
}

}  // namespace

size_t key_weights_bytes(const MkbsKeyWeights& w) { return Plan(w).bytes; }

cudaError_t key_weights_launch(const MkbsKeyWeights& w, cudaStream_t s) {
    const Plan p(w);
    return w.dim == 64 ? choose<64>(w, p, s) : choose<128>(w, p, s);
}

}  // namespace mkbs
