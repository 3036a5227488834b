// The softmax weight that a run of queries gives each cached key, summed over the queries and the heads that share the key:
//   w[j] += sum_r exp2(z_rj - log2 sum_i exp2 z_ri),  z = scale log2(e) q k,  r = (query, head of the group).
// Two passes over the scores, since a row's sum has to be known before its share of a key's weight is.
//
// More than 16 rows: scores on tcgen05.mma, both passes.
//   rows   128 rows of queries (M) x 128 keys: a thread has a row and a quarter of its keys, and keeps their running maximum and
//          sum; keys are split over blocks where there are few rows (then a small launch joins the parts);
//   keys   128 keys (M) x 128 rows: a thread has a key and a quarter of the rows, so that a key's weight is a sum in registers.  Where
//          there are few tiles of keys a cluster shares their rows.
// The exponentials bound both (16 a clock and SM: 0.54 us for 128 x 128 scores at 1.9 GHz, products 0.07 - 0.13).
// Up to 16 rows (a token's heads): the keys' traffic bounds it.  They are read once, straight into mma.sync fragments; the scores go
// through memory (4 bytes a row where a key has 128 or 256).
#include "hybrid_kernels.h"
#include "hybrid_tcgen05.cuh"
#include "sequence_kernels.h"

namespace mkbs {
namespace {

using namespace mkbh;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 128, kSlab = kTile * 128;  // a slab: 128 rows of 64 bf16
constexpr int kWarps = 16, kCols = kTile / (kWarps / 4), kThreads = 64 + 32 * kWarps;  // softmax warps, columns of a thread
constexpr int kBuffers = 4;                      // of 128 columns of tensor memory
constexpr int kFew = 16;                         // rows of a fragment

struct WeightArgs {
    int sequences, queries, heads, kv_heads, positions, length, per, rows, row_tiles, splits, shares;
    float scale;  // to base 2
    const int32_t* lengths;
    const bf16 *q, *k;
    int64_t q_layer, q_sequence, k_layer, k_sequence;
    float* weights;
    int64_t w_layer, w_sequence, w_head;
    float2* parts;  // [item][row tile][split][128]: maximum and sum;  few rows: [item][split][16]
    float* offs;    // [item][row tile][128]: log2 of a row's sum, infinite where a row sees no key or there is no row
    float* scores;  // few rows: [item][position][row], rows rounded up to 4, 8 or 16
    int* status;
    unsigned long long timeout_ns;
};
struct Item {
    int g, b, layer, n;
    __device__ __forceinline__ Item(const WeightArgs& a, int item)
        : g(item % a.kv_heads), b(item / a.kv_heads % a.sequences), layer(item / a.kv_heads / a.sequences),
          n(length_of(a.lengths, a.length, a.positions, b)) {}
    __device__ __forceinline__ float* weights(const WeightArgs& a) const { return a.weights + layer * a.w_layer + b * a.w_sequence + g * a.w_head; }
};

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
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

// Shared memory of both kernels: `held` operands of the outer loop, a ring of `stages` of the inner one's with 512 bytes each.
template <int kDim>
struct Smem {
    static constexpr int kOperand = kDim / 64 * kSlab, kExtra = 512;
    static constexpr int stages = kDim == 64 ? 6 : 4;
    static constexpr int kHeld = 2;  // (rows: one)
    int ring, extra, cross, bars, ctl, total;
    __host__ __device__ explicit Smem(bool keys) {
        ring = (keys ? kHeld : 1) * kOperand;
        extra = ring + stages * kOperand;
        cross = extra + stages * kExtra;
        bars = cross + kWarps / 4 * kTile * 8;
        ctl = bars + (2 * kHeld + 2 * stages + 2 * kBuffers + 4) * 8;
        total = ctl + 16;
    }
};
static_assert((6 + 2) * kSlab + 6 * 512 + 4096 + 2048 < 227 * 1024 - kStaticShared && (4 + 2) * 2 * kSlab + 4 * 512 + 4096 + 2048 < 227 * 1024 - kStaticShared, "shared memory of a block");

// What the roles of both kernels share.
template <int kDim, bool kKeys>
struct Block {
    using S = Smem<kDim>;
    const S sm;
    uint32_t base, tmem;
    char* at;
    volatile int* ctl;  // [0] dead, [1] tensor memory
    int warp, lane;
    unsigned long long timeout_ns;
    int* status;
    __device__ __forceinline__ uint32_t bar(int i) const { return base + sm.bars + i * 8; }
    __device__ __forceinline__ uint32_t held_full(int i) const { return bar(i); }
    __device__ __forceinline__ uint32_t held_empty(int i) const { return bar(2 + i); }
    __device__ __forceinline__ uint32_t full(int i) const { return bar(4 + i); }
    __device__ __forceinline__ uint32_t empty(int i) const { return bar(4 + S::stages + i); }
    __device__ __forceinline__ uint32_t scored(int i) const { return bar(4 + 2 * S::stages + i); }
    __device__ __forceinline__ uint32_t read(int i) const { return bar(4 + 2 * S::stages + kBuffers + i); }
    __device__ __forceinline__ uint32_t meeting(int i) const { return bar(4 + 2 * S::stages + 2 * kBuffers + i); }
    __device__ __forceinline__ uint32_t stage(int i) const { return base + sm.ring + i * S::kOperand; }
    __device__ __forceinline__ uint32_t held(int i) const { return base + i * S::kOperand; }
    __device__ __forceinline__ bool wait(uint32_t b, uint32_t parity, int role) const { return tc_wait(b, parity & 1u, ctl, timeout_ns, status, role); }
    __device__ __forceinline__ bool wait_all(uint32_t b, uint32_t parity) const { return __all_sync(0xffffffffu, wait(b, parity, 2)); }

    __device__ __forceinline__ Block(uint8_t* raw, const WeightArgs& a, bool clear)
        : sm(kKeys), warp(threadIdx.x >> 5), lane(threadIdx.x & 31), timeout_ns(a.timeout_ns), status(a.status) {
        const uint32_t raw32 = mkb::smem_u32(raw);
        base = (raw32 + 1023u) & ~1023u;
        at = reinterpret_cast<char*>(raw) + (base - raw32);
        ctl = reinterpret_cast<volatile int*>(at + sm.ctl);
        if (clear) {  // rows that the copies leave out are finite
            for (int i = threadIdx.x; i < sm.extra / 16; i += kThreads) reinterpret_cast<uint4*>(at)[i] = make_uint4(0, 0, 0, 0);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        if (threadIdx.x == 0) {
            for (int i = 0; i < 2; ++i) mkb::mbar_init(held_full(i), 1), mkb::mbar_init(held_empty(i), 1);
            for (int i = 0; i < S::stages; ++i) mkb::mbar_init(full(i), 1), mkb::mbar_init(empty(i), kKeys ? 1 + kWarps : 1);
            for (int i = 0; i < kBuffers; ++i) mkb::mbar_init(scored(i), 1), mkb::mbar_init(read(i), kWarps);
            for (int i = 0; i < 4; ++i) mkb::mbar_init(meeting(i), kWarps / 4);
            ctl[0] = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        if (warp == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + sm.ctl + 4), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
        tc_before_sync();
        __syncthreads();
        tc_after_sync();
        tmem = (uint32_t)ctl[1];
    }
    // scores of step `t`: a (M) times b (N)
    __device__ __forceinline__ void multiply(uint32_t a, uint32_t b, int t) const {
        const uint32_t desc = tc_idesc(kTile, kTile);
#pragma unroll
        for (int i = 0; i < kDim / 64; ++i)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
                tc_mma(tmem + t % kBuffers * kTile, tc_desc(a + i * kSlab + kk * 32), tc_desc(b + i * kSlab + kk * 32), desc, (uint32_t)((i | kk) != 0));
    }
    // the thread's columns of step `t`
    __device__ __forceinline__ void scores(int t, int quarter, int part, uint32_t (&x)[kCols]) const {
        static_assert(kCols == 32, "a load of 32 columns");
        tc_load32(tmem + ((uint32_t)(quarter * 32) << 16) + t % kBuffers * kTile + part * kCols, x);
        tc_before_sync();
        __syncwarp();
        if (lane == 0) mkb::mbar_arrive(read(t % kBuffers));
    }
    __device__ __forceinline__ void leave() const {
        tc_before_sync();
        __syncthreads();
        if (*ctl) tc_settle();
        if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
};

template <int kDim>
__global__ void __launch_bounds__(kThreads, 1) weights_rows_kernel(const __grid_constant__ WeightMaps maps, const WeightArgs a) {
    extern __shared__ uint8_t raw[];
    let_next();
    const Item it(a, blockIdx.z);
    const int tile = a.row_tiles - 1 - (int)blockIdx.y, of_tile = kTile / a.per, query0 = tile * of_tile, r0 = query0 * a.per;  // (the longest first)
    const int last_query = min(query0 + of_tile, a.queries) - 1, before = it.n - a.queries;  // query t sees rows 0 .. before + t
    const int tiles = (max(before + last_query + 1, 0) + kTile - 1) / kTile;
    const int first = (int)((int64_t)tiles * blockIdx.x / a.splits), count = (int)((int64_t)tiles * (blockIdx.x + 1) / a.splits) - first;
    using S = Smem<kDim>;
    const Block<kDim, false> c(raw, a, kTile % a.per != 0);
    const int box_bytes = of_tile * a.per * 128;

    float2 mine = make_float2(-INFINITY, 0.f);
    if (c.warp == 0 && c.lane == 0 && count > 0) {
        mkb::mbar_expect_tx(c.held_full(0), kDim / 64 * box_bytes);
        load_queries(c.held(0), &maps.q, it, kDim, a.per, query0, c.held_full(0));
        bool ok = true;
        int t = 0;
        for (; t < count; ++t) {
            const int st = t % S::stages;
            ok = c.wait(c.empty(st), (uint32_t)(t / S::stages) ^ 1u, 0);
            if (!ok) break;
            mkb::mbar_expect_tx(c.full(st), S::kOperand);
            load_keys(c.stage(st), &maps.k, it, kDim, (first + t) * kTile, c.full(st));
        }
        // no copy may be in flight when the block's shared memory goes away
        tc_wait(c.held_full(0), 0, nullptr, a.timeout_ns, a.status, 0);
        for (int i = max(t - S::stages, 0); i < t; ++i) tc_wait(c.full(i % S::stages), (uint32_t)(i / S::stages) & 1u, nullptr, a.timeout_ns, a.status, 0);
    } else if (c.warp == 1 && c.lane == 0 && count > 0) {
        bool ok = c.wait(c.held_full(0), 0, 1);
        for (int t = 0; t < count && ok; ++t) {
            const int st = t % S::stages;
            ok = c.wait(c.full(st), (uint32_t)(t / S::stages), 1) && c.wait(c.read(t % kBuffers), (uint32_t)(t / kBuffers) ^ 1u, 1);
            if (!ok) break;
            tc_after_sync();
            c.multiply(c.held(0), c.stage(st), t);
            tc_commit(c.empty(st));
            tc_commit(c.scored(t % kBuffers));
        }
    } else if (c.warp >= 2) {
        const int quarter = c.warp & 3, part = (c.warp - 2) >> 2;  // (a warp may touch 32 lanes of tensor memory)
        const int warp_row = quarter * 32, r = warp_row + c.lane, have = min(of_tile * a.per, a.rows - r0);
        const int last = before + (r0 + r) / a.per, warp_last = before + (r0 + warp_row) / a.per;
        for (int t = 0; t < count; ++t) {
            if (!c.wait_all(c.scored(t % kBuffers), (uint32_t)(t / kBuffers))) break;
            tc_after_sync();
            uint32_t x[kCols];
            c.scores(t, quarter, part, x);
            if (warp_row >= have) continue;
            const int j0 = (first + t) * kTile + part * kCols;
            float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, s4[4] = {0.f, 0.f, 0.f, 0.f}, mul = a.scale;
            if (j0 + kCols - 1 <= warp_last && a.scale > 0.f) {  // every row sees all of these keys
#pragma unroll
                for (int i = 0; i < kCols; ++i) m4[i & 3] = fmaxf(m4[i & 3], __uint_as_float(x[i]));
            } else {
                mul = 1.f;
#pragma unroll
                for (int i = 0; i < kCols; ++i) {
                    const float z = j0 + i <= last ? __uint_as_float(x[i]) * a.scale : -INFINITY;
                    m4[i & 3] = fmaxf(m4[i & 3], z);
                    x[i] = __float_as_uint(z);
                }
            }
            const float top = fmaxf(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * mul, mine.x);
            if (top == -INFINITY) continue;
            const float keep = fast_exp2(mine.x - top);  // (0 from minus infinity)
#pragma unroll
            for (int i = 0; i < kCols; ++i) s4[i & 3] += fast_exp2(fmaf(__uint_as_float(x[i]), mul, -top));
            mine = make_float2(top, fmaf(mine.y, keep, (s4[0] + s4[1]) + (s4[2] + s4[3])));
        }
    }
    float2* const cross = reinterpret_cast<float2*>(c.at + c.sm.cross);
    if (c.warp >= 2) cross[((c.warp - 2) >> 2) * kTile + (c.warp & 3) * 32 + c.lane] = mine;
    c.leave();
    if (threadIdx.x < kTile) {
        const int r = threadIdx.x;
        float2 all = cross[r];
        for (int i = 1; i < kWarps / 4; ++i) all = join(all, cross[i * kTile + r]);
        if (r >= of_tile * a.per || r0 + r >= a.rows) all = make_float2(-INFINITY, 0.f);
        const int64_t row_tile = (int64_t)blockIdx.z * a.row_tiles + tile;
        if (a.splits > 1) a.parts[(row_tile * a.splits + blockIdx.x) * kTile + r] = all;
        else a.offs[row_tile * kTile + r] = off_of(all.x, all.y);
    }
}

// A row's parts to the logarithm of its sum.
__global__ void __launch_bounds__(kTile) weights_join_kernel(const WeightArgs a) {
    let_next();
    after_previous();
    const float2* const parts = a.parts + (int64_t)blockIdx.x * a.splits * kTile + threadIdx.x;
    float top = -INFINITY, sum = 0.f;
    for (int i = 0; i < a.splits; ++i) top = fmaxf(top, parts[i * kTile].x);
    for (int i = 0; i < a.splits; ++i) {
        const float2 p = parts[i * kTile];
        if (p.x > -INFINITY) sum += p.y * fast_exp2(p.x - top);
    }
    a.offs[(int64_t)blockIdx.x * kTile + threadIdx.x] = off_of(top, sum);
}

template <int kDim>
__global__ void __launch_bounds__(kThreads, 1) weights_keys_kernel(const __grid_constant__ WeightMaps maps, const WeightArgs a, int parts) {
    extern __shared__ uint8_t raw[];
    const Item it(a, blockIdx.y);
    const int share = blockIdx.x / parts, rank = blockIdx.x - share * parts;
    const int of_tile = kTile / a.per, before = it.n - a.queries, tiles = (it.n + kTile - 1) / kTile;
    using S = Smem<kDim>;
    const Block<kDim, true> c(raw, a, kTile % a.per != 0);
    const int box_bytes = of_tile * a.per * 128;
    // Steps: tiles of keys share, share + shares, ...; of each the row tiles that see one of its keys, every `parts`-th of them
    auto first_rows = [&](int kt) { return max(kt * kTile - before, 0) / of_tile + rank; };
    auto rows_of = [&](int kt) { return max(a.row_tiles - first_rows(kt) + parts - 1, 0) / parts; };
    float* const cross = reinterpret_cast<float*>(c.at + c.sm.cross);  // [parity][4][128]
    float* const weights = it.weights(a);
    after_previous();

    if (c.warp == 0 && c.lane == 0) {
        bool ok = true;
        int t = 0, held = 0;
        for (int kt = share; kt < tiles && ok; kt += a.shares) {
            const int steps = rows_of(kt);
            if (steps == 0) continue;
            ok = c.wait(c.held_empty(held & 1), (uint32_t)(held >> 1) ^ 1u, 0);
            if (!ok) break;
            mkb::mbar_expect_tx(c.held_full(held & 1), S::kOperand);
            load_keys(c.held(held & 1), &maps.k, it, kDim, kt * kTile, c.held_full(held & 1));
            ++held;
            for (int i = 0; i < steps && ok; ++i) {
                const int st = t % S::stages, tile = first_rows(kt) + i * parts;
                ok = c.wait(c.empty(st), (uint32_t)(t / S::stages) ^ 1u, 0);
                if (!ok) break;
                mkb::mbar_expect_tx(c.full(st), kDim / 64 * box_bytes + S::kExtra);
                load_queries(c.stage(st), &maps.q, it, kDim, a.per, tile * of_tile, c.full(st));
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(c.base + c.sm.extra + st * S::kExtra),
                             "l"(a.offs + ((int64_t)blockIdx.y * a.row_tiles + tile) * kTile), "r"(S::kExtra), "r"(c.full(st))
                             : "memory");
                ++t;
            }
        }
        for (int i = max(held - 2, 0); i < held; ++i) tc_wait(c.held_full(i & 1), (uint32_t)(i >> 1) & 1u, nullptr, a.timeout_ns, a.status, 0);
        for (int i = max(t - S::stages, 0); i < t; ++i) tc_wait(c.full(i % S::stages), (uint32_t)(i / S::stages) & 1u, nullptr, a.timeout_ns, a.status, 0);
    } else if (c.warp == 1 && c.lane == 0) {
        bool ok = true;
        int t = 0, held = 0;
        for (int kt = share; kt < tiles && ok; kt += a.shares) {
            const int steps = rows_of(kt);
            if (steps == 0) continue;
            ok = c.wait(c.held_full(held & 1), (uint32_t)(held >> 1), 1);
            for (int i = 0; i < steps && ok; ++i, ++t) {
                const int st = t % S::stages;
                ok = c.wait(c.full(st), (uint32_t)(t / S::stages), 1) && c.wait(c.read(t % kBuffers), (uint32_t)(t / kBuffers) ^ 1u, 1);
                if (!ok) break;
                tc_after_sync();
                c.multiply(c.held(held & 1), c.stage(st), t);
                tc_commit(c.empty(st));
                if (i == steps - 1) tc_commit(c.held_empty(held & 1));
                tc_commit(c.scored(t % kBuffers));
            }
            ++held;
        }
    } else if (c.warp >= 2) {
        const int quarter = c.warp & 3, part = (c.warp - 2) >> 2;
        bool ok = true;
        int t = 0, turn = 0;
        for (int kt = share; kt < tiles && ok; kt += a.shares, ++turn) {
            const int steps = rows_of(kt), j = kt * kTile + quarter * 32 + c.lane;
            const int own_row = max(j - before, 0) * a.per, last_row = max(kt * kTile + quarter * 32 + 31 - before, 0) * a.per;  // the first that sees it
            float s4[4] = {0.f, 0.f, 0.f, 0.f};
            for (int i = 0; i < steps; ++i, ++t) {
                const int st = t % S::stages, r0 = (first_rows(kt) + i * parts) * of_tile * a.per + part * kCols;
                ok = c.wait_all(c.scored(t % kBuffers), (uint32_t)(t / kBuffers)) && c.wait_all(c.full(st), (uint32_t)(t / S::stages));
                if (!ok) break;
                tc_after_sync();
                uint32_t x[kCols];
                c.scores(t, quarter, part, x);
                const float4* const off = reinterpret_cast<const float4*>(c.at + c.sm.extra + st * S::kExtra) + part * (kCols / 4);
                if (last_row <= r0) {
#pragma unroll
                    for (int n = 0; n < kCols / 4; ++n) {
                        const float4 o = off[n];
                        s4[0] += fast_exp2(fmaf(__uint_as_float(x[4 * n]), a.scale, -o.x));
                        s4[1] += fast_exp2(fmaf(__uint_as_float(x[4 * n + 1]), a.scale, -o.y));
                        s4[2] += fast_exp2(fmaf(__uint_as_float(x[4 * n + 2]), a.scale, -o.z));
                        s4[3] += fast_exp2(fmaf(__uint_as_float(x[4 * n + 3]), a.scale, -o.w));
                    }
                } else {
                    const int hidden = own_row - r0;  // columns before that do not see the key
#pragma unroll
                    for (int n = 0; n < kCols / 4; ++n) {
                        const float4 o = off[n];
                        const float p[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float y = fast_exp2(fmaf(__uint_as_float(x[4 * n + e]), a.scale, -p[e]));
                            s4[e] += 4 * n + e >= hidden ? y : 0.f;
                        }
                    }
                }
                __syncwarp();
                if (c.lane == 0) mkb::mbar_arrive(c.empty(st));
            }
            if (!ok) break;
            // the four threads of a key
            float* const at = cross + (turn & 1) * kWarps / 4 * kTile + quarter * 32 + c.lane;
            at[part * kTile] = (s4[0] + s4[1]) + (s4[2] + s4[3]);
            __syncwarp();
            if (c.lane == 0) mkb::mbar_arrive(c.meeting(quarter));
            ok = c.wait_all(c.meeting(quarter), (uint32_t)turn);
            if (ok && part == 0) {
                float sum = at[0];
#pragma unroll
                for (int i = 1; i < kWarps / 4; ++i) sum += at[i * kTile];
                if (parts > 1) at[0] = sum;  // (one tile of keys per block)
                else if (j < it.n) weights[j] += sum;
            }
        }
    }
    c.leave();
    if (parts > 1) {
        tc_cluster_sync();
        const int j = share * kTile + threadIdx.x;
        if (rank == 0 && threadIdx.x < kTile && j < it.n) {
            float sum = cross[threadIdx.x];
            for (int i = 1; i < parts; ++i) {
                float v;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(tc_peer(mkb::smem_u32(cross + threadIdx.x), i)) : "memory");
                sum += v;
            }
            weights[j] += sum;
        }
        tc_cluster_sync();
    }
}

// ---- up to 16 rows ------------------------------------------------------------------------------ //
constexpr int kFewThreads = 256, kFewWarps = kFewThreads / 32, kAhead = 4;  // groups of 8 keys whose loads a warp has under way

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Rows are the M side, 8 keys the N side.  The contraction's order is free: lane (n, c) of a warp, n = lane / 4 and c = lane % 4, holds the
// neighbours 8 c + 32 i .. + 7 of key n, two products' worth, so a key is read in 16-byte pieces straight into fragments.
template <int kDim, int kRowsPad>
__global__ void __launch_bounds__(kFewThreads) weights_few_kernel(const WeightArgs a) {
    let_next();
    constexpr int kPieces = kDim / 32;
    __shared__ float2 shared[kFewWarps][kFew];
    const Item it(a, blockIdx.y);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane / 4, c = lane % 4, before = it.n - a.queries;
    const bf16* const keys = a.k + it.layer * a.k_layer + it.b * a.k_sequence + it.g * kDim + c * 8;
    const int64_t key_row = (int64_t)a.kv_heads * kDim;
    float* const scores = a.scores + (int64_t)blockIdx.y * a.positions * kRowsPad;
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
    const int groups = (it.n + 7) / 8, total = (int)gridDim.x * kFewWarps, me = (int)blockIdx.x * kFewWarps + warp;
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
                const float z0 = j <= last[h] ? d[2 * h] * a.scale : -INFINITY, z1 = j + 1 <= last[h] ? d[2 * h + 1] * a.scale : -INFINITY;
                const float top = fmaxf(fmaxf(z0, z1), stats[h].x);
                if (n + 8 * h < kRowsPad) {
                    if (j < it.n) scores[(int64_t)j * kRowsPad + n + 8 * h] = z0;
                    if (j + 1 < it.n) scores[(int64_t)(j + 1) * kRowsPad + n + 8 * h] = z1;
                }
                if (top > -INFINITY) stats[h] = make_float2(top, stats[h].y * fast_exp2(stats[h].x - top) + fast_exp2(z0 - top) + fast_exp2(z1 - top));
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
        a.parts[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kFew + threadIdx.x] = all;
    }
}

template <int kRowsPad>
__global__ void __launch_bounds__(kFewThreads) weights_sum_kernel(const WeightArgs a) {
    __shared__ float off[kFew];
    const Item it(a, blockIdx.y);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    after_previous();
    for (int r = warp; r < kRowsPad; r += kFewWarps) {
        const float2* const parts = a.parts + (int64_t)blockIdx.y * a.splits * kFew + r;
        float2 all = make_float2(-INFINITY, 0.f);
        for (int i = lane; i < a.splits; i += 32) all = join(all, parts[i * kFew]);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) all = join(all, make_float2(__shfl_xor_sync(0xffffffffu, all.x, o), __shfl_xor_sync(0xffffffffu, all.y, o)));
        if (lane == 0) off[r] = off_of(all.x, all.y);
    }
    __syncthreads();
    const float* const scores = a.scores + (int64_t)blockIdx.y * a.positions * kRowsPad;
    float* const weights = it.weights(a);
    for (int j = blockIdx.x * kFewThreads + threadIdx.x; j < it.n; j += gridDim.x * kFewThreads) {
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < kRowsPad; r += 4) {
            const float4 z = *reinterpret_cast<const float4*>(scores + (int64_t)j * kRowsPad + r);
            sum += (fast_exp2(z.x - off[r]) + fast_exp2(z.y - off[r + 1])) + (fast_exp2(z.z - off[r + 2]) + fast_exp2(z.w - off[r + 3]));
        }
        weights[j] += sum;
    }
}

// ---- host ------------------------------------------------------------------------------------------ //
struct Plan {
    WeightArgs a;
    int items, parts, rows_pad;
    bool few;
    size_t bytes;
    explicit Plan(const MkbsKeyWeights& w) {
        const int per = w.heads / w.kv_heads, rows = w.queries * per;
        items = w.layers * w.sequences * w.kv_heads;
        const int longest = w.lengths != nullptr ? w.positions : w.length, tiles = longest > kTile ? (longest + kTile - 1) / kTile : 1;
        few = rows <= kFew;
        const int row_tiles = (w.queries + kTile / per - 1) / (kTile / per);
        a = {w.sequences, w.queries, w.heads, w.kv_heads, w.positions, w.length, per, rows, row_tiles, 1, 1, w.scale * kLog2e, w.lengths,
             static_cast<const bf16*>(w.q), static_cast<const bf16*>(w.k), w.q_layer, w.q_sequence, w.k_layer, w.k_sequence,
             w.weights, w.w_layer, w.w_sequence, w.w_head, nullptr, nullptr, nullptr, w.status,
             w.wait_timeout_ms ? w.wait_timeout_ms * 1000000ull : kWaitNs};
        auto up = [](int n, int of) { return (n + of - 1) / of; };
        char* const base = static_cast<char*>(w.workspace);
        if (few) {
            rows_pad = rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
            // four blocks per SM, none with less than 64 keys a warp
            a.splits = up(4 * kSms, items);
            if (a.splits > up(longest, 64 * kFewWarps)) a.splits = up(longest, 64 * kFewWarps);
            if (a.splits < 1) a.splits = 1;
            const size_t scores = ((size_t)items * w.positions * rows_pad * 4 + 255) / 256 * 256;
            a.scores = reinterpret_cast<float*>(base);
            a.parts = reinterpret_cast<float2*>(base + scores);
            bytes = scores + (size_t)items * a.splits * kFew * 8;
            return;
        }
        // rows: a block per SM; keys as well, and where there are not as many tiles, clusters
        a.splits = kSms / (items * row_tiles);
        a.splits = a.splits < 1 ? 1 : a.splits > tiles ? tiles : a.splits;
        a.shares = kSms / items;
        a.shares = a.shares < 1 ? 1 : a.shares > tiles ? tiles : a.shares;
        for (parts = 1; a.shares == tiles && parts < 8 && 2 * parts <= row_tiles && items * a.shares * parts < 2 * kSms;) parts *= 2;
        const size_t offs = (size_t)items * row_tiles * kTile * 4;
        a.offs = reinterpret_cast<float*>(base);
        a.parts = reinterpret_cast<float2*>(base + offs);
        bytes = offs + (a.splits > 1 ? (size_t)items * row_tiles * a.splits * kTile * 8 : 0);
    }
};

// 4 or 5 dimensions of bf16 with the 128-byte swizzle; what lies outside reads as zero
cudaError_t encode(CUtensorMap* map, const bf16* ptr, int dims, const cuuint64_t* size, const cuuint64_t* stride_bytes, const cuuint32_t* box) {
    static EncodeFn fn = nullptr;
    if (fn == nullptr) {
        void* found = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &found, cudaEnableDefault, &q); e != cudaSuccess) return e;
        if (q != cudaDriverEntryPointSuccess || found == nullptr) return cudaErrorNotSupported;
        fn = reinterpret_cast<EncodeFn>(found);
    }
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
    const int rows_smem = Smem<kDim>(false).total + 1024, keys_smem = Smem<kDim>(true).total + 1024;
    if ((e = allow_shared_memory<weights_rows_kernel<kDim>>()) != cudaSuccess) return e;
    if ((e = allow_shared_memory<weights_keys_kernel<kDim>>()) != cudaSuccess) return e;
    weights_rows_kernel<kDim><<<dim3(a.splits, a.row_tiles, p.items), kThreads, rows_smem, s>>>(maps, a);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    if (a.splits > 1 && (e = launch_early(weights_join_kernel, dim3(p.items * a.row_tiles), dim3(kTile), 0, s, a)) != cudaSuccess) return e;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(a.shares * p.parts, p.items);
    c.blockDim = dim3(kThreads);
    c.dynamicSmemBytes = keys_smem;
    c.stream = s;
    cudaLaunchAttribute attrs[2] = {may_begin_early()};
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = p.parts;
    attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
    c.attrs = attrs;
    c.numAttrs = p.parts > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&c, weights_keys_kernel<kDim>, maps, a, p.parts);
}

template <int kDim, int kRowsPad>
cudaError_t launch_few(const Plan& p, cudaStream_t s) {
    weights_few_kernel<kDim, kRowsPad><<<dim3(p.a.splits, p.items), kFewThreads, 0, s>>>(p.a);
    if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
    return launch_early(weights_sum_kernel<kRowsPad>, dim3(p.a.splits, p.items), dim3(kFewThreads), 0, s, p.a);
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
