// Product of 8-bit rows: out[m][n] = sum over k of a[m][k] * 2^(ea - 127) * b[n][k] * 2^(eb - 127), a scale per 128 columns of a row.
//
// The tensor cores multiply e4m3 blocks with E8M0 scales themselves (tcgen05.mma kind::mxf8f6f4, one scale byte per row and 32
// columns): the four instructions of a 128-column group name the same byte, so scales are neither repeated in memory nor applied
// by other units, and the sum stays in tensor memory, in 32 bits, from the first group to the last.
//
// Pairs of CTAs (clusters of two, cta_group::2) walk output tiles of 256 x tile_n.  A CTA holds 128 rows of a and half of the tile's rows of b,
// so that an operand byte in shared memory feeds twice the multiplications it would in a CTA alone, and its tensor memory the sums of its
// 128 rows.  The warps of a CTA:
//   copier    a ring slot holds 256 columns of the CTA's share of both operands (four tensor-map copies, 128-byte swizzle).  Short contractions
//             have a ring for b alone: the rows of a stay while the pair walks the tiles of those rows, which halves what crosses from L2.
//   issuer    of the first CTA only; eight instructions per slot, and per eight groups the copies of the scales into tensor memory
//   3 scalers fetch the scale bytes of eight groups (two words per row) and lay them out for those copies: row r of 128 at
//             (r % 32) * 16 + (r / 32) * 4.  Both CTAs need all scales of b.  The words of the next octets are under way meanwhile: fetched
//             one quad after the other by one warp, 131072 x 1152 x 768 took 200 us, by two with the next words under way 156, by four 138.
//   4 storers read the sums of a finished tile out of tensor memory, one lane a row, round them and send them out through shared memory
//             with tensor-map copies of 32 rows x 64 bytes, while the issuer is at the next tile (two accumulators up to 224 columns).
// An operand whose rows are neighbours in memory (dg_rows8.by_column) is copied as 128 rows x 128 columns too, and the instruction told.
// Measured: 8192 x 8192 x 8192 432 us, 2.5 PFLOP/s; 131072 x 1152 x 768 into bf16 120 to 126 us over the same operands again, 142 to 149 over others in every
// call, 1.6 (its 302 MB of output alone take 80 at the 3.8 TB/s of a plain fill, its multiplications alone 80, its copies 55: they do not quite hide one another); 1152 x 768 x 57600 61 us, where copies out of L2 end at
// 10 TB/s; 7 x 1024 x 768 6 us, all latency.  Accuracy: 1.5e-8 of the result over 128 columns, 3e-7 over 8192,
// which no part of a contraction exceeds (dg::plan_product).
// Waits are bounded: a CTA that runs out of patience counts itself (dg_product_status) and leaves.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "kernels.h"
#include "tokens.h"

namespace dg {

namespace {

constexpr uint32_t kTileM = kProductTileM, kRowsPerCta = kTileM / 2;
constexpr uint32_t kScalers = 3, kScaleStages = kScalers;  // a slot's fillings are all one warp's: it cannot miss one of them
constexpr uint32_t kABytes = kProductABytes;  // of a group; a slot holds two
constexpr uint32_t kScaleBytes = 512 * 3;  // of four groups: 128 rows of a, 256 of b; a slot holds eight groups'
constexpr uint32_t kOutBytes = 32 * 64, kPieces = 3;  // a storer's piece of the output: 32 rows x 64 bytes; pieces it has room for
constexpr uint32_t kThreads = 9 * 32, kSlots = kProductSlots;
constexpr uint32_t kOutAt = kProductRingBytes, kScalesAt = kOutAt + 4 * kPieces * kOutBytes;
constexpr uint32_t kSmemBytes = kScalesAt + kScaleStages * 2 * kScaleBytes + 1024;
static_assert(kSmemBytes <= 232448 - 512, "what a CTA may have, and the barriers");
// tensor memory: the accumulators from column 0 and, up to kProductTwoSums wide, from column kProductTwoSums; then, twice, scales of eight groups
// (for each four of them 4 columns of a and 8 of b)
constexpr uint32_t kSecond = kProductTwoSums, kScaleColumns = 2 * kProductTwoSums;
static_assert(kScaleColumns + 2 * 24 <= 512 && kScaleColumns >= kProductMaxTileN, "the scales fit behind the sums");
constexpr uint32_t kWaitLimit = 1u << 20;  // waits of up to 2 us each

__device__ unsigned int g_gave_up;  // never set back: each context remembers what it has reported

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t cluster_bar) {  // of either CTA of the pair
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// far: what the other CTA's threads wrote before they arrived is read next
template <bool FAR = false>
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    if constexpr (FAR)
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
                     : "=r"(done) : "r"(bar), "r"(parity), "r"(2000u) : "memory");
    else
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(done) : "r"(bar), "r"(parity), "r"(2000u) : "memory");
    return done != 0;
}
// One lane of a warp that is all here.  The copying and the issuing warp stay together, lane by lane, and only such a lane copies or issues: the
// operands of those instructions are uniform registers, and in code that a lane runs alone every one of them was gathered anew
// (8192 x 8192 x 8192: 557 us instead of 449).
__device__ __forceinline__ bool chosen() {
    uint32_t yes;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(yes));
    return yes != 0;
}
__device__ __forceinline__ uint32_t in_first_cta(uint32_t at) {  // the same place in the shared memory of the pair's first CTA
    uint32_t there;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(there) : "r"(at));
    return there;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// One box into this CTA's shared memory; its bytes are counted on a barrier of either CTA of the pair.
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, uint32_t cluster_bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void store_box(const CUtensorMap* map, int32_t x, int32_t y, int32_t z, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];\n cp.async.bulk.commit_group;"
                 ::"l"(map), "r"(x), "r"(y), "r"(z), "r"(src) : "memory");
}
// arrives on the barrier at this place in both CTAs when all tensor-core work that this thread has issued is done
__device__ __forceinline__ void commit_to(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// Shared-memory descriptors.  Operands: 128-byte swizzle over eight lines of 128 bytes (1024 bytes).  A line is a row of 128 columns,
// eight rows of the tile then follow after 1024 bytes; or (by column) a column of 128 rows, eight columns follow after 1024 bytes, and 128 more
// rows, of which there are none, after 16384.  Scales: no swizzle, eight rows of 16 bytes (128 bytes) apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t at) {
    return (uint64_t)((at >> 4) & 0x3FFFu) | (uint64_t)(16384 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
__device__ __forceinline__ uint64_t scales_desc(uint32_t at) { return (uint64_t)((at >> 4) & 0x3FFFu) | (uint64_t)(128 >> 4) << 32 | 1ull << 46; }
__device__ __forceinline__ void copy_scales(uint32_t columns, uint32_t at) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(columns), "l"(scales_desc(at)) : "memory");
}
__device__ __forceinline__ void multiply(uint32_t acc, uint64_t a, uint64_t b, uint32_t what, uint32_t a_scales, uint32_t b_scales, bool add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
                 " tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}"
                 ::"r"(acc), "l"(a), "l"(b), "r"(what), "r"(a_scales), "r"(b_scales), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void read_16(uint32_t at, uint32_t v[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                   "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(at));
}

__device__ __forceinline__ uint32_t pair(float lo, float hi, __nv_bfloat16) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t pair(float lo, float hi, __half) {
    const __half2 p = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
}
template <class T> __device__ __forceinline__ T one(float v);
template <> __device__ __forceinline__ float one<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 one<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half one<__half>(float v) { return __float2half_rn(v); }

struct Place {  // in a ring: the slot, and the parity of its fillings so far
    uint32_t slot = 0, phase = 0;
    __device__ __forceinline__ void next(uint32_t n) {
        if (++slot == n) { slot = 0; phase ^= 1u; }
    }
};

// Four scale bytes (groups 4 q .. 4 q + 3, those that there are) of the row that has its first at p.
__device__ __forceinline__ uint32_t scale_word(const uint8_t* p, uint32_t q, uint32_t left) {
    p += 4 * (uint64_t)q;
    if (left >= 4) return *reinterpret_cast<const uint32_t*>(p);  // the same for all rows: the loads of a warp's twelve words go out together
    return (left > 1 ? (uint32_t)*reinterpret_cast<const uint16_t*>(p) : p[0]) | (left == 3 ? (uint32_t)p[2] << 16 : 0u);
}

// RAGGED: the output's rows begin at multiples of 16 bytes, but end inside one.
template <class T, bool RAGGED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) k_product(const __grid_constant__ ProductJob j, T* out, uint64_t ld, uint64_t part_elements) {
    extern __shared__ unsigned char raw_smem[];
    __shared__ __align__(8) unsigned long long s_bar[4 * kSlots + 2 * kScaleStages + 5];
    __shared__ uint32_t s_tmem;
    __shared__ volatile uint32_t s_quit;
    const uint32_t smem = ((uint32_t)__cvta_generic_to_shared(raw_smem) + 1023u) & ~1023u;  // the swizzle counts from multiples of 1024
    const uint32_t scales_at = smem + kScalesAt;
    const uint32_t bar = (uint32_t)__cvta_generic_to_shared(s_bar);
    // slots of b (and of a, where it comes along), of a where it stays, of the scales: full in the first CTA, for the issuer; empty in both
    auto full = [&](uint32_t i) { return bar + 8 * i; };
    auto empty = [&](uint32_t i) { return bar + 8 * (kSlots + i); };
    auto a_full = [&](uint32_t i) { return bar + 8 * (2 * kSlots + i); };
    auto a_empty = [&](uint32_t i) { return bar + 8 * (3 * kSlots + i); };
    const uint32_t bar2 = bar + 8 * 4 * kSlots;
    auto scales_full = [&](uint32_t i) { return bar2 + 8 * i; };
    auto scales_empty = [&](uint32_t i) { return bar2 + 8 * (kScaleStages + i); };
    // accumulators: full in both, empty in the first CTA
    auto sums_full = [&](uint32_t i) { return bar2 + 8 * (2 * kScaleStages + i); };
    auto sums_empty = [&](uint32_t i) { return bar2 + 8 * (2 * kScaleStages + 2 + i); };
    const uint32_t over = bar2 + 8 * (2 * kScaleStages + 4);
    const uint32_t warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31u, rank = blockIdx.x & 1u;
    let_next_start();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"((uint32_t)__cvta_generic_to_shared(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kSlots; ++i) { bar_init(full(i), 1); bar_init(empty(i), 1); bar_init(a_full(i), 1); bar_init(a_empty(i), 1); }
        for (uint32_t i = 0; i < kScaleStages; ++i) { bar_init(scales_full(i), 2); bar_init(scales_empty(i), 1); }
        for (uint32_t i = 0; i < 2; ++i) { bar_init(sums_full(i), 1); bar_init(sums_empty(i), 8); }
        bar_init(over, 1);
        s_quit = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;
    wait_for_previous();

    // false once some thread of the CTA has given up
    auto wait_for = [&](uint32_t at, uint32_t parity) {
        uint32_t polls = 0;
        while (!bar_try(at, parity)) {
            if (s_quit) return false;
            if (++polls > kWaitLimit) { s_quit = 1; return false; }
        }
        return true;
    };
    auto wait_for_both = [&](uint32_t at, uint32_t parity) {  // for threads of both CTAs
        if (!wait_for(at, parity)) return false;
        return bar_try<true>(at, parity);
    };
    auto all_wait_for = [&](uint32_t at, uint32_t parity) { return (bool)__all_sync(0xFFFFFFFFu, wait_for(at, parity)); };  // a whole warp
    const uint32_t tile_n = j.plan.tile_n, tiles_n = j.plan.tiles_n, per_split = j.plan.tiles_m * tiles_n;
    const uint32_t tiles = per_split * j.plan.splits, sums = j.plan.sums;
    const uint32_t groups = (uint32_t)((j.k + kScaleGroup - 1) / kScaleGroup);
    // what a tile index stands for: the part of the contraction, the first row and column, the groups; whether the tiles before and after it have
    // the same rows
    struct Tile { uint32_t split, m0, n0, g0, g1; bool same_before, same_after; };
    // Where a stays, a pair walks neighbouring tiles, which share their rows of a.  Elsewhere all pairs are at neighbouring tiles, which share
    // more of what is in L2 (8192 x 8192 x 8192 449 us, with neighbouring tiles to a pair 535).
    const bool a_stays = j.plan.a_stays;
    const uint32_t pairs = gridDim.x >> 1, me = blockIdx.x >> 1, step = a_stays ? 1 : pairs;
    const uint32_t first = a_stays ? (uint32_t)((uint64_t)tiles * me / pairs) : me, end = a_stays ? (uint32_t)((uint64_t)tiles * (me + 1) / pairs) : tiles;
    auto tile_at = [&](uint32_t i) {
        Tile t;
        t.split = i / per_split;
        const uint32_t r = i - t.split * per_split, tm = r / tiles_n, tn = r - tm * tiles_n;
        t.m0 = tm * kTileM + rank * kRowsPerCta;  // of this CTA
        t.n0 = tn * tile_n;
        t.same_before = a_stays && tn != 0 && i != first;
        t.same_after = a_stays && tn + 1 != tiles_n && i + 1 != end;
        t.g0 = j.first_group + t.split * j.plan.split_groups;
        t.g1 = min(groups, t.g0 + j.plan.split_groups);
        return t;
    };
    // the rings: slots of b behind those of a
    const uint32_t slots = j.plan.slots, b_bytes = (j.b_by_column ? 128 : tile_n / 2) * 128, b_at = smem + (a_stays ? groups : 2 * slots) * kABytes;

    if (warp == 0) {  // ---- copier
        Place at;
        uint32_t filled = 0, a_filled = 0;  // slots; rows of tiles whose a has been copied
        const bool a_by_column = j.a_by_column, b_by_column = j.b_by_column;
        const uint32_t bytes = 2 * (b_bytes + (a_stays ? 0 : kABytes));  // of a group, in both CTAs
        bool go_on = true;
        for (uint32_t i = first; go_on && i < end; i += step) {
            const Tile t = tile_at(i);
            const int32_t m0 = (int32_t)t.m0, n0 = (int32_t)(t.n0 + rank * (tile_n / 2));
            const bool new_a = a_stays && !t.same_before;
            for (uint32_t g = t.g0; g < t.g1; g += 2) {
                const uint32_t count = min(2u, t.g1 - g);
                if (new_a) {  // not split: the groups are the slots
                    if (a_filled) go_on = all_wait_for(a_empty(g >> 1), (a_filled - 1) & 1u);
                    if (!go_on) break;
                    if (chosen()) {
                        if (rank == 0) bar_expect(a_full(g >> 1), count * 2 * kABytes);
                        for (uint32_t k = g; k < g + count; ++k)
                            copy_box(smem + k * kABytes, &j.a, a_by_column ? m0 : (int32_t)(k * 128), a_by_column ? (int32_t)(k * 128) : m0, in_first_cta(a_full(g >> 1)));
                    }
                }
                if (filled >= slots) go_on = all_wait_for(empty(at.slot), at.phase ^ 1u);
                if (!go_on) break;
                if (chosen()) {
                    const uint32_t there = in_first_cta(full(at.slot));
                    if (rank == 0) bar_expect(full(at.slot), count * bytes);
                    for (uint32_t k = 0; k < count; ++k) {
                        const int32_t k0 = (int32_t)((g + k) * 128);
                        if (!a_stays) copy_box(smem + (2 * at.slot + k) * kABytes, &j.a, a_by_column ? m0 : k0, a_by_column ? k0 : m0, there);
                        copy_box(b_at + (2 * at.slot + k) * b_bytes, &j.b, b_by_column ? n0 : k0, b_by_column ? k0 : n0, there);
                    }
                }
                ++filled;
                at.next(slots);
            }
            if (new_a) ++a_filled;
        }
        // nothing may arrive in the shared memory of a CTA that has gone: the slots' multiplications, and so their copies, are over when
        // both CTAs meet at the end.  Only a CTA that gives up leaves copies behind, which the first CTA waits for.
        if (!go_on && rank == 0) {
            for (uint32_t c = filled > slots ? filled - slots : 0; c < filled; ++c) {
                uint32_t polls = 0;
                while (!bar_try(full(c % slots), (c / slots) & 1u) && ++polls <= kWaitLimit) {}
            }
            for (uint32_t g = 0; a_stays && a_filled && 2 * g < groups; ++g) {
                uint32_t polls = 0;
                while (!bar_try(a_full(g), (a_filled - 1) & 1u) && ++polls <= kWaitLimit) {}
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {  // ---- issuer
            // the instruction: e4m3 by e4m3, E8M0 scales, 32-bit sums, 256 x tile_n; the scale byte of a group is filled in below
            const uint32_t base = 1u << 23 | (tile_n >> 3) << 17 | (kTileM >> 7) << 27 | (j.a_by_column ? 1u << 15 : 0u) | (j.b_by_column ? 1u << 16 : 0u);
            // 32 columns further: 32 bytes of the swizzled lines, or 32 lines
            const uint32_t a_step = j.a_by_column ? 4096 >> 4 : 32 >> 4, b_step = j.b_by_column ? 4096 >> 4 : 32 >> 4;
            Place at, sc, sum;
            uint32_t octets = 0, done = 0, a_read = 0;
            bool go_on = true;
            for (uint32_t i = first; go_on && i < end; i += step, ++done) {
                const Tile t = tile_at(i);
                const uint32_t acc = tmem + sum.slot * kSecond;
                if (done >= sums && !(go_on = all_wait_for(sums_empty(sum.slot), sum.phase ^ 1u))) break;
                for (uint32_t g = t.g0; g < t.g1; g += 2) {
                    const uint32_t nth = (g - t.g0) & 7u, columns = tmem + kScaleColumns + (octets & 1u) * 24;
                    if (nth == 0) {
                        // the columns that these scales go to were read by the instructions of the octet before the last
                        if (octets >= 2) {
                            const uint32_t o = octets - 2;
                            if (!(go_on = all_wait_for(scales_empty(o % kScaleStages), (o / kScaleStages) & 1u))) break;
                        }
                        if (!(go_on = (bool)__all_sync(0xFFFFFFFFu, wait_for_both(scales_full(sc.slot), sc.phase)))) break;
                    }
                    if (a_stays && !t.same_before && !(go_on = all_wait_for(a_full(g >> 1), a_read & 1u))) break;
                    if (!(go_on = all_wait_for(full(at.slot), at.phase))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const bool last = nth == 6 || g + 2 >= t.g1;
                    if (chosen()) {
                        if (nth == 0) {
                            const uint32_t from = scales_at + sc.slot * 2 * kScaleBytes;
                            for (uint32_t q = 0; q < (t.g1 - g > 4 ? 2u : 1u); ++q) {
                                copy_scales(columns + 12 * q, from + q * kScaleBytes);
                                copy_scales(columns + 12 * q + 4, from + q * kScaleBytes + 512);
                                if (tile_n > 128) copy_scales(columns + 12 * q + 8, from + q * kScaleBytes + 1024);
                            }
                        }
                        uint64_t da = operand_desc(smem + (a_stays ? g : 2 * at.slot) * kABytes), db = operand_desc(b_at + 2 * at.slot * b_bytes);
                        const uint32_t scales = columns + 12 * (nth >> 2);
#pragma unroll
                        for (uint32_t k = 0; k < 2; ++k) {
                            if (g + k >= t.g1) break;
                            const uint32_t byte = (nth + k) & 3u, what = base | byte << 4 | byte << 29;
                            const uint64_t left = j.k - 128ull * (g + k);
                            multiply(acc, da, db, what, scales, scales + 4, k != 0 || g != t.g0);
                            if (left > 32) multiply(acc, da + a_step, db + b_step, what, scales, scales + 4, true);
                            if (left > 64) multiply(acc, da + 2 * a_step, db + 2 * b_step, what, scales, scales + 4, true);
                            if (left > 96) multiply(acc, da + 3 * a_step, db + 3 * b_step, what, scales, scales + 4, true);
                            da += kABytes >> 4;
                            db += b_bytes >> 4;
                        }
                        commit_to(empty(at.slot));
                        if (a_stays && !t.same_after) commit_to(a_empty(g >> 1));
                        if (last) commit_to(scales_empty(sc.slot));
                        if (g + 2 >= t.g1) commit_to(sums_full(sum.slot));
                    }
                    __syncwarp();
                    at.next(slots);
                    if (last) {
                        sc.next(kScaleStages);
                        ++octets;
                    }
                }
                if (!go_on) break;
                if (!t.same_after) ++a_read;
                sum.next(sums);
            }
            if (!go_on) {  // what has been issued ends before the CTAs do
                uint32_t polls = 0;
                if (chosen()) commit_to(over);
                while (!bar_try(over, 0) && ++polls <= kWaitLimit) {}
            }
        }
    } else if (warp < 4 || warp >= 8) {  // ---- scalers: octets in turn, the words of the next one of each under way
        struct Octet { uint32_t i, g, g1, m0, n0; } now;
        auto enter = [&](Octet& o) {  // the tile that o.i names
            if (o.i < end) { const Tile t = tile_at(o.i); o.g = t.g0; o.g1 = t.g1; o.m0 = t.m0; o.n0 = t.n0; }
        };
        auto next = [&](Octet& o) {
            if (o.i < end && (o.g += 8) >= o.g1) { o.i += step; enter(o); }
        };
        const uint8_t *const pa = from_previous(j.a_scales), *const pb = from_previous(j.b_scales);
        const uint32_t last_m = (uint32_t)j.m - 1, last_n = (uint32_t)j.n - 1, a_shift = j.a_block == 1 ? 0 : 7, b_shift = j.b_block == 1 ? 0 : 7;
        auto fetch = [&](const Octet& o, uint32_t w[24]) {  // rows that a matrix does not have take the last one's: what they scale is not stored
            if (o.i >= end) return;
#pragma unroll
            for (uint32_t q = 0; q < 2; ++q) {
                if (o.g + 4 * q >= o.g1) break;
                const uint32_t left = groups - o.g - 4 * q, word = (o.g >> 2) + q;
#pragma unroll
                for (uint32_t r = 0; r < 4; ++r) w[12 * q + r] = scale_word(pa + (uint64_t)(min(o.m0 + lane + 32 * r, last_m) >> a_shift) * j.a_scale_ld, word, left);
#pragma unroll
                for (uint32_t r = 0; r < 8; ++r)
                    if (32 * r < tile_n) w[12 * q + 4 + r] = scale_word(pb + (uint64_t)(min(o.n0 + lane + 32 * r, last_n) >> b_shift) * j.b_scale_ld, word, left);
            }
        };
        now.i = first;
        enter(now);
        const uint32_t turn = warp < 4 ? warp - 2 : warp - 6;
        for (uint32_t k = 0; k < turn; ++k) next(now);
        uint32_t w[24] = {}, coming[24] = {};
        fetch(now, coming);
        for (uint32_t octet = turn; now.i < end; octet += kScalers) {
            const bool both = now.g + 4 < now.g1;
#pragma unroll
            for (int k = 0; k < 24; ++k) w[k] = coming[k];
#pragma unroll
            for (uint32_t k = 0; k < kScalers; ++k) next(now);
            fetch(now, coming);
            const uint32_t slot = octet % kScaleStages;
            if (octet >= kScaleStages && !all_wait_for(scales_empty(slot), (octet / kScaleStages - 1) & 1u)) break;
            const uint32_t to = scales_at + slot * 2 * kScaleBytes + lane * 16;
#pragma unroll
            for (int b = 0; b < 6; ++b)
                if (b < 3 || both)
                    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(to + 512 * b), "r"(w[4 * b]), "r"(w[4 * b + 1]), "r"(w[4 * b + 2]), "r"(w[4 * b + 3]) : "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(in_first_cta(scales_full(slot)));
        }
    } else {  // ---- storers
        constexpr uint32_t kPiece = 64 / sizeof(T);  // columns of a piece
        const uint32_t rows = (warp & 3u) * 32, mine = smem + kOutAt + (warp & 3u) * kPieces * kOutBytes;
        const bool by_map = j.map_cols != 0, by_word = sizeof(T) == 4 || ((reinterpret_cast<uintptr_t>(out) | (ld * sizeof(T)) | (part_elements * sizeof(T))) & 3u) == 0;
        Place room;
        Place sum;
        bool go_on = true;
        for (uint32_t i = first; go_on && i < end; i += step) {
            const Tile t = tile_at(i);
            go_on = all_wait_for(sums_full(sum.slot), sum.phase);
            if (!go_on) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t from = tmem + sum.slot * kSecond + (rows << 16);
            const uint64_t row0 = (uint64_t)t.m0 + rows;
            const uint32_t live = row0 < j.m ? (uint32_t)min((uint64_t)32, j.m - row0) : 0;  // rows of this warp that the matrix has
            const uint32_t width = (uint32_t)min((uint64_t)tile_n, j.n - t.n0);
            const uint32_t mapped = RAGGED ? min(width, max((uint32_t)j.map_cols, t.n0) - t.n0) : width;  // columns of the tile that the map has
            uint32_t v[kPiece], w[16];
            auto read = [&](uint32_t c) {
#pragma unroll
                for (uint32_t k = 0; k < kPiece; k += 16) read_16(from + c + k, v + k);
            };
            read(0);
            for (uint32_t c = 0; c < width; c += kPiece) {
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    if constexpr (sizeof(T) == 4) w[k] = v[k];
                    else w[k] = pair(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1]), T());
                }
                // the next sums are on their way while these leave; after the last ones the accumulator is free
                if (c + kPiece < width) read(c + kPiece);
                else {
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) bar_arrive(in_first_cta(sums_empty(sum.slot)));
                }
                if (!live) continue;  // nothing leaves: what is still being read of the pieces stays as it is
                const uint32_t piece = mine + room.slot * kOutBytes;
                room.next(kPieces);
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kPieces - 1) : "memory");  // the piece that was here has left
                __syncwarp();
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k)  // 64-byte swizzle: 16 bytes k of row r at k ^ (r / 2 % 4)
                    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(piece + lane * 64 + ((k ^ ((lane >> 1) & 3u)) << 4)), "r"(w[4 * k]), "r"(w[4 * k + 1]),
                                 "r"(w[4 * k + 2]), "r"(w[4 * k + 3]) : "memory");
                if (by_map) {  // rows and columns outside the map are not written
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        if (!RAGGED || c < mapped) store_box(&j.out_map, (int32_t)(t.n0 + c), (int32_t)row0, (int32_t)t.split, piece);
                        else asm volatile("cp.async.bulk.commit_group;" ::: "memory");  // pieces are counted by it
                    }
                    // what is left behind the map's last sixteen bytes is one part of sixteen more: by the lane that has put its row there
                    if (RAGGED && mapped < width && c + kPiece > mapped && lane < live) {
                        uint32_t q[4];
                        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3])
                                     : "r"(piece + lane * 64 + ((((mapped - c) * (uint32_t)sizeof(T) >> 4) ^ ((lane >> 1) & 3u)) << 4)));
                        T* const to = out + (row0 + lane) * ld + t.n0 + mapped;
                        const uint32_t bytes = (width - mapped) * sizeof(T);
                        if (bytes & 8u) *reinterpret_cast<uint2*>(to) = make_uint2(q[0], q[1]);
                        if (bytes & 4u) reinterpret_cast<uint32_t*>(to)[bytes & 8u ? 2 : 0] = bytes & 8u ? q[2] : q[0];
                        if (bytes & 2u) reinterpret_cast<uint16_t*>(to)[(bytes >> 1) - 1] = (uint16_t)(bytes & 8u ? bytes & 4u ? q[3] : q[2] : bytes & 4u ? q[1] : q[0]);
                    }
                } else {  // two rows at a time, neighbouring lanes neighbouring words (or elements, of rows that do not begin at words)
                    __syncwarp();
                    T* const to = out + t.split * part_elements + row0 * ld + t.n0 + c;
                    const uint32_t left = width - c, k = lane & 15u;
                    for (uint32_t r = lane >> 4; r < live; r += 2) {
                        uint32_t word;
                        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(word) : "r"(piece + r * 64 + (((k >> 2) ^ ((r >> 1) & 3u)) << 4) + (k & 3u) * 4));
                        if constexpr (sizeof(T) == 4) {
                            if (k < left) reinterpret_cast<uint32_t*>(to + r * ld)[k] = word;
                        } else {
                            uint16_t* const p = reinterpret_cast<uint16_t*>(to + r * ld) + 2 * k;
                            if (by_word && 2 * k + 1 < left) *reinterpret_cast<uint32_t*>(p) = word;
                            else {
                                if (2 * k < left) p[0] = (uint16_t)word;
                                if (2 * k + 1 < left) p[1] = (uint16_t)(word >> 16);
                            }
                        }
                    }
                }
            }
            sum.next(sums);
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0 && s_quit) atomicAdd(&g_gave_up, 1u);
    cluster_sync();  // neither CTA's shared or tensor memory is in use by the other any more
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// The parts of a split contraction, added up in their order, behind the sum of those before them (before: NULL where there are none).
template <class T>
__global__ void __launch_bounds__(256) k_add_parts(const float* before, const float* parts, uint32_t splits, uint64_t part_elements, uint64_t m, uint64_t n, uint64_t part_ld,
                                                   T* out, uint64_t ld) {
    let_next_start();
    wait_for_previous();
    parts = from_previous(parts);
    before = from_previous(before);
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < m * (part_ld / 4); i += (uint64_t)gridDim.x * 256) {
        const uint64_t row = i / (part_ld / 4), col = (i - row * (part_ld / 4)) * 4;
        float4 sum = before ? *reinterpret_cast<const float4*>(before + row * part_ld + col) : make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t p = 0; p < splits; ++p) {
            const float4 v = *reinterpret_cast<const float4*>(parts + p * part_elements + row * part_ld + col);
            sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        const float s[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (col + k < n) out[row * ld + col + k] = one<T>(s[k]);
    }
}

// The kernel's shared memory, allowed once on every device (devices beyond 63: with every call).
template <class T, bool RAGGED>
cudaError_t allow_smem() {
    static std::atomic<uint64_t> done{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = device >= 0 && device < 64 ? 1ull << device : 0;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(k_product<T, RAGGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

template <class T, bool RAGGED>
cudaError_t product_into(const ProductJob& j, T* out, uint64_t ld, uint64_t part_elements, cudaStream_t s) {
    const cudaError_t e = allow_smem<T, RAGGED>();
    if (e != cudaSuccess) return e;
    const uint32_t tiles = j.plan.tiles_m * j.plan.tiles_n * j.plan.splits;
    launch_after(k_product<T, RAGGED>, 2 * std::min<uint32_t>(tiles, kSms / 2), kThreads, kSmemBytes, s, j, out, ld, part_elements);
    return cudaGetLastError();
}
template <class T>
cudaError_t product(const ProductJob& j, cudaStream_t s) {
    // What a warp does about a row's end costs the others too (131072 x 1152 x 768 124 us instead of 120): products without one have a kernel without it.
    if (j.plan.splits == 1) return j.map_cols && j.map_cols < j.n ? product_into<T, true>(j, (T*)j.out, j.ld, 0, s) : product_into<T, false>(j, (T*)j.out, j.ld, 0, s);
    const uint64_t part_ld = product_part_ld(j.n), part = j.m * part_ld;
    const uint32_t ctas = (uint32_t)std::min<uint64_t>((j.m * (part_ld / 4) + 255) / 256, (uint64_t)kSms * 8), splits = j.plan.splits;
    float* const sum = j.parts + j.plan.together * part;  // of the parts so far, where they are not all made together
    ProductJob some = j;
    for (uint32_t first = 0; first < splits; first += some.plan.splits) {
        some.first_group = first * j.plan.split_groups;
        some.plan.splits = std::min(j.plan.together, splits - first);
        const cudaError_t e = product_into<float, false>(some, j.parts, part_ld, part, s);
        if (e != cudaSuccess) return e;
        const float* const before = first ? sum : nullptr;
        if (first + some.plan.splits < splits) launch_after(k_add_parts<float>, ctas, 256, 0, s, before, j.parts, some.plan.splits, part, j.m, j.n, part_ld, sum, part_ld);
        else launch_after(k_add_parts<T>, ctas, 256, 0, s, before, j.parts, some.plan.splits, part, j.m, j.n, part_ld, (T*)j.out, j.ld);
    }
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_product(const ProductJob& j, cudaStream_t s) {
    if (j.dtype == DG_F32) return product<float>(j, s);
    if (j.dtype == DG_BF16) return product<__nv_bfloat16>(j, s);
    return product<__half>(j, s);
}

cudaError_t product_gave_up(unsigned int* count, cudaStream_t s) {
    void* at = nullptr;
    cudaError_t e = cudaGetSymbolAddress(&at, g_gave_up);
    *count = 0;
    if (e == cudaSuccess) e = cudaMemcpyAsync(count, at, sizeof *count, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    return e;
}

}  // namespace dg
