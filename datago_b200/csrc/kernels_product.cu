// Product of 8-bit rows: out[m][n] = sum over k of a[m][k] * 2^(ea - 127) * b[n][k] * 2^(eb - 127), a scale per 128 columns of a row.
//
// The tensor cores multiply e4m3 blocks with E8M0 scales themselves (tcgen05.mma kind::mxf8f6f4, one scale byte per row and 32
// columns): the four instructions of a 128-column group name the same byte, so scales are neither repeated in memory nor applied
// by other units, and the sum stays in tensor memory, in 32 bits, from the first group to the last.
//
// A persistent CTA per SM walks output tiles of 128 x tile_n.  Its warps:
//   copier    one thread; a ring slot holds 128 columns of both operands (two tensor-map copies, 128-byte swizzle)
//   issuer    one thread; four instructions per slot, and per four groups the copies of the scales into tensor memory
//   scaler    one warp; fetches the scale bytes of four groups (a word per row) and lays them out for those copies: row r of 128 at
//             (r % 32) * 16 + (r / 32) * 4
//   4 storers read the sums of a finished tile out of tensor memory, one lane a row, round and store them, while the issuer is at
//             the next tile (two accumulators)
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

constexpr uint32_t kTileM = kProductTileM, kMaxTileN = kProductMaxTileN;
constexpr uint32_t kStages = 4, kScaleStages = 4;
constexpr uint32_t kABytes = kTileM * 128, kBBytes = kMaxTileN * 128, kStageBytes = kABytes + kBBytes;
constexpr uint32_t kScaleBytes = 512 * 3;  // of four groups: 128 rows of a, 256 of b
constexpr uint32_t kThreads = 256;
constexpr uint32_t kSmemBytes = kStages * kStageBytes + kScaleStages * kScaleBytes + 1024;
// tensor memory: the accumulators from columns 0 and 256, behind each of them the scales of every other four groups (a: 4 columns, b: 8)
constexpr uint32_t kSecond = 256, kScalesAt = kMaxTileN;
static_assert(kScalesAt + 12 <= kSecond, "the scales fit behind an accumulator");
constexpr uint32_t kWaitLimit = 1u << 20;  // waits of up to 2 us each

__device__ unsigned int g_gave_up;

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(done) : "r"(bar), "r"(parity), "r"(2000u) : "memory");
    return done != 0;
}
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
// arrives on the barrier when all tensor-core work that this thread has issued is done
__device__ __forceinline__ void commit_to(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// Shared-memory descriptors.  Operands: rows of 128 bytes, 128-byte swizzle, eight rows (1024 bytes) apart.  Scales: no swizzle,
// eight rows of 16 bytes (128 bytes) apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t at) {
    return (uint64_t)((at >> 4) & 0x3FFFu) | 1ull << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
__device__ __forceinline__ uint64_t scales_desc(uint32_t at) { return (uint64_t)((at >> 4) & 0x3FFFu) | (uint64_t)(128 >> 4) << 32 | 1ull << 46; }
__device__ __forceinline__ void copy_scales(uint32_t columns, uint32_t at) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(columns), "l"(scales_desc(at)) : "memory");
}
__device__ __forceinline__ void multiply(uint32_t acc, uint64_t a, uint64_t b, uint32_t what, uint32_t a_scales, uint32_t b_scales, bool add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}"
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

// sixteen neighbouring columns of a row, `left` of them inside the matrix
template <class T>
__device__ __forceinline__ void store_16(T* p, const uint32_t v[16], uint64_t left, bool whole) {
    if (whole && left >= 16) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) reinterpret_cast<uint4*>(p)[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        } else {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = pair(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]), T());
            reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
            reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j)
            if (j < left) p[j] = one<T>(__uint_as_float(v[j]));
    }
}

struct Place {  // in a ring: the slot, and the parity of its fillings so far
    uint32_t slot = 0, phase = 0;
    __device__ __forceinline__ void next(uint32_t n) {
        if (++slot == n) { slot = 0; phase ^= 1u; }
    }
};

// Four scale bytes (groups 4 q .. 4 q + 3) of row r; 0 for rows that the matrix does not have.
__device__ __forceinline__ uint32_t scale_word(const uint8_t* scales, uint64_t ld, uint32_t block, uint64_t r, uint64_t rows, uint32_t q) {
    return r < rows ? *reinterpret_cast<const uint32_t*>(scales + (block == 1 ? r : r / kScaleGroup) * ld + 4ull * q) : 0u;
}

template <class T>
__global__ void __launch_bounds__(kThreads, 1) k_product(const __grid_constant__ ProductJob j, T* out, uint64_t ld, uint64_t part_elements, bool whole) {
    extern __shared__ unsigned char raw_smem[];
    __shared__ __align__(8) unsigned long long s_bar[2 * kStages + 2 * kScaleStages + 5];
    __shared__ uint32_t s_tmem;
    __shared__ volatile uint32_t s_quit;
    const uint32_t smem = ((uint32_t)__cvta_generic_to_shared(raw_smem) + 1023u) & ~1023u;  // the swizzle counts from multiples of 1024
    const uint32_t scales_at = smem + kStages * kStageBytes;
    const uint32_t bar = (uint32_t)__cvta_generic_to_shared(s_bar);
    auto full = [&](uint32_t i) { return bar + 8 * i; };
    auto empty = [&](uint32_t i) { return bar + 8 * (kStages + i); };
    auto scales_full = [&](uint32_t i) { return bar + 8 * (2 * kStages + i); };
    auto scales_empty = [&](uint32_t i) { return bar + 8 * (2 * kStages + kScaleStages + i); };
    auto sums_full = [&](uint32_t i) { return bar + 8 * (2 * kStages + 2 * kScaleStages + i); };
    auto sums_empty = [&](uint32_t i) { return bar + 8 * (2 * kStages + 2 * kScaleStages + 2 + i); };
    const uint32_t over = bar + 8 * (2 * kStages + 2 * kScaleStages + 4);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    let_next_start();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"((uint32_t)__cvta_generic_to_shared(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kStages; ++i) { bar_init(full(i), 1); bar_init(empty(i), 1); }
        for (uint32_t i = 0; i < kScaleStages; ++i) { bar_init(scales_full(i), 1); bar_init(scales_empty(i), 1); }
        for (uint32_t i = 0; i < 2; ++i) { bar_init(sums_full(i), 1); bar_init(sums_empty(i), 4); }
        bar_init(over, 1);
        s_quit = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
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
    const uint32_t tile_n = j.plan.tile_n, tiles_n = j.plan.tiles_n, per_split = j.plan.tiles_m * tiles_n;
    const uint32_t tiles = per_split * j.plan.splits;
    const uint32_t groups = (uint32_t)((j.k + kScaleGroup - 1) / kScaleGroup);
    // what a tile index stands for: the part of the contraction, the first row and column, the groups
    struct Tile { uint32_t split, m0, n0, g0, g1; };
    auto tile_at = [&](uint32_t i) {
        Tile t;
        t.split = i / per_split;
        const uint32_t r = i - t.split * per_split, tm = r / tiles_n;
        t.m0 = tm * kTileM;
        t.n0 = (r - tm * tiles_n) * tile_n;
        t.g0 = t.split * j.plan.split_groups;
        t.g1 = min(groups, t.g0 + j.plan.split_groups);
        return t;
    };

    if (warp == 0) {
        if (lane == 0) {  // ---- copier
            Place at;
            uint32_t filled = 0;
            const uint32_t bytes = kABytes + tile_n * 128;
            bool go_on = true;
            for (uint32_t i = blockIdx.x; go_on && i < tiles; i += gridDim.x) {
                const Tile t = tile_at(i);
                for (uint32_t g = t.g0; go_on && g < t.g1; ++g) {
                    if (filled >= kStages) go_on = wait_for(empty(at.slot), at.phase ^ 1u);
                    if (!go_on) break;
                    bar_expect(full(at.slot), bytes);
                    const uint32_t to = smem + at.slot * kStageBytes;
                    copy_box(to, &j.a, (int32_t)(g * 128), (int32_t)t.m0, full(at.slot));
                    copy_box(to + kABytes, &j.b, (int32_t)(g * 128), (int32_t)t.n0, full(at.slot));
                    ++filled;
                    at.next(kStages);
                }
            }
            // nothing may arrive in the shared memory of a CTA that has gone
            for (uint32_t c = filled > kStages ? filled - kStages : 0; c < filled; ++c) {
                uint32_t polls = 0;
                while (!bar_try(full(c % kStages), (c / kStages) & 1u) && ++polls <= kWaitLimit) {}
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {  // ---- issuer
            // the instruction: e4m3 by e4m3, E8M0 scales, 32-bit sums, 128 x tile_n; the scale byte of a group is filled in below
            const uint32_t base = 1u << 23 | (tile_n >> 3) << 17 | (kTileM >> 7) << 27;
            Place at, sc;
            uint32_t quads = 0, done = 0;
            bool go_on = true;
            for (uint32_t i = blockIdx.x; go_on && i < tiles; i += gridDim.x, ++done) {
                const Tile t = tile_at(i);
                const uint32_t which = done & 1u, acc = tmem + which * kSecond;
                if (done >= 2 && !(go_on = wait_for(sums_empty(which), ((done >> 1) & 1u) ^ 1u))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t a_scales = 0, b_scales = 0;
                for (uint32_t g = t.g0; g < t.g1; ++g) {
                    const uint32_t byte = (g - t.g0) & 3u;
                    if (byte == 0) {
                        // the columns that these scales go to were read by the instructions of the quad before the last
                        if (quads >= 2) {
                            const uint32_t q = quads - 2;
                            if (!(go_on = wait_for(scales_empty(q % kScaleStages), (q / kScaleStages) & 1u))) break;
                        }
                        if (!(go_on = wait_for(scales_full(sc.slot), sc.phase))) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        a_scales = tmem + (quads & 1u) * kSecond + kScalesAt;
                        b_scales = a_scales + 4;
                        const uint32_t from = scales_at + sc.slot * kScaleBytes;
                        copy_scales(a_scales, from);
                        copy_scales(b_scales, from + 512);
                        if (tile_n > 128) copy_scales(b_scales + 4, from + 1024);
                    }
                    if (!(go_on = wait_for(full(at.slot), at.phase))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t da = operand_desc(smem + at.slot * kStageBytes), db = operand_desc(smem + at.slot * kStageBytes + kABytes);
                    const uint32_t what = base | byte << 4 | byte << 29;
                    const uint32_t steps = (uint32_t)min((uint64_t)4, (uint64_t)(j.k - 128ull * g + 31) / 32);
                    for (uint32_t s = 0; s < steps; ++s)  // 32 columns: 32 bytes further in the swizzled rows
                        multiply(acc, da + 2 * s, db + 2 * s, what, a_scales, b_scales, g != t.g0 || s != 0);
                    commit_to(empty(at.slot));
                    at.next(kStages);
                    if (byte == 3 || g + 1 == t.g1) {
                        commit_to(scales_empty(sc.slot));
                        sc.next(kScaleStages);
                        ++quads;
                    }
                }
                if (!go_on) break;
                commit_to(sums_full(which));
            }
            if (!go_on) {  // what has been issued ends before the CTA does
                uint32_t polls = 0;
                commit_to(over);
                while (!bar_try(over, 0) && ++polls <= kWaitLimit) {}
            }
        }
    } else if (warp == 2) {  // ---- scaler
        Place sc;
        uint32_t quads = 0;
        bool go_on = true;
        const uint8_t *const pa = from_previous(j.a_scales), *const pb = from_previous(j.b_scales);
        for (uint32_t i = blockIdx.x; go_on && i < tiles; i += gridDim.x) {
            const Tile t = tile_at(i);
            for (uint32_t g = t.g0; g < t.g1; g += 4, ++quads) {
                uint32_t w[12];
#pragma unroll
                for (int r = 0; r < 4; ++r) w[r] = scale_word(pa, j.a_scale_ld, j.a_block, (uint64_t)t.m0 + lane + 32 * r, j.m, g >> 2);
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    w[4 + r] = 32 * r < tile_n ? scale_word(pb, j.b_scale_ld, j.b_block, (uint64_t)t.n0 + lane + 32 * r, j.n, g >> 2) : 0u;
                if (quads >= kScaleStages) go_on = __all_sync(0xFFFFFFFFu, wait_for(scales_empty(sc.slot), sc.phase ^ 1u));
                if (!go_on) break;
                const uint32_t to = scales_at + sc.slot * kScaleBytes + lane * 16;
#pragma unroll
                for (int b = 0; b < 3; ++b)
                    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(to + 512 * b), "r"(w[4 * b]), "r"(w[4 * b + 1]), "r"(w[4 * b + 2]),
                                 "r"(w[4 * b + 3]) : "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) bar_arrive(scales_full(sc.slot));
                sc.next(kScaleStages);
            }
        }
    } else if (warp >= 4) {  // ---- storers
        const uint32_t rows = (warp & 3u) * 32;
        uint32_t done = 0;
        bool go_on = true;
        for (uint32_t i = blockIdx.x; go_on && i < tiles; i += gridDim.x, ++done) {
            const Tile t = tile_at(i);
            const uint32_t which = done & 1u;
            go_on = __all_sync(0xFFFFFFFFu, wait_for(sums_full(which), (done >> 1) & 1u));
            if (!go_on) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t from = tmem + which * kSecond + (rows << 16);
            const uint64_t row = (uint64_t)t.m0 + rows + lane;
            T* const to = out + t.split * part_elements + row * ld + t.n0;
            for (uint32_t c = 0; c < tile_n; c += 16) {
                uint32_t v[16];
                read_16(from + c, v);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (row < j.m && t.n0 + c < j.n) store_16(to + c, v, j.n - t.n0 - c, whole);
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(sums_empty(which));
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0 && s_quit) atomicAdd(&g_gave_up, 1u);
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// The parts of a split contraction, added up in their order.
template <class T>
__global__ void __launch_bounds__(256) k_add_parts(const float* parts, uint32_t splits, uint64_t part_elements, uint64_t m, uint64_t n, uint64_t part_ld, T* out,
                                                   uint64_t ld) {
    let_next_start();
    wait_for_previous();
    parts = from_previous(parts);
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < m * (part_ld / 4); i += (uint64_t)gridDim.x * 256) {
        const uint64_t row = i / (part_ld / 4), col = (i - row * (part_ld / 4)) * 4;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
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
template <class T>
cudaError_t allow_smem() {
    static std::atomic<uint64_t> done{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = device >= 0 && device < 64 ? 1ull << device : 0;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(k_product<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

template <class T>
cudaError_t product_into(const ProductJob& j, T* out, uint64_t ld, uint64_t part_elements, cudaStream_t s) {
    const cudaError_t e = allow_smem<T>();
    if (e != cudaSuccess) return e;
    const uint32_t tiles = j.plan.tiles_m * j.plan.tiles_n * j.plan.splits;
    const bool whole = ((reinterpret_cast<uintptr_t>(out) | (ld * sizeof(T)) | (part_elements * sizeof(T))) & 15u) == 0;
    launch_after(k_product<T>, std::min<uint32_t>(tiles, kSms), kThreads, kSmemBytes, s, j, out, ld, part_elements, whole);
    return cudaGetLastError();
}
template <class T>
cudaError_t product(const ProductJob& j, cudaStream_t s) {
    if (j.plan.splits == 1) return product_into<T>(j, (T*)j.out, j.ld, 0, s);
    const uint64_t part_ld = (j.n + 3) / 4 * 4, part = j.m * part_ld;
    const cudaError_t e = product_into<float>(j, j.parts, part_ld, part, s);
    if (e != cudaSuccess) return e;
    const uint32_t ctas = (uint32_t)std::min<uint64_t>((j.m * (part_ld / 4) + 255) / 256, (uint64_t)kSms * 8);
    launch_after(k_add_parts<T>, ctas, 256, 0, s, j.parts, j.plan.splits, part, j.m, j.n, part_ld, (T*)j.out, j.ld);
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
    if (e == cudaSuccess && *count) {
        e = cudaMemsetAsync(at, 0, sizeof *count, s);
        if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    }
    return e;
}

}  // namespace dg
