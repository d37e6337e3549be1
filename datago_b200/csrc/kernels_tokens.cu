// Token rows: patches and matrices as 8-bit rows, the norm after the positions have been added, dropout.
//
// All of these read their inputs once and write their outputs once; memory bounds them.  A thread owns vectors of eight neighbouring
// columns (16 bytes of bf16), so that sixteen neighbouring lanes hold the 128 columns that share a scale: the group's largest
// magnitude is four shuffles, and nothing between the load and the store leaves the registers.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdint>

#include "kernels.h"
#include "tokens.h"

namespace dg {

namespace {

using bf16 = __nv_bfloat16;

// ---- eight neighbouring elements ---------------------------------------------------------------------------------------
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 narrow<bf16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ void unpack8(const uint4& r, float v[8], bf16) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void unpack8(const uint4& r, float v[8], __half) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, bf16) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
    const __half2 p = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
}

// Up to eight elements from p on (`valid` of them; the others are 0).  whole: p is 16-byte aligned.  Plain loads: what an earlier
// kernel wrote is read.
template <class T>
__device__ __forceinline__ void load8(const T* p, uint32_t valid, bool whole, float v[8]) {
    if (whole && valid >= 8) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            unpack8(*reinterpret_cast<const uint4*>(p), v, T());
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) v[j] = j < valid ? widen(p[j]) : 0.f;
    }
}
template <class T>
__device__ __forceinline__ void store8(T* p, uint32_t valid, bool whole, const float v[8]) {
    if (whole && valid >= 8) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            if (j < valid) p[j] = narrow<T>(v[j]);
    }
}
__device__ __forceinline__ void load8_any(const void* p, uint64_t at, int32_t dtype, uint32_t valid, bool whole, float v[8]) {
    if (dtype == DG_F32) load8(reinterpret_cast<const float*>(p) + at, valid, whole, v);
    else if (dtype == DG_BF16) load8(reinterpret_cast<const bf16*>(p) + at, valid, whole, v);
    else load8(reinterpret_cast<const __half*>(p) + at, valid, whole, v);
}
template <class T> bool rows_aligned(const void* p, uint64_t ld) { return ((reinterpret_cast<uintptr_t>(p) | (ld * sizeof(T))) & 15u) == 0; }

// ---- scales -------------------------------------------------------------------------------------------------------------
// Magnitudes are compared as bit patterns: those of finite numbers order like the numbers, an infinity is above them and a NaN above that.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint32_t largest8(const float v[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, magnitude(v[j]));
    return m;
}
__device__ __forceinline__ uint32_t largest_of_16_lanes(uint32_t m) {
#pragma unroll
    for (int d = 8; d; d >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
    return m;
}
// The scale byte of a group whose largest magnitude has the bits m.  448 = 1.75 * 2^8: the exponent of m less 8, one more where the
// mantissa is above 1.75 (which adding 0x1FFFFF carries into the exponent).
__device__ __forceinline__ uint32_t scale_byte(uint32_t m) {
    return m >= 0x7F800000u ? 255u : (uint32_t)max((int32_t)((m + 0x1FFFFFu) >> 23) - 8, 0);
}
// 1 / scale, exactly: e is at most 247 for a finite group.  NaN for e = 255.
__device__ __forceinline__ float inverse_scale(uint32_t e) { return __uint_as_float(e == 255u ? 0x7FFFFFFFu : (254u - e) << 23); }
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | (uint32_t)hi << 16;
}
__device__ __forceinline__ uint2 quantize8(const float v[8], float inverse) {
    return make_uint2(e4m3x4(v[0] * inverse, v[1] * inverse, v[2] * inverse, v[3] * inverse),
                      e4m3x4(v[4] * inverse, v[5] * inverse, v[6] * inverse, v[7] * inverse));
}
// p is 8-byte aligned: rows of values start at multiples of 16
__device__ __forceinline__ void store_values8(uint8_t* p, uint32_t valid, uint2 q) {
    if (valid >= 8) *reinterpret_cast<uint2*>(p) = q;
    else
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            if (j < valid) p[j] = (uint8_t)((j < 4 ? q.x : q.y) >> (8 * (j & 3)));
}

// ---- rows of a matrix or of a bucket's patches -----------------------------------------------------------------------------
template <class T> struct MatrixSource {
    const T* data;
    uint64_t ld;
    bool whole;
    __device__ __forceinline__ void load(uint64_t row, uint32_t col, uint32_t valid, float v[8]) const {
        load8(from_previous(data) + row * ld + col, valid, whole, v);
    }
};
// C channels.  A patch's row of pixels is patch * C neighbouring bytes; whole: those begin at multiples of eight, everywhere.
template <int C> struct PatchSource {
    const uint8_t* pixels;
    uint32_t grid_w, per_image, patch, segment;  // patches per row and per image; segment = patch * C
    uint64_t pitch, image;                       // bytes of a row of pixels and of an image
    float gain[C], shift[C];
    bool whole;
    __device__ __forceinline__ void load(uint64_t row, uint32_t col, uint32_t valid, float v[8]) const {
        const uint64_t i = row / per_image;
        const uint32_t r = (uint32_t)(row - i * per_image), Y = r / grid_w, X = r - Y * grid_w;
        const uint8_t* p = from_previous(pixels) + i * image + (uint64_t)Y * patch * pitch + (uint64_t)X * segment;
        uint32_t y = col / segment, b = col - y * segment;
        const uint32_t phase = col % C;  // channel of the first feature
        uint32_t px[8];
        if (whole && valid >= 8) {
            const uint2 w = *reinterpret_cast<const uint2*>(p + y * pitch + b);
#pragma unroll
            for (int j = 0; j < 8; ++j) px[j] = ((j < 4 ? w.x : w.y) >> (8 * (j & 3))) & 255u;
        } else {
            const uint8_t* q = p + y * pitch;
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                px[j] = j < valid ? q[b] : 0;
                if (++b == segment) { b = 0; q += pitch; }
            }
        }
        float g[C], s[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            g[c] = gain[c];
            s[c] = shift[c];
#pragma unroll
            for (int k = 1; k < C; ++k)
                if (phase == (uint32_t)k) { g[c] = gain[(c + k) % C]; s[c] = shift[(c + k) % C]; }
        }
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) v[j] = j < valid ? fmaf((float)px[j], g[j % C], s[j % C]) : 0.f;
    }
};

constexpr uint32_t kRowThreads = 256;

// Sixteen lanes per group of 128 columns; four groups of a half-warp in flight.
template <class Source>
__global__ void __launch_bounds__(kRowThreads) k_rows8(Source src, uint64_t ngroups, uint32_t groups, uint32_t cols, uint8_t* values, uint64_t ld,
                                                       uint8_t* scales, uint64_t scale_ld) {
    let_next_start();
    wait_for_previous();
    const uint32_t lane = threadIdx.x & 15u;
    const uint64_t stride = (uint64_t)gridDim.x * (kRowThreads / 16);
    // whole half-warps leave together, and a warp's two halves differ by one group: both stay while the lower one has work
    for (uint64_t g = (uint64_t)blockIdx.x * (kRowThreads / 16) + (threadIdx.x >> 4); (g & ~1ull) < ngroups; g += stride) {
        const uint64_t row = g / groups;
        const uint32_t group = (uint32_t)(g - row * groups), col = group * kScaleGroup + lane * 8;
        const uint32_t valid = g < ngroups && col < cols ? min(8u, cols - col) : 0;
        float v[8] = {};
        if (valid) src.load(row, col, valid, v);
        const uint32_t e = scale_byte(largest_of_16_lanes(largest8(v)));
        if (valid) store_values8(values + row * ld + col, valid, quantize8(v, inverse_scale(e)));
        if (lane == 0 && valid) scales[row * scale_ld + group] = (uint8_t)e;
    }
}

template <class Source, class T>
__global__ void __launch_bounds__(kRowThreads) k_rows(Source src, uint64_t nvec, uint32_t per_row, uint32_t cols, T* out, uint64_t ld, bool whole) {
    let_next_start();
    wait_for_previous();
    for (uint64_t i = (uint64_t)blockIdx.x * kRowThreads + threadIdx.x; i < nvec; i += (uint64_t)gridDim.x * kRowThreads) {
        const uint64_t row = i / per_row;
        const uint32_t col = (uint32_t)(i - row * per_row) * 8, valid = min(8u, cols - col);
        float v[8];
        src.load(row, col, valid, v);
        store8(out + row * ld + col, valid, whole, v);
    }
}

uint32_t grid_for(uint64_t items, uint32_t per_cta, uint32_t ctas_per_sm) {
    return (uint32_t)std::min<uint64_t>((items + per_cta - 1) / per_cta, (uint64_t)kSms * ctas_per_sm);
}

template <class Source>
void rows8(const Source& src, const dg_rows8& out, cudaStream_t s) {
    const uint64_t groups = scale_groups(out.cols), n = out.rows * groups;
    launch_after(k_rows8<Source>, grid_for(n, kRowThreads / 16, 32), kRowThreads, 0, s, src, n, (uint32_t)groups, (uint32_t)out.cols, out.values, out.ld,
                 out.scales, out.scale_ld);
}
template <class Source, class T>
void rows_as(const Source& src, const dg_matrix& out, cudaStream_t s) {
    const uint64_t per_row = (out.cols + 7) / 8, n = out.rows * per_row;
    launch_after(k_rows<Source, T>, grid_for(n, kRowThreads, 32), kRowThreads, 0, s, src, n, (uint32_t)per_row, (uint32_t)out.cols, (T*)out.data, out.ld,
                 rows_aligned<T>(out.data, out.ld));
}

template <int C>
void patch_rows(const PatchJob& j, const dg_rows8* out8, const dg_matrix* out, cudaStream_t s) {
    PatchSource<C> src;
    src.pixels = j.pixels;
    src.grid_w = j.w / j.patch;
    src.per_image = src.grid_w * (j.h / j.patch);
    src.patch = j.patch;
    src.segment = j.patch * C;
    src.pitch = (uint64_t)j.w * C;
    src.image = src.pitch * j.h;
    src.whole = ((reinterpret_cast<uintptr_t>(j.pixels) | src.pitch | src.segment) & 7u) == 0;
    for (int c = 0; c < C; ++c) { src.gain[c] = j.gain[c]; src.shift[c] = j.shift[c]; }
    if (out8) rows8(src, *out8, s);
    else if (out->dtype == DG_F32) rows_as<PatchSource<C>, float>(src, *out, s);
    else if (out->dtype == DG_BF16) rows_as<PatchSource<C>, bf16>(src, *out, s);
    else rows_as<PatchSource<C>, __half>(src, *out, s);
}

// ---- scales along the rows of the source, and of 128 x 128 blocks -------------------------------------------------------------
// The transpose of a matrix stays in the order of the matrix (dg_rows8.by_column): only its scales run along the rows.  A warp holds 256 columns
// of ROWS rows as they were loaded; the warps of a CTA have 128 rows, the group of a scale, and meet twice over its 256 columns' maxima.
template <class T> constexpr int kColumnRows = sizeof(T) == 4 ? 8 : 16;  // what fits the registers
template <class T> constexpr uint32_t kColumnThreads = 128 / kColumnRows<T> * 32;
constexpr uint32_t kColumnTile = 256;

template <class T> struct Raw8 {  // eight neighbouring elements as they are in memory
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void widen(float v[8]) const {
        if constexpr (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(&w[0]), b = *reinterpret_cast<const float4*>(&w[1]);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            unpack8(w[0], v, T());
        }
    }
    __device__ __forceinline__ void load(const T* p, uint32_t valid, bool whole) {
        if (whole && valid >= 8) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
        } else {
            T e[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) e[j] = j < valid ? p[j] : narrow<T>(0.f);
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(e)[i];
        }
    }
};
// Magnitudes of two 16-bit elements compared at once: like those of 32 bits, they order as whole numbers.
__device__ __forceinline__ uint32_t larger(uint32_t top, uint32_t v, bf16) { return __vmaxu2(top, v & 0x7FFF7FFFu); }
__device__ __forceinline__ uint32_t larger(uint32_t top, uint32_t v, __half) { return __vmaxu2(top, v & 0x7FFF7FFFu); }
__device__ __forceinline__ uint32_t larger(uint32_t top, uint32_t v, float) { return max(top, v & 0x7FFFFFFFu); }
// the magnitude of 32 bits of one of them
__device__ __forceinline__ uint32_t magnitude_of(uint32_t half, bf16) { return half << 16; }
__device__ __forceinline__ uint32_t magnitude_of(uint32_t half, __half) { return __float_as_uint(__half2float(__ushort_as_half((unsigned short)half))); }

// BLOCK: one scale for 128 columns too.  scale_row / scale_col: how far apart the scales of neighbouring groups of rows and of neighbouring
// columns (blocks of 128 columns) are.
template <class T, bool BLOCK>
__global__ void __launch_bounds__(kColumnThreads<T>, 2) k_columns8(const T* src, uint64_t rows, uint64_t cols, uint64_t ld, bool whole, uint32_t tiles_x, uint64_t tiles,
                                                                   uint8_t* values, uint64_t out_ld, uint8_t* scales, uint64_t scale_row, uint64_t scale_col) {
    constexpr int R = kColumnRows<T>, kWarps = 128 / R, kWords = sizeof(T) * 2;
    __shared__ __align__(16) uint32_t s_top[kWarps][32][kWords];
    __shared__ __align__(16) float s_inverse[kColumnTile];
    let_next_start();
    wait_for_previous();
    src = from_previous(src);
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    for (uint64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const uint64_t ty = tile / tiles_x, c0 = (tile - ty * tiles_x) * kColumnTile, col = c0 + 8 * lane, r0 = ty * 128 + warp * R;
        const uint32_t valid = col < cols ? (uint32_t)min((uint64_t)8, cols - col) : 0;
        Raw8<T> x[R];
#pragma unroll
        for (int i = 0; i < R; ++i) x[i].load(src + (r0 + i) * ld + col, r0 + i < rows ? valid : 0, whole);
        uint32_t top[kWords] = {};
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int k = 0; k < kWords / 4; ++k) {
                top[4 * k] = larger(top[4 * k], x[i].w[k].x, T());
                top[4 * k + 1] = larger(top[4 * k + 1], x[i].w[k].y, T());
                top[4 * k + 2] = larger(top[4 * k + 2], x[i].w[k].z, T());
                top[4 * k + 3] = larger(top[4 * k + 3], x[i].w[k].w, T());
            }
#pragma unroll
        for (int k = 0; k < kWords / 4; ++k) *reinterpret_cast<uint4*>(&s_top[warp][lane][4 * k]) = make_uint4(top[4 * k], top[4 * k + 1], top[4 * k + 2], top[4 * k + 3]);
        __syncthreads();
        for (uint32_t c = threadIdx.x; c < kColumnTile; c += kColumnThreads<T>) {  // a thread per column
            uint32_t m = 0;
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int w = 0; w < kWarps; ++w) m = max(m, s_top[w][c >> 3][c & 7u]);
            } else {
#pragma unroll
                for (int w = 0; w < kWarps; ++w) m = max(m, s_top[w][c >> 3][(c & 7u) >> 1] >> (16 * (c & 1u)) & 0xFFFFu);
                m = magnitude_of(m, T());
            }
            if constexpr (BLOCK) {  // 128 columns are four whole warps
                m = __reduce_max_sync(0xFFFFFFFFu, m);
                __shared__ uint32_t s_warp[kColumnTile / 32];
                if (lane == 0) s_warp[c >> 5] = m;
                asm volatile("bar.sync 1, 256;" ::: "memory");  // the 256 threads that are here
                const uint32_t first = c >> 7 << 2;
                m = max(max(s_warp[first], s_warp[first + 1]), max(s_warp[first + 2], s_warp[first + 3]));
                if ((c & 127u) == 0 && c0 + c < cols) scales[ty * scale_row + (c0 + c) / 128 * scale_col] = (uint8_t)scale_byte(m);
            } else if (c0 + c < cols) {
                scales[ty * scale_row + (c0 + c) * scale_col] = (uint8_t)scale_byte(m);
            }
            s_inverse[c] = inverse_scale(scale_byte(m));
        }
        __syncthreads();
        float inverse[8];
        *reinterpret_cast<float4*>(inverse) = *reinterpret_cast<const float4*>(&s_inverse[8 * lane]);
        *reinterpret_cast<float4*>(inverse + 4) = *reinterpret_cast<const float4*>(&s_inverse[8 * lane + 4]);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (!valid || r0 + i >= rows) continue;
            float v[8];
            x[i].widen(v);
            store_values8(values + (r0 + i) * out_ld + col, valid,
                          make_uint2(e4m3x4(v[0] * inverse[0], v[1] * inverse[1], v[2] * inverse[2], v[3] * inverse[3]),
                                     e4m3x4(v[4] * inverse[4], v[5] * inverse[5], v[6] * inverse[6], v[7] * inverse[7])));
        }
    }
}

template <class T>
void quantize_rows(const dg_matrix& m, const dg_rows8& out, cudaStream_t s) {
    const bool whole = rows_aligned<T>(m.data, m.ld);
    if (!out.by_column && out.block == 1) {
        rows8(MatrixSource<T>{(const T*)m.data, m.ld, whole}, out, s);
        return;
    }
    const uint32_t tiles_x = (uint32_t)((m.cols + kColumnTile - 1) / kColumnTile);
    const uint64_t tiles = scale_groups(m.rows) * tiles_x;
    auto go = [&](auto kernel) {
        launch_after(kernel, grid_for(tiles, 1, 32), kColumnThreads<T>, 0, s, (const T*)m.data, m.rows, m.cols, m.ld, whole, tiles_x, tiles, out.values, out.ld,
                     out.scales, out.by_column ? 1 : out.scale_ld, out.by_column ? out.scale_ld : 1);
    };
    if (out.block == 1) go(k_columns8<T, false>);
    else go(k_columns8<T, true>);
}

// ---- norm ----------------------------------------------------------------------------------------------------------------------
// TPR threads hold a row, V vectors of eight columns each, consecutive threads consecutive vectors.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* s_part) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
    if constexpr (TPR > 32) {  // the warps of the row, added up in their order by every thread
        constexpr int kWarps = TPR / 32;
        const uint32_t first = threadIdx.x / TPR * kWarps;
        if ((threadIdx.x & 31u) == 0) s_part[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) v += s_part[first + i];
        __syncthreads();
    }
    return v;
}

template <class T, int V, int TPR, int THREADS>
__global__ void __launch_bounds__(THREADS) k_rms_norm(const NormJob a, bool x_whole, bool r_whole, bool w_whole, bool s_whole, bool y_whole) {
    __shared__ float s_part[THREADS / 32];
    let_next_start();
    wait_for_previous();
    const T *const px = from_previous(reinterpret_cast<const T*>(a.x)), *const pr = from_previous(reinterpret_cast<const T*>(a.residual));
    const void* const pw = from_previous(a.weight);
    constexpr uint32_t kRows = THREADS / TPR;
    const uint32_t t = threadIdx.x % TPR, mine = threadIdx.x / TPR;
    const float per_col = 1.f / (float)a.cols;
    for (uint64_t r0 = (uint64_t)blockIdx.x * kRows; r0 < a.rows; r0 += (uint64_t)gridDim.x * kRows) {
        const uint64_t row = r0 + mine;
        const bool live = row < a.rows;
        float h[V][8];
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const uint32_t col = (k * TPR + t) * 8, valid = live && col < a.cols ? min(8u, a.cols - col) : 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) h[k][j] = 0.f;
            if (valid) load8(px + row * a.x_ld + col, valid, x_whole, h[k]);
        }
        if (pr) {
            const uint64_t rr = row % a.residual_rows;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const uint32_t col = (k * TPR + t) * 8, valid = live && col < a.cols ? min(8u, a.cols - col) : 0;
                if (valid) {
                    float r[8];
                    load8(pr + rr * a.residual_ld + col, valid, r_whole, r);
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[k][j] += r[j];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(h[k][j], h[k][j], sum);
        const float rstd = 1.f / sqrtf(row_sum<TPR>(sum, s_part) * per_col + a.eps);
        if (live && t == 0 && a.rstd) a.rstd[row] = rstd;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const uint32_t col = (k * TPR + t) * 8, valid = live && col < a.cols ? min(8u, a.cols - col) : 0;
            if (a.sum && valid) store8(reinterpret_cast<T*>(a.sum) + row * a.sum_ld + col, valid, s_whole, h[k]);
            float w[8];
            if (pw && valid) {
                load8_any(pw, col, a.weight_dtype, valid, w_whole, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) h[k][j] = h[k][j] * rstd * w[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) h[k][j] *= rstd;
            }
            if (a.y && valid) store8(reinterpret_cast<T*>(a.y) + row * a.y_ld + col, valid, y_whole, h[k]);
            if (a.y8.values) {
                const uint32_t e = scale_byte(largest_of_16_lanes(largest8(h[k])));
                if (valid) {
                    store_values8(a.y8.values + row * a.y8.ld + col, valid, quantize8(h[k], inverse_scale(e)));
                    if ((t & 15u) == 0) a.y8.scales[row * a.y8.scale_ld + col / kScaleGroup] = (uint8_t)e;
                }
            }
        }
    }
}

template <class T>
void rms_norm(const NormJob& j, cudaStream_t s) {
    auto go = [&](auto kernel, uint32_t threads, uint32_t rows_per_cta) {
        launch_after(kernel, grid_for(j.rows, rows_per_cta, 2048 / threads * 4), threads, 0, s, j, rows_aligned<T>(j.x, j.x_ld), rows_aligned<T>(j.residual, j.residual_ld),
                     (reinterpret_cast<uintptr_t>(j.weight) & 15u) == 0, rows_aligned<T>(j.sum, j.sum_ld), rows_aligned<T>(j.y, j.y_ld));
    };
    const uint32_t vecs = (j.cols + 7) / 8;
    if (vecs <= 32) go(k_rms_norm<T, 1, 32, 256>, 256, 8);
    else if (vecs <= 64) go(k_rms_norm<T, 2, 32, 256>, 256, 8);
    else if (vecs <= 96) go(k_rms_norm<T, 3, 32, 256>, 256, 8);
    else if (vecs <= 128) go(k_rms_norm<T, 4, 32, 256>, 256, 8);
    else if (vecs <= 160) go(k_rms_norm<T, 5, 32, 256>, 256, 8);
    else if (vecs <= 192) go(k_rms_norm<T, 6, 32, 256>, 256, 8);
    else if (vecs <= 256) go(k_rms_norm<T, 8, 32, 256>, 256, 8);
    else if (vecs <= 512) go(k_rms_norm<T, 2, 256, 256>, 256, 1);
    else if (vecs <= 1024) go(k_rms_norm<T, 4, 256, 256>, 256, 1);
    else go(k_rms_norm<T, 4, 512, 512>, 512, 1);
}

// Backward.  A unit is a residual row t and a part of the rows r with r % period == t; TPR threads take a unit's rows one after the other
// and keep the sums of dx (for dresidual) of the unit and of dy * hat (for dweight) of all their units in registers.  CTAs write their
// dweight sums to the workspace; so do units their dresidual sums where a residual row has more than one unit.
template <class T, int V, int TPR, int THREADS>
__global__ void __launch_bounds__(THREADS) k_rms_norm_backward(const NormBackwardJob a, uint32_t parts, float* w_parts, float* r_parts, bool y_whole,
                                                               bool h_whole, bool w_whole, bool s_whole, bool x_whole) {
    constexpr uint32_t kRows = THREADS / TPR;
    __shared__ float s_part[THREADS / 32];
    __shared__ float s_sum[kRows > 1 ? V * TPR * 8 : 1];
    let_next_start();
    wait_for_previous();
    const T *const py = from_previous(reinterpret_cast<const T*>(a.dy)), *const ph = from_previous(reinterpret_cast<const T*>(a.h)),
            *const ps = from_previous(reinterpret_cast<const T*>(a.dsum));
    const void* const pw = from_previous(a.weight);
    const float* const prstd = from_previous(a.rstd);
    const uint32_t t = threadIdx.x % TPR, mine = threadIdx.x / TPR;
    const uint64_t units = a.period * parts, images = a.rows / a.period;
    const float per_col = 1.f / (float)a.cols;
    float dw[V][8] = {};
    for (uint64_t u0 = (uint64_t)blockIdx.x * kRows; u0 < units; u0 += (uint64_t)gridDim.x * kRows) {
        const uint64_t unit = u0 + mine, part = unit / a.period, at = unit - part * a.period;
        const bool there = unit < units;
        const uint64_t first = images * part / parts, last = there ? images * (part + 1) / parts : first;
        float dr[V][8] = {};
        // all threads of the CTA go through the same number of rows (they may meet in row_sum)
        const uint64_t most = (images + parts - 1) / parts;
        for (uint64_t i = 0; i < most; ++i) {
            const bool live = first + i < last;
            const uint64_t row = (first + i) * a.period + at;
            const float rstd = live ? prstd[row] : 0.f;
            float g[V][8], hat[V][8];
            float along = 0.f;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const uint32_t col = (k * TPR + t) * 8, valid = live && col < a.cols ? min(8u, a.cols - col) : 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) g[k][j] = hat[k][j] = 0.f;
                if (valid) {
                    load8(py + row * a.dy_ld + col, valid, y_whole, g[k]);
                    load8(ph + row * a.h_ld + col, valid, h_whole, hat[k]);
                }
            }
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const uint32_t col = (k * TPR + t) * 8, valid = live && col < a.cols ? min(8u, a.cols - col) : 0;
                float w[8];
                if (pw && valid) load8_any(pw, col, a.weight_dtype, valid, w_whole, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    hat[k][j] *= rstd;
                    dw[k][j] = fmaf(g[k][j], hat[k][j], dw[k][j]);
                    if (pw && valid) g[k][j] *= w[j];
                    along = fmaf(g[k][j], hat[k][j], along);
                }
            }
            along = row_sum<TPR>(along, s_part) * per_col;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const uint32_t col = (k * TPR + t) * 8, valid = live && col < a.cols ? min(8u, a.cols - col) : 0;
                float d[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) d[j] = rstd * (g[k][j] - hat[k][j] * along);
                if (ps && valid) {
                    float extra[8];
                    load8(ps + row * a.dsum_ld + col, valid, s_whole, extra);
#pragma unroll
                    for (int j = 0; j < 8; ++j) d[j] += extra[j];
                }
                if (a.dx && valid) store8(reinterpret_cast<T*>(a.dx) + row * a.dx_ld + col, valid, x_whole, d);
                if (valid)
#pragma unroll
                    for (int j = 0; j < 8; ++j) dr[k][j] += d[j];
            }
        }
        if (a.dresidual && there) {
            float* const to = (parts > 1 ? r_parts + part * a.period * a.cols : a.dresidual) + at * a.cols;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const uint32_t col = (k * TPR + t) * 8, valid = col < a.cols ? min(8u, a.cols - col) : 0;
                if (valid) store8(to + col, valid, (a.cols & 3u) == 0 && (reinterpret_cast<uintptr_t>(to) & 15u) == 0, dr[k]);
            }
        }
    }
    if (!a.dweight) return;
    float* const to = w_parts + (uint64_t)blockIdx.x * a.cols;
    if constexpr (kRows > 1) {  // the CTA's rows in their order
        for (uint32_t r = 0; r < kRows; ++r) {
            if (mine == r)
#pragma unroll
                for (int k = 0; k < V; ++k)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float& sum = s_sum[(k * TPR + t) * 8 + j];
                        sum = r ? sum + dw[k][j] : dw[k][j];
                    }
            __syncthreads();
        }
        for (uint32_t c = threadIdx.x; c < a.cols; c += THREADS) to[c] = s_sum[c];
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const uint32_t col = (k * TPR + t) * 8, valid = col < a.cols ? min(8u, a.cols - col) : 0;
            if (valid) store8(to + col, valid, false, dw[k]);
        }
    }
}

// out[i] = the sum of parts[p][i] in a fixed order: eight threads a column, each every eighth part
__global__ void __launch_bounds__(256) k_sum_parts(const float* parts, uint32_t count, uint64_t n, float* out) {
    __shared__ float s_sum[8][33];
    let_next_start();
    wait_for_previous();
    parts = from_previous(parts);
    const uint32_t lane = threadIdx.x & 31u, part = threadIdx.x >> 5;
    for (uint64_t i0 = (uint64_t)blockIdx.x * 32; i0 < n; i0 += (uint64_t)gridDim.x * 32) {
        const uint64_t i = i0 + lane;
        float sum = 0.f;
        if (i < n)
            for (uint32_t p = part; p < count; p += 8) sum += parts[p * n + i];
        s_sum[part][lane] = sum;
        __syncthreads();
        if (part == 0 && i < n) {
#pragma unroll
            for (int p = 1; p < 8; ++p) sum += s_sum[p][lane];
            out[i] = sum;
        }
        __syncthreads();
    }
}
__global__ void k_zero(float* out, uint64_t n) {
    wait_for_previous();
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (uint64_t)gridDim.x * blockDim.x) out[i] = 0.f;
}

template <class T>
void rms_norm_backward(const NormBackwardJob& j, float* workspace, cudaStream_t s) {
    const NormBackwardSplit d = norm_backward_split(j.rows, j.cols, j.period, j.dresidual != nullptr);
    float* const r_parts = workspace + (uint64_t)d.ctas * j.cols;
    auto go = [&](auto kernel, uint32_t threads) {
        launch_after(kernel, d.ctas, threads, 0, s, j, d.parts, workspace, r_parts, rows_aligned<T>(j.dy, j.dy_ld), rows_aligned<T>(j.h, j.h_ld),
                     (reinterpret_cast<uintptr_t>(j.weight) & 15u) == 0, rows_aligned<T>(j.dsum, j.dsum_ld), rows_aligned<T>(j.dx, j.dx_ld));
    };
    const uint32_t vecs = (j.cols + 7) / 8;
    if (vecs <= 32) go(k_rms_norm_backward<T, 1, 32, 256>, 256);
    else if (vecs <= 64) go(k_rms_norm_backward<T, 2, 32, 256>, 256);
    else if (vecs <= 96) go(k_rms_norm_backward<T, 3, 32, 256>, 256);
    else if (vecs <= 128) go(k_rms_norm_backward<T, 4, 32, 256>, 256);
    else if (vecs <= 160) go(k_rms_norm_backward<T, 5, 32, 256>, 256);
    else if (vecs <= 256) go(k_rms_norm_backward<T, 2, 128, 256>, 256);
    else if (vecs <= 512) go(k_rms_norm_backward<T, 4, 128, 256>, 256);
    else if (vecs <= 1024) go(k_rms_norm_backward<T, 2, 512, 512>, 512);
    else go(k_rms_norm_backward<T, 4, 512, 512>, 512);
    auto add_up = [&](const float* parts, uint32_t count, uint64_t n, float* out) {
        launch_after(k_sum_parts, grid_for(n, 32, 8), 256, 0, s, parts, count, n, out);
    };
    if (j.dweight) add_up(workspace, d.ctas, j.cols, j.dweight);
    if (j.dresidual && d.parts > 1) add_up(r_parts, d.parts, j.period * j.cols, j.dresidual);
}

// ---- dropout -------------------------------------------------------------------------------------------------------------------
// Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; 2011)
__device__ __forceinline__ uint4 philox(uint64_t counter, uint64_t seed) {
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = 0, c3 = 0, k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t u = (uint64_t)c0 * 0xD2511F53u, v = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(v >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)v;
        c2 = (uint32_t)(u >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)u;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}
// 16 bits for each of the eight indices from `index` on, two to a word
__device__ __forceinline__ void bits_of_8(uint64_t index, uint64_t seed, uint32_t bits[4]) {
    const uint4 a = philox(index >> 3, seed);
    bits[0] = a.x; bits[1] = a.y; bits[2] = a.z; bits[3] = a.w;
    const uint32_t skip = (uint32_t)index & 7u;
    if (skip) {  // the same for all threads of a launch whose rows are multiples of eight long
        const uint4 b = philox((index >> 3) + 1, seed);
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t lo = 0, hi = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if ((skip >> 1) == (uint32_t)k) { lo = w[i + k]; hi = w[i + k + 1]; }
            bits[i] = skip & 1u ? lo >> 16 | hi << 16 : lo;
        }
    }
}

template <class T>
__global__ void __launch_bounds__(kRowThreads) k_dropout(const DropoutJob a, uint64_t nvec, uint64_t per_row, float scale, bool x_whole, bool y_whole) {
    let_next_start();
    wait_for_previous();
    const T* const x = from_previous(reinterpret_cast<const T*>(a.x));
    T* const y = reinterpret_cast<T*>(a.y);
    for (uint64_t i = (uint64_t)blockIdx.x * kRowThreads + threadIdx.x; i < nvec; i += (uint64_t)gridDim.x * kRowThreads) {
        const uint64_t row = i / per_row, col = (i - row * per_row) * 8;
        const uint32_t valid = (uint32_t)min((uint64_t)8, a.cols - col);
        float v[8];
        load8(x + row * a.x_ld + col, valid, x_whole, v);
        uint32_t bits[4];
        if (a.per_row) {
            bits_of_8(a.offset + row, a.seed, bits);
            bits[0] = bits[1] = bits[2] = bits[3] = (bits[0] & 0xFFFFu) * 0x10001u;
        } else {
            bits_of_8(a.offset + row * a.cols + col, a.seed, bits);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t b = j & 1 ? bits[j >> 1] >> 16 : bits[j >> 1] & 0xFFFFu;
            v[j] = b >= a.threshold ? v[j] * scale : 0.f;
        }
        store8(y + row * a.y_ld + col, valid, y_whole, v);
    }
}

template <class T>
void dropout(DropoutJob j, cudaStream_t s) {
    if (!j.per_row && (j.rows == 1 || (j.x_ld == j.cols && j.y_ld == j.cols))) {  // one long row
        j.cols *= j.rows;
        j.x_ld = j.y_ld = (j.cols + 7) / 8 * 8;
        j.rows = 1;
    }
    const uint64_t per_row = (j.cols + 7) / 8, n = j.rows * per_row;
    launch_after(k_dropout<T>, grid_for(n, kRowThreads, 32), kRowThreads, 0, s, j, n, per_row, 65536.f / (float)(65536u - j.threshold),
                 rows_aligned<T>(j.x, j.x_ld), rows_aligned<T>(j.y, j.y_ld));
}

}  // namespace

void launch_patch_rows(const PatchJob& j, const dg_rows8* out8, const dg_matrix* out, cudaStream_t s) {
    switch (j.channels) {
        case 1: return patch_rows<1>(j, out8, out, s);
        case 2: return patch_rows<2>(j, out8, out, s);
        case 3: return patch_rows<3>(j, out8, out, s);
        default: return patch_rows<4>(j, out8, out, s);
    }
}

void launch_quantize_rows(const dg_matrix& src, const dg_rows8& out, cudaStream_t s) {
    if (src.dtype == DG_F32) quantize_rows<float>(src, out, s);
    else if (src.dtype == DG_BF16) quantize_rows<bf16>(src, out, s);
    else quantize_rows<__half>(src, out, s);
}

void launch_rms_norm(const NormJob& j, cudaStream_t s) {
    if (j.dtype == DG_F32) rms_norm<float>(j, s);
    else if (j.dtype == DG_BF16) rms_norm<bf16>(j, s);
    else rms_norm<__half>(j, s);
}

void launch_rms_norm_backward(const NormBackwardJob& j, float* workspace, cudaStream_t s) {
    if (j.rows == 0) {
        if (j.dweight) launch_after(k_zero, grid_for(j.cols, 256, 1), 256, 0, s, j.dweight, (uint64_t)j.cols);
        if (j.dresidual) launch_after(k_zero, grid_for(j.period * j.cols, 256, 4), 256, 0, s, j.dresidual, j.period * j.cols);
        return;
    }
    if (j.dtype == DG_F32) rms_norm_backward<float>(j, workspace, s);
    else if (j.dtype == DG_BF16) rms_norm_backward<bf16>(j, workspace, s);
    else rms_norm_backward<__half>(j, workspace, s);
}

void launch_dropout(const DropoutJob& j, cudaStream_t s) {
    if (j.dtype == DG_F32) dropout<float>(j, s);
    else if (j.dtype == DG_BF16) dropout<bf16>(j, s);
    else dropout<__half>(j, s);
}

}  // namespace dg
