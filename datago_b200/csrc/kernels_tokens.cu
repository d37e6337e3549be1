// Token rows: patches and matrices as 8-bit rows, the norm after the positions have been added, dropout.
//
// All of these read their inputs once and write their outputs once; memory bounds them (a plain copy moves 6.55 TB/s, a plain fill writes
// 3.8).  A thread owns vectors of eight neighbouring columns (16 bytes of bf16), so that sixteen neighbouring lanes hold the 128
// columns that share a scale: the group's largest magnitude is four shuffles, and nothing between the load and the store leaves the registers.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
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

// Eight 16-bit elements that start at an element: by words where they start at one, else by the half word before and behind three words.
template <class T> __device__ __forceinline__ uint4 load_any(const T* p) {
    if ((reinterpret_cast<uintptr_t>(p) & 2u) == 0) {
        const uint32_t* const w = reinterpret_cast<const uint32_t*>(p);
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    const uint16_t* const h = reinterpret_cast<const uint16_t*>(p);
    const uint32_t* const w = reinterpret_cast<const uint32_t*>(h + 1);
    const uint32_t first = h[0], a = w[0], b = w[1], c = w[2], last = h[7];
    return make_uint4(first | a << 16, a >> 16 | b << 16, b >> 16 | c << 16, c >> 16 | last << 16);
}
template <class T> __device__ __forceinline__ void store_any(T* p, const uint4& v) {
    if ((reinterpret_cast<uintptr_t>(p) & 2u) == 0) {
        uint32_t* const w = reinterpret_cast<uint32_t*>(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        return;
    }
    uint16_t* const h = reinterpret_cast<uint16_t*>(p);
    uint32_t* const w = reinterpret_cast<uint32_t*>(h + 1);
    h[0] = (uint16_t)v.x;
    w[0] = v.x >> 16 | v.y << 16;
    w[1] = v.y >> 16 | v.z << 16;
    w[2] = v.z >> 16 | v.w << 16;
    h[7] = (uint16_t)(v.w >> 16);
}
// Up to eight elements from p on (`valid` of them; the others are 0).  whole: p is 16-byte aligned.  Plain loads: what an earlier
// kernel wrote is read.
template <class T>
__device__ __forceinline__ void load8(const T* p, uint32_t valid, bool whole, float v[8]) {
    if constexpr (sizeof(T) == 2) {
        if (valid >= 8) {
            unpack8(whole ? *reinterpret_cast<const uint4*>(p) : load_any(p), v, T());
            return;
        }
    } else if (whole && valid >= 8) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        return;
    }
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) v[j] = j < valid ? widen(p[j]) : 0.f;
}
template <class T>
__device__ __forceinline__ void store8(T* p, uint32_t valid, bool whole, const float v[8]) {
    if constexpr (sizeof(T) == 2) {
        if (valid >= 8) {
            const uint4 q = make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
            if (whole) *reinterpret_cast<uint4*>(p) = q;
            else store_any(p, q);
            return;
        }
    } else if (whole && valid >= 8) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
        return;
    }
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j)
        if (j < valid) p[j] = narrow<T>(v[j]);
}
__device__ __forceinline__ void load8_any(const void* p, uint64_t at, int32_t dtype, uint32_t valid, bool whole, float v[8]) {
    if (dtype == DG_F32) load8(reinterpret_cast<const float*>(p) + at, valid, whole, v);
    else if (dtype == DG_BF16) load8(reinterpret_cast<const bf16*>(p) + at, valid, whole, v);
    else load8(reinterpret_cast<const __half*>(p) + at, valid, whole, v);
}
template <class T> bool rows_aligned(const void* p, uint64_t ld) { return ((reinterpret_cast<uintptr_t>(p) | (ld * sizeof(T))) & 15u) == 0; }

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
    __device__ __forceinline__ void load_whole(const T* p, bool there) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = there ? reinterpret_cast<const uint4*>(p)[i] : make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void load(const T* p, uint32_t valid, bool whole) {
        if (whole && valid >= 8) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
        } else if (sizeof(T) == 2 && valid >= 8) {
            w[0] = load_any(p);
        } else {
            T e[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) e[j] = j < valid ? p[j] : narrow<T>(0.f);
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(e)[i];
        }
    }
};

// ---- two floats at a time ------------------------------------------------------------------------------------------------
// The 32-bit units multiply and add pairs (fma.rn.f32x2): these kernels issue as many instructions as the chip can while memory is busy.
typedef unsigned long long Pair;
__device__ __forceinline__ Pair pair_of(float lo, float hi) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi));
    return p;
}
__device__ __forceinline__ void parts_of(Pair p, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p)); }
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
// max(top, |lo|, |hi|); NaN as soon as one of them is
__device__ __forceinline__ float larger2(float top, Pair p) {
    float lo, hi, d;
    parts_of(p, lo, hi);
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(top), "f"(lo), "f"(hi));
    return d;
}
template <class T> __device__ __forceinline__ void pairs_of(const Raw8<T>& x, Pair p[4]) {
    float v[8];
    x.widen(v);
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = pair_of(v[2 * i], v[2 * i + 1]);
}
__device__ __forceinline__ void floats_of(const Pair p[4], float v[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) parts_of(p[i], v[2 * i], v[2 * i + 1]);
}

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
__device__ __forceinline__ uint32_t e4m3x4(Pair a, Pair b) {
    float v[4];
    parts_of(a, v[0], v[1]);
    parts_of(b, v[2], v[3]);
    return e4m3x4(v[0], v[1], v[2], v[3]);
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

constexpr uint32_t kRowThreads = 256;

uint32_t grid_for(uint64_t items, uint32_t per_cta, uint32_t ctas_per_sm) {
    return (uint32_t)std::min<uint64_t>((items + per_cta - 1) / per_cta, (uint64_t)kSms * ctas_per_sm);
}

// Division of n < 2^31 by a number that is the same for a whole launch: with 2^s >= d, n / d = n * ceil(2^(31 + s) / d) / 2^(31 + s) rounded down,
// because the ceiling is off by less than n / 2^(31 + s) < 1 / d.
struct Divisor {
    uint32_t d, factor, shift;
    explicit Divisor(uint32_t by) : d(by), factor(0), shift(31) {
        while ((1ull << (shift - 31)) < by) ++shift;
        factor = (uint32_t)(((1ull << shift) + by - 1) / by);
    }
    __device__ __forceinline__ uint32_t of(uint32_t n, uint32_t& rest) const {
        const uint32_t q = (uint32_t)((uint64_t)n * factor >> shift);
        rest = n - q * d;
        return q;
    }
};
constexpr uint64_t kMostItems = 1ull << 30;  // threads' worth of work of a launch; more rows go to further launches

// ---- rows of a matrix --------------------------------------------------------------------------------------------------
// 30000 x 1000 bf16: 19 us, 4.8 TB/s.
// Sixteen lanes per group of 128 columns, eight elements each; two groups of a half-warp under way.
template <class T>
__global__ void __launch_bounds__(kRowThreads) k_rows8(const T* src, uint64_t src_ld, bool whole, uint32_t items, Divisor per_row, uint32_t cols, uint8_t* values, uint64_t ld,
                                                       uint8_t* scales, uint64_t scale_ld) {
    let_next_start();
    wait_for_previous();
    src = from_previous(src);
    constexpr uint32_t kVecs = 2;
    // items are a multiple of 16 and steps of 32: the lanes of a half-warp stay together, and the shuffles have whole warps
    for (uint32_t i0 = blockIdx.x * kRowThreads * kVecs + threadIdx.x; (i0 & ~31u) < items; i0 += gridDim.x * kRowThreads * kVecs) {
        uint32_t row[kVecs], col[kVecs], valid[kVecs];
        Raw8<T> x[kVecs];
#pragma unroll
        for (uint32_t k = 0; k < kVecs; ++k) {
            const uint32_t i = i0 + k * kRowThreads;
            row[k] = per_row.of(i, col[k]);
            col[k] *= 8;
            valid[k] = i < items && col[k] < cols ? min(8u, cols - col[k]) : 0;
            x[k].load(src + row[k] * src_ld + col[k], valid[k], whole);
        }
#pragma unroll
        for (uint32_t k = 0; k < kVecs; ++k) {
            float v[8];
            x[k].widen(v);
            const uint32_t e = scale_byte(largest_of_16_lanes(largest8(v)));
            if (valid[k]) {
                store_values8(values + row[k] * ld + col[k], valid[k], quantize8(v, inverse_scale(e)));
                if ((threadIdx.x & 15u) == 0) scales[row[k] * scale_ld + col[k] / kScaleGroup] = (uint8_t)e;
            }
        }
    }
}

template <class T>
void rows8(const dg_matrix& m, const dg_rows8& out, cudaStream_t s) {
    const uint64_t per_row = scale_groups(m.cols) * 16, most = std::max<uint64_t>(1, kMostItems / per_row);
    for (uint64_t r = 0; r < m.rows; r += most) {
        const uint32_t items = (uint32_t)(std::min(most, m.rows - r) * per_row);
        launch_after(k_rows8<T>, grid_for(items, kRowThreads * 2, 32), kRowThreads, 0, s, (const T*)m.data + r * m.ld, m.ld, rows_aligned<T>(m.data, m.ld), items,
                     Divisor((uint32_t)per_row), (uint32_t)m.cols, out.values + r * out.ld, out.ld, out.scales + r * out.scale_ld, out.scale_ld);
    }
}

// ---- patches ---------------------------------------------------------------------------------------------------------------
// A thread makes sixteen neighbouring features of a patch, eight lanes the 128 of a scale.  A patch's row of pixels is `segment` = patch * C
// neighbouring bytes, of which features 16 k .. 16 k + 15 are sixteen neighbouring ones where the segment is a multiple of sixteen.  48 images of
// 1152 x 896 x 3 in patches of 16: 60 to 64 us, 4.7 to 5.0 TB/s; instructions bound it, 74 % of the places to issue one (eight features a thread and a division each took 206 us, one patch a
// thread 76).
// Out: uint8_t for 8-bit rows, else the type of the matrix.
template <int C> struct PatchView {
    const uint8_t* pixels;
    uint64_t pitch, image;  // bytes of a row of pixels and of an image
    uint32_t patch, segment, cols, grid_w;
    float gain[C], shift[C];
};
template <class Out> struct PatchOut {
    Out* data;
    uint64_t ld;
    uint8_t* scales;
    uint64_t scale_ld;
    bool whole;
};

// Gains and shifts of neighbouring features, two at a time, the first of them of channel `phase`.
template <int C> struct Coefficients {
    static constexpr int kPairs = C % 2 ? C : C / 2;  // after so many pairs they repeat
    Pair gain[kPairs], shift[kPairs];
    __device__ __forceinline__ Coefficients(const PatchView<C>& in, uint32_t phase) {
        float g[C], b[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            g[c] = in.gain[c];
            b[c] = in.shift[c];
#pragma unroll
            for (int k = 1; k < C; ++k)
                if (phase == (uint32_t)k) { g[c] = in.gain[(c + k) % C]; b[c] = in.shift[(c + k) % C]; }
        }
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
            gain[j] = pair_of(g[2 * j % C], g[(2 * j + 1) % C]);
            shift[j] = pair_of(b[2 * j % C], b[(2 * j + 1) % C]);
        }
    }
    // pixel bytes, four to a word, to values.  2^23 + pixel, as a float, has the pixel in its low byte.
    __device__ __forceinline__ void normalise(const uint32_t w[4], Pair v[8]) const {
        const Pair less = pair_of(-8388608.f, -8388608.f);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t word = w[j >> 1], at = 2 * (j & 1);
            const Pair u = pair_of(__uint_as_float(__byte_perm(word, 0x4B000000u, 0x7650 + at)), __uint_as_float(__byte_perm(word, 0x4B000000u, 0x7651 + at)));
            v[j] = fma2(add2(u, less), gain[j % kPairs], shift[j % kPairs]);
        }
    }
};

// Sixteen features of a row from `col` on, `valid` of them; all lanes of a warp are here.
template <class Out>
__device__ __forceinline__ void store16(const PatchOut<Out>& out, uint64_t row, uint32_t col, uint32_t valid, Pair v[8]) {
    if constexpr (sizeof(Out) == 1) {
        if (valid < 16) {  // what is not there has no part in the scale
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                float lo, hi;
                parts_of(v[j], lo, hi);
                v[j] = pair_of(valid > 2 * j ? lo : 0.f, valid > 2 * j + 1 ? hi : 0.f);
            }
        }
        float largest = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) largest = larger2(largest, v[j]);
        uint32_t top = magnitude(largest);
#pragma unroll
        for (int d = 4; d; d >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
        const uint32_t e = scale_byte(top);
        const float inverse = inverse_scale(e);
        if (!valid) return;
        uint8_t* const p = out.data + row * out.ld + col;
        const Pair by = pair_of(inverse, inverse);
        uint32_t q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = e4m3x4(mul2(v[2 * j], by), mul2(v[2 * j + 1], by));
        if (valid >= 16) *reinterpret_cast<uint4*>(p) = make_uint4(q[0], q[1], q[2], q[3]);
        else
#pragma unroll
            for (uint32_t j = 0; j < 16; ++j)
                if (j < valid) p[j] = (uint8_t)(q[j >> 2] >> (8 * (j & 3)));
        if ((threadIdx.x & 7u) == 0) out.scales[row * out.scale_ld + col / kScaleGroup] = (uint8_t)e;
    } else {
        Out* const p = out.data + row * out.ld + col;
        float f[16];
        floats_of(v, f);
        floats_of(v + 4, f + 8);
        store8(p, valid, out.whole, f);
        if (valid > 8) store8(p + 8, valid - 8, out.whole, f + 8);
    }
}

constexpr uint32_t kAcross = 4;  // neighbouring patches whose features from `col` on a thread makes: their places and coefficients are found once
template <int C, class Out>
__global__ void __launch_bounds__(kRowThreads) k_patches(const PatchView<C> in, const PatchOut<Out> out, uint32_t items, Divisor per_row, Divisor sets, Divisor grid_h, Divisor segment) {
    let_next_start();
    wait_for_previous();
    const uint8_t* const pixels = from_previous(in.pixels);
    for (uint32_t i0 = blockIdx.x * kRowThreads + threadIdx.x; (i0 & ~31u) < items; i0 += gridDim.x * kRowThreads) {
        uint32_t col, set, Y, b;
        const uint32_t band = sets.of(per_row.of(i0, col), set), i = grid_h.of(band, Y), x0 = set * kAcross;
        col *= 16;
        const uint32_t y = segment.of(col, b);
        const uint32_t count = i0 < items && col < in.cols ? min(kAcross, in.grid_w - x0) : 0;
        const uint8_t* const from = pixels + i * in.image + ((uint64_t)Y * in.patch + y) * in.pitch + (uint64_t)x0 * in.segment + b;
        uint4 w[kAcross];
#pragma unroll
        for (uint32_t k = 0; k < kAcross; ++k) w[k] = k < count ? *reinterpret_cast<const uint4*>(from + k * in.segment) : make_uint4(0, 0, 0, 0);
        const Coefficients<C> by(in, C == 3 ? col % 3 : 0);  // 16 is a multiple of 1, 2 and 4
        const uint64_t row = (uint64_t)band * in.grid_w + x0;
#pragma unroll
        for (uint32_t k = 0; k < kAcross; ++k) {
            const uint32_t words[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
            Pair v[8];
            by.normalise(words, v);
            store16(out, row + k, col, k < count ? 16 : 0, v);
        }
    }
}

// Segments that are no multiple of sixteen bytes, or do not start at one: a CTA brings its patches' rows of pixels (up to `across` patches of a row of
// patches) into shared memory first, word by word where the bytes begin at words, and gathers the features from there.  24 images of 980 x 700 x 3
// in patches of 14: 82 us, 1.2 TB/s, bound by instructions.
constexpr uint32_t kStripBytes = 40 * 1024;
__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// from any place in shared memory; up to three bytes on either side are read too
__device__ __forceinline__ void sixteen_bytes(uint32_t at, uint32_t w[4]) {
    uint32_t v[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[i]) : "r"((at & ~3u) + 4 * i));
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(v[i], v[i + 1], 8 * (at & 3u));
}

template <int C, class Out>
__global__ void __launch_bounds__(kRowThreads) k_patches_staged(const PatchView<C> in, const PatchOut<Out> out, uint32_t across, Divisor strips_x, Divisor grid_h, uint32_t strips,
                                                                uint32_t strip_pitch, Divisor per_patch, Divisor segment) {
    extern __shared__ __align__(16) uint8_t s_strip[];
    let_next_start();
    wait_for_previous();
    const uint8_t* const pixels = from_previous(in.pixels);
    for (uint32_t strip = blockIdx.x; strip < strips; strip += gridDim.x) {
        uint32_t sx, Y;
        const uint32_t band = strips_x.of(strip, sx), i = grid_h.of(band, Y), x0 = sx * across, count = min(across, in.grid_w - x0), bytes = count * in.segment;
        const uint8_t* const from = pixels + i * in.image + (uint64_t)Y * in.patch * in.pitch + (uint64_t)x0 * in.segment;
        __syncthreads();  // the strip before this one has been read
        for (uint32_t y = threadIdx.x >> 5; y < in.patch; y += kRowThreads / 32) {  // a warp per row of pixels
            const uint8_t* const p = from + y * in.pitch;
            const uint32_t lead = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 3u), lane = threadIdx.x & 31u;
            uint8_t* const to = s_strip + y * strip_pitch + lead;  // words to words
            const uint32_t head = min(bytes, (4 - lead) & 3u), words = (bytes - head) >> 2;
            for (uint32_t k = lane; k < words; k += 32) *reinterpret_cast<uint32_t*>(to + head + 4 * k) = *reinterpret_cast<const uint32_t*>(p + head + 4 * k);
            if (lane < head) to[lane] = p[lane];
            if (lane < bytes - head - 4 * words) to[head + 4 * words + lane] = p[head + 4 * words + lane];
        }
        __syncthreads();
        const uint32_t items = count * per_patch.d;
        for (uint32_t k = threadIdx.x; (k & ~31u) < items; k += kRowThreads) {
            uint32_t col, b, w[4] = {};
            const uint32_t x = per_patch.of(k, col);
            col *= 16;
            const uint32_t valid = k < items && col < in.cols ? min(16u, in.cols - col) : 0;
            uint32_t y = segment.of(col, b);
            auto line = [&] { return s_strip + y * strip_pitch + (uint32_t)((reinterpret_cast<uintptr_t>(from) + y * in.pitch) & 3u) + x * in.segment; };
            if (valid && in.segment >= 16) {
                // sixteen bytes cross into the next row of pixels once at most: `here` of them are of this one, and the next one's are read from
                // as far before its start as puts them behind those
                const uint32_t here = min(16u, in.segment - b);
                sixteen_bytes(shared_address(line() + b), w);
                if (here < valid) {
                    uint32_t next[4];
                    ++y;
                    sixteen_bytes(shared_address(line()) - here, next);
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        const uint32_t mine = here >= 4 * j + 4 ? ~0u : here <= 4 * j ? 0u : (1u << (8 * (here - 4 * j))) - 1;
                        w[j] = (w[j] & mine) | (next[j] & ~mine);
                    }
                }
            } else if (valid) {
                const uint8_t* q = line();
#pragma unroll
                for (uint32_t j = 0; j < 16; ++j) {
                    if (j < valid) w[j >> 2] |= (uint32_t)q[b] << (8 * (j & 3));
                    if (++b == in.segment && j + 1 < valid) { b = 0; ++y; q = line(); }
                }
            }
            Pair v[8];
            Coefficients<C>(in, col % C).normalise(w, v);
            store16(out, (uint64_t)band * in.grid_w + x0 + x, col, valid, v);
        }
    }
}

template <int C, class Out>
void patches(const PatchJob& j, PatchOut<Out> out, cudaStream_t s) {
    PatchView<C> in;
    in.pixels = j.pixels;
    in.pitch = (uint64_t)j.w * C;
    in.image = in.pitch * j.h;
    in.patch = j.patch;
    in.segment = j.patch * C;
    in.cols = j.patch * in.segment;
    in.grid_w = j.w / j.patch;
    for (int c = 0; c < C; ++c) { in.gain[c] = j.gain[c]; in.shift[c] = j.shift[c]; }
    const uint32_t grid_h = j.h / j.patch, per_row = (in.cols + kScaleGroup - 1) / kScaleGroup * 8;
    const uint64_t per_image = (uint64_t)in.grid_w * grid_h;
    const bool straight = ((reinterpret_cast<uintptr_t>(j.pixels) | in.pitch | in.segment) & 15u) == 0;
    const uint32_t most = (uint32_t)std::max<uint64_t>(1, kMostItems / (per_image * per_row));  // images of a launch
    for (uint32_t i = 0; i < j.n; i += most) {
        const uint32_t n = std::min(most, j.n - i);
        PatchOut<Out> to = out;
        in.pixels = j.pixels + i * in.image;
        to.data += i * per_image * out.ld;
        if (sizeof(Out) == 1) to.scales += i * per_image * out.scale_ld;
        if (straight) {
            const uint32_t sets = (in.grid_w + kAcross - 1) / kAcross, items = n * grid_h * sets * per_row;
            launch_after(k_patches<C, Out>, grid_for(items, kRowThreads, 32), kRowThreads, 0, s, in, to, items, Divisor(per_row), Divisor(sets), Divisor(grid_h), Divisor(in.segment));
        } else {
            // patches of a strip: what the shared memory holds, but no more than spreads the work over the chip
            const uint32_t bands = n * grid_h, wanted = (uint32_t)std::max<uint64_t>(1, (uint64_t)bands * in.grid_w / (kSms * 8));
            const uint32_t most_across = std::max(1u, std::min({in.grid_w, (kStripBytes / j.patch - 8) / in.segment, std::max(wanted, 8u)}));
            const uint32_t strips_x = (in.grid_w + most_across - 1) / most_across, across = (in.grid_w + strips_x - 1) / strips_x;
            const uint32_t pitch = (across * in.segment + 3 + 7) / 4 * 4;
            launch_after(k_patches_staged<C, Out>, grid_for((uint64_t)bands * strips_x, 1, 16), kRowThreads, (size_t)pitch * j.patch + 24, s, in, to, across, Divisor(strips_x), Divisor(grid_h),
                         bands * strips_x, pitch, Divisor(per_row), Divisor(in.segment));
        }
    }
}

template <int C>
void patch_rows(const PatchJob& j, const dg_rows8* out8, const dg_matrix* out, cudaStream_t s) {
    if (out8) patches<C, uint8_t>(j, {out8->values, out8->ld, out8->scales, out8->scale_ld, true}, s);
    else if (out->dtype == DG_F32) patches<C, float>(j, {(float*)out->data, out->ld, nullptr, 0, rows_aligned<float>(out->data, out->ld)}, s);
    else if (out->dtype == DG_BF16) patches<C, bf16>(j, {(bf16*)out->data, out->ld, nullptr, 0, rows_aligned<bf16>(out->data, out->ld)}, s);
    else patches<C, __half>(j, {(__half*)out->data, out->ld, nullptr, 0, rows_aligned<__half>(out->data, out->ld)}, s);
}

// ---- scales along the rows of the source, and of 128 x 128 blocks -------------------------------------------------------------
// The transpose of a matrix stays in the order of the matrix (dg_rows8.by_column): only its scales run along the rows.  A CTA holds 128 x 128 elements
// as they were loaded, a thread eight rows of eight columns, and meets twice over its columns' maxima.
// 37003 x 1000 bf16: 23.5 us, 4.7 TB/s; each CTA waits for its loads once, and four of 64 registers a thread to an SM hide more of that than two of 128
// did (26).  Transposing the values through shared memory as well took 46.
constexpr uint32_t kColumnThreads = 256, kColumnTile = 128;
constexpr int kColumnRows = 8;  // of a thread

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
__global__ void __launch_bounds__(kColumnThreads, sizeof(T) == 4 ? 2 : 4) k_columns8(const T* src, uint64_t rows, uint64_t cols, uint64_t ld, bool whole, uint32_t tiles_x, uint64_t tiles,
                                                                                     uint8_t* values, uint64_t out_ld, uint8_t* scales, uint64_t scale_row, uint64_t scale_col) {
    constexpr int R = kColumnRows, kWarps = kColumnThreads / 32, kWords = sizeof(T) * 2;
    __shared__ __align__(16) uint32_t s_top[kWarps][16][kWords];
    __shared__ __align__(16) float s_inverse[kColumnTile];
    __shared__ uint32_t s_warp[kColumnTile / 32];
    let_next_start();
    wait_for_previous();
    src = from_previous(src);
    const uint32_t cv = threadIdx.x & 15u, warp = threadIdx.x >> 5, first = (threadIdx.x >> 4) * R;  // eight columns from 8 cv, R rows from `first`
    for (uint64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const uint64_t ty = tile / tiles_x, c0 = (tile - ty * tiles_x) * kColumnTile, col = c0 + 8 * cv, r0 = ty * 128 + first;
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
        for (int k = 0; k < kWords; ++k) top[k] = larger(top[k], __shfl_xor_sync(0xFFFFFFFFu, top[k], 16), T());  // the warp's other rows
        if ((threadIdx.x & 16u) == 0)
#pragma unroll
            for (int k = 0; k < kWords / 4; ++k) *reinterpret_cast<uint4*>(&s_top[warp][cv][4 * k]) = make_uint4(top[4 * k], top[4 * k + 1], top[4 * k + 2], top[4 * k + 3]);
        __syncthreads();
        if (threadIdx.x < kColumnTile) {  // a thread per column
            const uint32_t c = threadIdx.x;
            uint32_t m = 0;
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int w = 0; w < kWarps; ++w) m = max(m, s_top[w][c >> 3][c & 7u]);
            } else {
#pragma unroll
                for (int w = 0; w < kWarps; ++w) m = max(m, s_top[w][c >> 3][(c & 7u) >> 1] >> (16 * (c & 1u)) & 0xFFFFu);
                m = magnitude_of(m, T());
            }
            if constexpr (BLOCK) {
                m = __reduce_max_sync(0xFFFFFFFFu, m);
                if ((c & 31u) == 0) s_warp[warp] = m;
                asm volatile("bar.sync 1, 128;" ::: "memory");  // the threads that are here
                m = max(max(s_warp[0], s_warp[1]), max(s_warp[2], s_warp[3]));
                if (c == 0) scales[ty * scale_row + c0 / 128 * scale_col] = (uint8_t)scale_byte(m);
            } else if (c0 + c < cols) {
                scales[ty * scale_row + (c0 + c) * scale_col] = (uint8_t)scale_byte(m);
            }
            s_inverse[c] = inverse_scale(scale_byte(m));
        }
        __syncthreads();
        Pair inverse[4];
        {
            const ulonglong2 *const p = reinterpret_cast<const ulonglong2*>(&s_inverse[8 * cv]), lo = p[0], hi = p[1];
            inverse[0] = lo.x; inverse[1] = lo.y; inverse[2] = hi.x; inverse[3] = hi.y;
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (!valid || r0 + i >= rows) continue;
            Pair v[4];
            pairs_of(x[i], v);
            store_values8(values + (r0 + i) * out_ld + col, valid,
                          make_uint2(e4m3x4(mul2(v[0], inverse[0]), mul2(v[1], inverse[1])), e4m3x4(mul2(v[2], inverse[2]), mul2(v[3], inverse[3]))));
        }
    }
}

template <class T>
void quantize_rows(const dg_matrix& m, const dg_rows8& out, cudaStream_t s) {
    const bool whole = rows_aligned<T>(m.data, m.ld);
    if (!out.by_column && out.block == 1) {
        rows8<T>(m, out, s);
        return;
    }
    const uint32_t tiles_x = (uint32_t)((m.cols + kColumnTile - 1) / kColumnTile);
    const uint64_t tiles = scale_groups(m.rows) * tiles_x;
    auto go = [&](auto kernel) {
        launch_after(kernel, grid_for(tiles, 1, 32), kColumnThreads, 0, s, (const T*)m.data, m.rows, m.cols, m.ld, whole, tiles_x, tiles, out.values, out.ld,
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

// WHOLE: every row of every matrix starts at a multiple of 16 bytes and holds whole vectors.  The weight waits in shared memory as floats.
template <class T, int V, int TPR, int THREADS, bool WHOLE>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 2 : 1) k_rms_norm(const NormJob a, bool x_whole, bool r_whole, bool s_whole, bool y_whole) {
    extern __shared__ __align__(16) float s_weight[];
    __shared__ float s_part[THREADS / 32];
    let_next_start();
    wait_for_previous();
    const T *const px = from_previous(reinterpret_cast<const T*>(a.x)), *const pr = from_previous(reinterpret_cast<const T*>(a.residual));
    if (a.weight) {
        const void* const pw = from_previous(a.weight);
        for (uint32_t c = threadIdx.x; c < a.cols; c += THREADS)
            s_weight[c] = a.weight_dtype == DG_F32 ? reinterpret_cast<const float*>(pw)[c] : a.weight_dtype == DG_BF16 ? widen(reinterpret_cast<const bf16*>(pw)[c]) : widen(reinterpret_cast<const __half*>(pw)[c]);
        for (uint32_t c = a.cols + threadIdx.x; c < (a.cols + 7) / 8 * 8; c += THREADS) s_weight[c] = 0.f;
        __syncthreads();
    }
    constexpr uint32_t kRows = THREADS / TPR;
    const uint32_t t = threadIdx.x % TPR, mine = threadIdx.x / TPR;
    const float per_col = 1.f / (float)a.cols;
    // valid elements of vector k of a row
    auto valid_at = [&](int k) {
        const uint32_t col = (k * TPR + t) * 8;
        return col >= a.cols ? 0u : WHOLE ? 8u : min(8u, a.cols - col);
    };
    const uint64_t stride = (uint64_t)gridDim.x * kRows;
    uint64_t row = (uint64_t)blockIdx.x * kRows + mine, rr = pr ? row % a.residual_rows : 0;
    const uint64_t rr_step = pr ? stride % a.residual_rows : 0;
    // the next row is under way while this one is worked on
    Raw8<T> x[V], r[V];
    auto fetch = [&](uint64_t at, uint64_t residual_row) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const T* const p = px + at * a.x_ld + (k * TPR + t) * 8;
            if constexpr (WHOLE) x[k].load_whole(p, at < a.rows && valid_at(k));
            else x[k].load(p, at < a.rows ? valid_at(k) : 0, x_whole);
        }
        if (!pr) return;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const T* const p = pr + residual_row * a.residual_ld + (k * TPR + t) * 8;
            if constexpr (WHOLE) r[k].load_whole(p, at < a.rows && valid_at(k));
            else r[k].load(p, at < a.rows ? valid_at(k) : 0, r_whole);
        }
    };
    fetch(row, rr);
    for (uint64_t r0 = (uint64_t)blockIdx.x * kRows; r0 < a.rows; r0 += stride, row += stride) {
        const bool live = row < a.rows;
        Pair h[V][4];
        Pair sums = pair_of(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            pairs_of(x[k], h[k]);
            if (pr) {
                Pair v[4];
                pairs_of(r[k], v);
#pragma unroll
                for (int j = 0; j < 4; ++j) h[k][j] = add2(h[k][j], v[j]);
            }
        }
        rr += rr_step;
        if (rr >= a.residual_rows) rr -= a.residual_rows;
        fetch(row + stride, rr);
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) sums = fma2(h[k][j], h[k][j], sums);
        float even, odd;
        parts_of(sums, even, odd);
        const float rstd = 1.f / sqrtf(row_sum<TPR>(even + odd, s_part) * per_col + a.eps);
        if (live && t == 0 && a.rstd) a.rstd[row] = rstd;
        if (a.sum) {
            T* const to = reinterpret_cast<T*>(a.sum) + row * a.sum_ld;
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (live && valid_at(k)) {
                    float v[8];
                    floats_of(h[k], v);
                    store8(to + (k * TPR + t) * 8, valid_at(k), WHOLE || s_whole, v);
                }
        }
        const Pair rstds = pair_of(rstd, rstd);
#pragma unroll
        for (int k = 0; k < V; ++k) {
#pragma unroll
            for (int j = 0; j < 4; ++j) h[k][j] = mul2(h[k][j], rstds);
            if (a.weight) {  // (the floats behind the last column are zeros)
                const ulonglong2 *const w = reinterpret_cast<const ulonglong2*>(s_weight + (valid_at(k) ? (k * TPR + t) * 8 : 0)), lo = w[0], hi = w[1];
                h[k][0] = mul2(h[k][0], lo.x);
                h[k][1] = mul2(h[k][1], lo.y);
                h[k][2] = mul2(h[k][2], hi.x);
                h[k][3] = mul2(h[k][3], hi.y);
            }
        }
        if (a.y) {
            T* const to = reinterpret_cast<T*>(a.y) + row * a.y_ld;
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (live && valid_at(k)) {
                    float v[8];
                    floats_of(h[k], v);
                    store8(to + (k * TPR + t) * 8, valid_at(k), WHOLE || y_whole, v);
                }
        }
        if (a.y8.values) {
            uint8_t *const to = a.y8.values + row * a.y8.ld, *const scales = a.y8.scales + row * a.y8.scale_ld;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                float top = 0.f;
                if (valid_at(k)) {  // lanes behind the last column have no part in a scale
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (!WHOLE && valid_at(k) < 8) {  // nor have elements
                            float lo, hi;
                            parts_of(h[k][j], lo, hi);
                            h[k][j] = pair_of(valid_at(k) > 2u * j ? lo : 0.f, valid_at(k) > 2u * j + 1 ? hi : 0.f);
                        }
                        top = larger2(top, h[k][j]);
                    }
                }
                const uint32_t e = scale_byte(largest_of_16_lanes(magnitude(top)));
                if (live && valid_at(k)) {
                    const float inverse = inverse_scale(e);
                    const Pair by = pair_of(inverse, inverse);
                    store_values8(to + (k * TPR + t) * 8, valid_at(k), make_uint2(e4m3x4(mul2(h[k][0], by), mul2(h[k][1], by)), e4m3x4(mul2(h[k][2], by), mul2(h[k][3], by))));
                    if ((t & 15u) == 0) scales[(k * TPR + t) / 16] = (uint8_t)e;
                }
            }
        }
    }
}

// ---- rows through shared memory -------------------------------------------------------------------------------------------
// Rows of 16-bit elements that start at multiples of 16 bytes, up to 1280 of them: a warp per row, whose next row is copied into shared memory while it
// works on this one (cp.async, sixteen bytes a lane; a lane reads what it has copied itself, so nothing but its own copies is waited for).  What is
// under way then costs no registers, and half as many warps again fit as with rows waiting in registers.  131072 x 1152 bf16 with positions, sum and 8-bit
// output: 135 to 145 us, 5.3 to 5.7 TB/s, six tenths of it writes (159 with the next row in registers; rows shared by five warps, which meet at a barrier,
// took 224 and more).
constexpr uint32_t kStagedCols = 1280;
__device__ __forceinline__ void copy16(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void end_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void await_all_copies_but_last() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }
template <class T> __device__ __forceinline__ void staged_pairs(const T* at, Pair p[4]) {
    Raw8<T> x;
    x.w[0] = *reinterpret_cast<const uint4*>(at);
    pairs_of(x, p);
}
// the weight as floats at the start of the dynamic shared memory
__device__ __forceinline__ void stage_weight(float* to, const void* weight, int32_t dtype, uint32_t cols) {
    for (uint32_t c = threadIdx.x; c < cols; c += blockDim.x)
        to[c] = dtype == DG_F32 ? reinterpret_cast<const float*>(weight)[c] : dtype == DG_BF16 ? widen(reinterpret_cast<const bf16*>(weight)[c]) : widen(reinterpret_cast<const __half*>(weight)[c]);
    __syncthreads();
}
__device__ __forceinline__ void scale_pairs(Pair p[4], const float* w) {
    const ulonglong2 lo = reinterpret_cast<const ulonglong2*>(w)[0], hi = reinterpret_cast<const ulonglong2*>(w)[1];
    p[0] = mul2(p[0], lo.x);
    p[1] = mul2(p[1], lo.y);
    p[2] = mul2(p[2], hi.x);
    p[3] = mul2(p[3], hi.y);
}

constexpr uint32_t kStagedNormThreads = 384;
// The last of a lane's V vectors may lie behind the row.
template <class T, int V, bool RESIDUAL, bool WEIGHT>
__global__ void __launch_bounds__(kStagedNormThreads, 2) k_rms_norm_staged(const NormJob a) {
    extern __shared__ __align__(16) float s_staged[];
    let_next_start();
    wait_for_previous();
    if (WEIGHT) stage_weight(s_staged, from_previous(a.weight), a.weight_dtype, a.cols);
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, vecs = a.cols / 8, warps = blockDim.x / 32;
    const T *const px = from_previous(reinterpret_cast<const T*>(a.x)) + 8 * lane, *const pr = from_previous(reinterpret_cast<const T*>(a.residual)) + 8 * lane;
    constexpr uint32_t kRows = RESIDUAL ? 2 : 1;  // rows of a stage
    T* const ring = reinterpret_cast<T*>(s_staged + (WEIGHT ? a.cols : 0)) + (size_t)warp * 2 * kRows * a.cols + 8 * lane;
    const float* const weight = s_staged + 8 * lane;
    const bool last = lane + 32 * (V - 1) < vecs;
    const float per_col = 1.f / (float)a.cols;
    const uint64_t stride = (uint64_t)gridDim.x * warps;
    uint64_t row = (uint64_t)blockIdx.x * warps + warp, rr = RESIDUAL ? row % a.residual_rows : 0;
    const uint64_t rr_step = RESIDUAL ? stride % a.residual_rows : 0;
    auto fetch = [&](uint64_t at, uint32_t stage) {
        if (at < a.rows) {
            const uint32_t to = shared_address(ring + stage * kRows * a.cols);
            const T *const x = px + at * a.x_ld, *const r = pr + rr * a.residual_ld;
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (k + 1 < V || last) {
                    copy16(to + 512 * k, x + 256 * k);
                    if (RESIDUAL) copy16(to + 2 * a.cols + 512 * k, r + 256 * k);
                }
        }
        end_copies();
        if (RESIDUAL) {
            rr += rr_step;
            if (rr >= a.residual_rows) rr -= a.residual_rows;
        }
    };
    fetch(row, 0);
    for (uint32_t stage = 0; row < a.rows; row += stride, stage ^= 1u) {
        fetch(row + stride, stage ^ 1u);
        await_all_copies_but_last();
        const T* const from = ring + stage * kRows * a.cols;
        Pair h[V][4], sums = pair_of(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            if (k + 1 < V || last) {
                staged_pairs(from + 256 * k, h[k]);
                if (RESIDUAL) {
                    Pair r[4];
                    staged_pairs(from + a.cols + 256 * k, r);
#pragma unroll
                    for (int j = 0; j < 4; ++j) h[k][j] = add2(h[k][j], r[j]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) h[k][j] = pair_of(0.f, 0.f);
            }
        }
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) sums = fma2(h[k][j], h[k][j], sums);
        float even, odd;
        parts_of(sums, even, odd);
        float sum = even + odd;
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
        if (a.sum) {
            T* const to = reinterpret_cast<T*>(a.sum) + row * a.sum_ld + 8 * lane;
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (k + 1 < V || last) {
                    float f[8];
                    floats_of(h[k], f);
                    store8(to + 256 * k, 8, true, f);
                }
        }
        const float rstd = 1.f / sqrtf(sum * per_col + a.eps);
        if (lane == 0 && a.rstd) a.rstd[row] = rstd;
        const Pair rstds = pair_of(rstd, rstd);
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (k + 1 < V || last) {
#pragma unroll
                for (int j = 0; j < 4; ++j) h[k][j] = mul2(h[k][j], rstds);
                if (WEIGHT) scale_pairs(h[k], weight + 256 * k);
            }
        if (a.y) {
            T* const to = reinterpret_cast<T*>(a.y) + row * a.y_ld + 8 * lane;
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (k + 1 < V || last) {
                    float f[8];
                    floats_of(h[k], f);
                    store8(to + 256 * k, 8, true, f);
                }
        }
        if (a.y8.values) {
            uint32_t top[V];
#pragma unroll
            for (int k = 0; k < V; ++k) {
                float largest = 0.f;
                if (k + 1 < V || last) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) largest = larger2(largest, h[k][j]);
                }
                top[k] = magnitude(largest);
            }
#pragma unroll
            for (int d = 8; d; d >>= 1)
#pragma unroll
                for (int k = 0; k < V; ++k) top[k] = max(top[k], __shfl_xor_sync(0xFFFFFFFFu, top[k], d));
            uint8_t *const to = a.y8.values + row * a.y8.ld + 8 * lane, *const scales = a.y8.scales + row * a.y8.scale_ld + (lane >> 4);
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (k + 1 < V || last) {
                    const uint32_t e = scale_byte(top[k]);
                    const float inverse = inverse_scale(e);
                    const Pair by = pair_of(inverse, inverse);
                    *reinterpret_cast<uint2*>(to + 256 * k) = make_uint2(e4m3x4(mul2(h[k][0], by), mul2(h[k][1], by)), e4m3x4(mul2(h[k][2], by), mul2(h[k][3], by)));
                    if ((lane & 15u) == 0) scales[2 * k] = (uint8_t)e;
                }
        }
    }
}

// A kernel's dynamic shared memory beyond 48 KB, allowed once on every device.
template <class K>
cudaError_t allow_smem(K kernel, uint32_t bytes, std::atomic<uint64_t>& done) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = device >= 0 && device < 64 ? 1ull << device : 0;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}
constexpr uint32_t kStagedBytes = 115200;  // of a CTA, two to an SM

template <class T, int V, bool RESIDUAL, bool WEIGHT>
void rms_norm_staged(const NormJob& j, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    allow_smem(k_rms_norm_staged<T, V, RESIDUAL, WEIGHT>, kStagedBytes, done);
    const uint32_t weight = WEIGHT ? j.cols * 4 : 0, each = (RESIDUAL ? 4 : 2) * j.cols * 2, warps = std::min(kStagedNormThreads / 32, (kStagedBytes - weight) / each);
    launch_after(k_rms_norm_staged<T, V, RESIDUAL, WEIGHT>, grid_for(j.rows, warps, 2), warps * 32, weight + warps * each, s, j);
}
template <class T, int V>
void rms_norm_staged(const NormJob& j, cudaStream_t s) {
    if (j.residual) j.weight ? rms_norm_staged<T, V, true, true>(j, s) : rms_norm_staged<T, V, true, false>(j, s);
    else j.weight ? rms_norm_staged<T, V, false, true>(j, s) : rms_norm_staged<T, V, false, false>(j, s);
}

template <class T>
void rms_norm(const NormJob& j, cudaStream_t s) {
    const bool x_whole = rows_aligned<T>(j.x, j.x_ld), r_whole = rows_aligned<T>(j.residual, j.residual_ld), s_whole = rows_aligned<T>(j.sum, j.sum_ld),
               y_whole = rows_aligned<T>(j.y, j.y_ld), whole = x_whole && r_whole && s_whole && y_whole && j.cols % 8 == 0;
    if constexpr (sizeof(T) == 2) {
        if (whole && j.cols <= kStagedCols) {
            switch ((j.cols + 255) / 256) {
                case 1: return rms_norm_staged<T, 1>(j, s);
                case 2: return rms_norm_staged<T, 2>(j, s);
                case 3: return rms_norm_staged<T, 3>(j, s);
                case 4: return rms_norm_staged<T, 4>(j, s);
                default: return rms_norm_staged<T, 5>(j, s);
            }
        }
    }
    auto go = [&](auto kernel, uint32_t threads, uint32_t rows_per_cta) {
        const size_t smem = j.weight ? (j.cols + 7) / 8 * 32 : 0;
        // 48 KB, the kernel's own s_part among them, need no allowance
        if (smem + threads / 32 * sizeof(float) > 48 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kNormMaxCols * 4));
        launch_after(kernel, grid_for(j.rows, rows_per_cta, 1024 / threads), threads, smem, s, j, x_whole, r_whole, s_whole, y_whole);
    };
#define DG_NORM(V, TPR, THREADS) (whole ? go(k_rms_norm<T, V, TPR, THREADS, true>, THREADS, THREADS / TPR) : go(k_rms_norm<T, V, TPR, THREADS, false>, THREADS, THREADS / TPR))
    const uint32_t vecs = (j.cols + 7) / 8;
    if (vecs <= 32) DG_NORM(1, 32, 256);
    else if (vecs <= 64) DG_NORM(2, 32, 256);
    else if constexpr (sizeof(T) == 4) {  // half as many elements to a thread
        if (vecs <= 128) DG_NORM(2, 64, 256);
        else if (vecs <= 256) DG_NORM(2, 128, 256);
        else if (vecs <= 512) DG_NORM(2, 256, 256);
        else if (vecs <= 1024) DG_NORM(2, 512, 512);
        else DG_NORM(4, 512, 512);
    } else {
        if (vecs <= 96) DG_NORM(3, 32, 256);
        else if (vecs <= 128) DG_NORM(4, 32, 256);
        else if (vecs <= 160) DG_NORM(5, 32, 256);
        else if (vecs <= 256) DG_NORM(4, 64, 256);
        else if (vecs <= 512) DG_NORM(4, 128, 256);
        else if (vecs <= 1024) DG_NORM(4, 256, 256);
        else DG_NORM(4, 512, 512);
    }
#undef DG_NORM
}

// Backward.  24 images of 2294 x 1152 bf16 with all gradients: 92 us, 4.2 TB/s, 6 of them in the last sums; what bounds it is the chain of a row: its loads,
// the sum along it across five warps, the stores (a warp per row has no barrier, but 160 registers of sums: 100 us and more, and 97
// with rows by cp.async and the sums for dweight in shared memory).
// A worker (a.split.row_threads threads, whole warps) takes units one after the other, and a unit's rows R at a time, so that the loads of R
// rows are under way at once and the R sums along them cross the worker's warps together.  A thread owns V vectors of eight columns of every row; it
// keeps the elements as they were loaded and widens them twice, before and after those sums.
//   Where a residual row has several images, a unit is a residual row t and a part of the rows r with r % period == t: their dx is added up in
//   registers, for dresidual.  Elsewhere a unit is kNormChunk neighbouring rows, and a row of dx is a row of dresidual.
// A worker adds dy * hat of all its rows up in registers, for dweight.  The sums of workers, and of units that share a residual row, go to the
// workspace and are added up in their order.
template <int R>
__device__ __forceinline__ void sums_across(float v[R], uint32_t row_warps, uint32_t worker_warp, uint32_t barrier, uint32_t threads, float (*s_part)[R]) {
    const uint32_t lane = threadIdx.x & 31u;
    // halves of the warp take over half of the sums each, then quarters: lane l is left with sum l / (32 / R)
    float mine;
    if constexpr (R == 4) {
        const bool up = lane & 16u;
        const float a = (up ? v[2] : v[0]) + __shfl_xor_sync(0xFFFFFFFFu, up ? v[0] : v[2], 16), b = (up ? v[3] : v[1]) + __shfl_xor_sync(0xFFFFFFFFu, up ? v[1] : v[3], 16);
        const bool odd = lane & 8u;
        mine = (odd ? b : a) + __shfl_xor_sync(0xFFFFFFFFu, odd ? a : b, 8);
    } else if constexpr (R == 2) {
        const bool up = lane & 16u;
        mine = (up ? v[1] : v[0]) + __shfl_xor_sync(0xFFFFFFFFu, up ? v[0] : v[1], 16);
        mine += __shfl_xor_sync(0xFFFFFFFFu, mine, 8);
    } else {
        mine = v[0] + __shfl_xor_sync(0xFFFFFFFFu, v[0], 16);
        mine += __shfl_xor_sync(0xFFFFFFFFu, mine, 8);
    }
#pragma unroll
    for (int d = 4; d; d >>= 1) mine += __shfl_xor_sync(0xFFFFFFFFu, mine, d);
    if (row_warps == 1) {
#pragma unroll
        for (int r = 0; r < R; ++r) v[r] = __shfl_sync(0xFFFFFFFFu, mine, r * (32 / R));
        return;
    }
    if ((lane & (32 / R - 1)) == 0) s_part[threadIdx.x >> 5][lane / (32 / R)] = mine;
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(threads) : "memory");
    const uint32_t first = (threadIdx.x >> 5) - worker_warp;
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = 0.f;
    for (uint32_t w = 0; w < row_warps; ++w)
#pragma unroll
        for (int r = 0; r < R; ++r) v[r] += s_part[first + w][r];
}

template <class T, int V, int R, int MOST, bool WHOLE>
__global__ void __launch_bounds__(MOST, MOST == 256 ? 2 : 1) k_rms_norm_backward(const NormBackwardJob a, float* w_parts, float* r_parts, bool y_whole, bool h_whole, bool w_whole,
                                                                         bool s_whole, bool x_whole) {
    __shared__ __align__(16) float s_part[2][MOST / 32][R];
    let_next_start();
    wait_for_previous();
    const T *const py = from_previous(reinterpret_cast<const T*>(a.dy)), *const ph = from_previous(reinterpret_cast<const T*>(a.h)),
            *const ps = from_previous(reinterpret_cast<const T*>(a.dsum));
    const float* const prstd = from_previous(a.rstd);
    const uint32_t row_threads = a.split.row_threads, parts = a.split.parts, worker = threadIdx.x / row_threads, t = threadIdx.x - worker * row_threads;
    const uint32_t workers = gridDim.x * a.split.cta_workers, me = blockIdx.x * a.split.cta_workers + worker;
    const bool by_image = a.split.by_image;
    const uint64_t images = by_image ? a.rows / a.period : 0;
    const uint64_t units = by_image ? a.period * parts : (a.rows + kNormChunk - 1) / kNormChunk;
    const float per_col = 1.f / (float)a.cols;
    uint32_t cols[V], valid[V];
    Pair w[V][4], dw[V][4] = {};
#pragma unroll
    for (int k = 0; k < V; ++k) {
        float v[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
        cols[k] = (k * row_threads + t) * 8;
        valid[k] = cols[k] >= a.cols ? 0u : WHOLE ? 8u : min(8u, a.cols - cols[k]);
        if (a.weight && valid[k]) load8_any(from_previous(a.weight), cols[k], a.weight_dtype, valid[k], w_whole, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[k][j] = pair_of(v[2 * j], v[2 * j + 1]);
    }
    uint32_t turn = 0;
    for (uint64_t unit = me; unit < units; unit += workers) {
        uint64_t row0, stride, count;
        if (by_image) {
            const uint64_t part = unit / a.period, first = images * part / parts;
            row0 = first * a.period + (unit - part * a.period);
            stride = a.period;
            count = images * (part + 1) / parts - first;
        } else {
            row0 = unit * kNormChunk;
            stride = 1;
            count = min((uint64_t)kNormChunk, a.rows - row0);
        }
        Pair dr[V][4] = {};  // (a pair of zeros is zero)
        Raw8<T> dy[R][V], h[R][V];
        float rstd[R];
        auto fetch = [&](uint64_t i) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const bool live = i + r < count;
                const uint64_t row = row0 + (i + r) * stride;
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    if constexpr (WHOLE) {
                        dy[r][k].load_whole(py + row * a.dy_ld + cols[k], live && valid[k]);
                        h[r][k].load_whole(ph + row * a.h_ld + cols[k], live && valid[k]);
                    } else {
                        dy[r][k].load(py + row * a.dy_ld + cols[k], live ? valid[k] : 0, y_whole);
                        h[r][k].load(ph + row * a.h_ld + cols[k], live ? valid[k] : 0, h_whole);
                    }
                }
                rstd[r] = live ? prstd[row] : 0.f;
            }
        };
        fetch(0);
        for (uint64_t i = 0; i < count; i += R, turn ^= 1u) {
            Raw8<T> dy_now[R][V], h_now[R][V];
            float rstd_now[R], along[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                rstd_now[r] = rstd[r];
#pragma unroll
                for (int k = 0; k < V; ++k) { dy_now[r][k] = dy[r][k]; h_now[r][k] = h[r][k]; }
            }
            if (i + R < count) fetch(i + R);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                Pair sums = pair_of(0.f, 0.f);
                const Pair rstds = pair_of(rstd_now[r], rstd_now[r]);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    Pair g[4], hat[4];
                    pairs_of(dy_now[r][k], g);
                    pairs_of(h_now[r][k], hat);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const Pair x = mul2(hat[j], rstds), gx = mul2(g[j], x);
                        dw[k][j] = add2(gx, dw[k][j]);
                        sums = fma2(gx, w[k][j], sums);
                    }
                }
                float even, odd;
                parts_of(sums, even, odd);
                along[r] = even + odd;
            }
            sums_across<R>(along, row_threads / 32, t >> 5, worker + 1, row_threads, s_part[turn]);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (i + r >= count) break;
                const uint64_t row = row0 + (i + r) * stride;
                // rstd * (g w - hat mean(g w hat)) = rstd * g w - h * (rstd^2 mean)
                const float back = -along[r] * per_col * rstd_now[r] * rstd_now[r];
                const Pair rstds = pair_of(rstd_now[r], rstd_now[r]), backs = pair_of(back, back);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    if (!valid[k]) continue;
                    Pair d[4], h2[4];
                    pairs_of(dy_now[r][k], d);
                    pairs_of(h_now[r][k], h2);
#pragma unroll
                    for (int j = 0; j < 4; ++j) d[j] = fma2(h2[j], backs, mul2(mul2(d[j], w[k][j]), rstds));
                    if (ps) {
                        float extra[8];
                        load8(ps + row * a.dsum_ld + cols[k], valid[k], WHOLE || s_whole, extra);
#pragma unroll
                        for (int j = 0; j < 4; ++j) d[j] = add2(d[j], pair_of(extra[2 * j], extra[2 * j + 1]));
                    }
                    float v[8];
                    floats_of(d, v);
                    if (a.dx) store8(reinterpret_cast<T*>(a.dx) + row * a.dx_ld + cols[k], valid[k], WHOLE || x_whole, v);
                    if (by_image) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) dr[k][j] = add2(dr[k][j], d[j]);
                    } else if (a.dresidual) {
                        store8(a.dresidual + row * a.cols + cols[k], valid[k], WHOLE && (reinterpret_cast<uintptr_t>(a.dresidual) & 15u) == 0, v);
                    }
                }
            }
        }
        if (by_image) {
            float* const to = parts > 1 ? r_parts + unit * a.cols : a.dresidual + unit * a.cols;
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (valid[k]) {
                    float v[8];
                    floats_of(dr[k], v);
                    store8(to + cols[k], valid[k], WHOLE && (reinterpret_cast<uintptr_t>(to) & 15u) == 0, v);
                }
        }
    }
    if (!a.dweight) return;
    float* const to = w_parts + (uint64_t)me * a.cols;
#pragma unroll
    for (int k = 0; k < V; ++k)
        if (valid[k]) {  // the workspace is aligned, and so are its rows if they are whole vectors
            float v[8];
            floats_of(dw[k], v);
            store8(to + cols[k], valid[k], WHOLE, v);
        }
}

// out[i] = the sum of parts[p][i] in a fixed order: eight columns a CTA, sixty-four threads a column, each every sixty-fourth part
constexpr uint32_t kSumThreads = 512, kSumCols = 8, kSumLanes = kSumThreads / kSumCols;
__global__ void __launch_bounds__(kSumThreads) k_sum_parts(const float* parts, uint32_t count, uint64_t n, float* out) {
    __shared__ float s_sum[kSumThreads / 32][kSumCols];
    let_next_start();
    wait_for_previous();
    parts = from_previous(parts);
    const uint32_t col = threadIdx.x % kSumCols, part = threadIdx.x / kSumCols;
    for (uint64_t i0 = (uint64_t)blockIdx.x * kSumCols; i0 < n; i0 += (uint64_t)gridDim.x * kSumCols) {
        const uint64_t i = i0 + col;
        float sum = 0.f;
        if (i < n) {
            uint32_t p = part;
            for (; p + 3 * kSumLanes < count; p += 4 * kSumLanes) {
                const float a = parts[p * n + i], b = parts[(p + kSumLanes) * n + i], c = parts[(p + 2 * kSumLanes) * n + i], d = parts[(p + 3 * kSumLanes) * n + i];
                sum += (a + b) + (c + d);
            }
            for (; p < count; p += kSumLanes) sum += parts[p * n + i];
        }
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 8);
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 16);
        if ((threadIdx.x & 31u) < kSumCols) s_sum[threadIdx.x >> 5][col] = sum;
        __syncthreads();
        if (threadIdx.x < kSumCols && i < n) {
            float all = 0.f;
#pragma unroll
            for (uint32_t w = 0; w < kSumThreads / 32; ++w) all += s_sum[w][col];
            out[i] = all;
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
    const NormBackwardSplit& d = j.split;
    const uint64_t workers = (uint64_t)d.ctas * d.cta_workers;
    float* const r_parts = workspace + workers * j.cols;
    const bool y_whole = rows_aligned<T>(j.dy, j.dy_ld), h_whole = rows_aligned<T>(j.h, j.h_ld), s_whole = rows_aligned<T>(j.dsum, j.dsum_ld),
               x_whole = rows_aligned<T>(j.dx, j.dx_ld), whole = y_whole && h_whole && s_whole && x_whole && j.cols % 8 == 0;
    auto go = [&](auto kernel) {
        launch_after(kernel, d.ctas, d.row_threads * d.cta_workers, 0, s, j, workspace, r_parts, y_whole, h_whole, (reinterpret_cast<uintptr_t>(j.weight) & 15u) == 0, s_whole,
                     x_whole);
    };
    // Rows at a time, and as many under way: what 128 registers hold.  Four at a time with none under way took 102 us (24 images of 2294 x 1152,
    // bf16), two with 85 registers 118 and more CTAs, two with the next two under way 97.
    constexpr int kRows = sizeof(T) == 4 ? 1 : 2;
    const uint64_t vecs = (j.cols + 7) / 8;
    if (vecs <= 256) whole ? go(k_rms_norm_backward<T, 1, kRows, 256, true>) : go(k_rms_norm_backward<T, 1, kRows, 256, false>);
    else if (vecs <= 512) whole ? go(k_rms_norm_backward<T, 1, kRows, 512, true>) : go(k_rms_norm_backward<T, 1, kRows, 512, false>);
    else if (vecs <= 1024) whole ? go(k_rms_norm_backward<T, 2, 1, 512, true>) : go(k_rms_norm_backward<T, 2, 1, 512, false>);
    else whole ? go(k_rms_norm_backward<T, 2, 1, 1024, true>) : go(k_rms_norm_backward<T, 2, 1, 1024, false>);
    auto add_up = [&](const float* parts, uint32_t count, uint64_t n, float* out) {
        launch_after(k_sum_parts, grid_for(n, kSumCols, 4), kSumThreads, 0, s, parts, count, n, out);
    };
    if (j.dweight) add_up(workspace, (uint32_t)workers, j.cols, j.dweight);
    if (d.by_image && d.parts > 1) add_up(r_parts, d.parts, j.period * j.cols, j.dresidual);
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

// 131072 x 1152 bf16: 107 to 116 us over inputs that differ from call to call, 5.2 to 5.6 TB/s, 70 % of the places to issue an instruction; ten rounds are 40
// of about 110 instructions for eight elements.  Whole tokens go the same way, with a generator's block for every eight columns: 1571 x 777 f32 7 us.
// One row: the matrix without gaps, as long as need be.  EIGHTS: every vector of eight begins with an index that is a multiple of eight.
constexpr int kDropoutVecs = 2;  // of a thread under way at once

template <class T, bool ONE_ROW, bool EIGHTS, bool PER_ROW>
__global__ void __launch_bounds__(kRowThreads) k_dropout(const DropoutJob a, uint64_t nvec, uint64_t per_row, float scale, bool x_whole, bool y_whole) {
    let_next_start();
    wait_for_previous();
    const T* const x = from_previous(reinterpret_cast<const T*>(a.x));
    T* const y = reinterpret_cast<T*>(a.y);
    const uint64_t step = (uint64_t)gridDim.x * kRowThreads * kDropoutVecs;
    const Pair scales = pair_of(scale, scale);
    const uint32_t least = a.threshold << 16;
    for (uint64_t i0 = (uint64_t)blockIdx.x * kRowThreads * kDropoutVecs + threadIdx.x; i0 < nvec; i0 += step) {
        uint64_t row[kDropoutVecs], col[kDropoutVecs];
        uint32_t valid[kDropoutVecs];
        Raw8<T> raw[kDropoutVecs];
#pragma unroll
        for (int k = 0; k < kDropoutVecs; ++k) {
            const uint64_t i = i0 + k * kRowThreads;
            row[k] = ONE_ROW ? 0 : i / per_row;
            col[k] = (i - row[k] * per_row) * 8;
            valid[k] = i < nvec ? (uint32_t)min((uint64_t)8, a.cols - col[k]) : 0;
            raw[k].load(x + row[k] * a.x_ld + col[k], valid[k], x_whole);
        }
#pragma unroll
        for (int k = 0; k < kDropoutVecs; ++k) {
            if (!valid[k]) continue;
            const uint64_t index = a.offset + (PER_ROW ? row[k] : row[k] * a.cols + col[k]);
            uint32_t bits[4];
            if constexpr (EIGHTS) {
                const uint4 b = philox(index >> 3, a.seed);
                bits[0] = b.x; bits[1] = b.y; bits[2] = b.z; bits[3] = b.w;
            } else {
                bits_of_8(index, a.seed, bits);
            }
            Pair p[4];
            pairs_of(raw[k], p);
            float v[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // a half is compared where it is the upper one: what lies below it does not matter
                const uint32_t lo = PER_ROW ? bits[0] << 16 : bits[j] << 16, hi = PER_ROW ? lo : bits[j];
                parts_of(mul2(p[j], scales), v[2 * j], v[2 * j + 1]);
                v[2 * j] = lo >= least ? v[2 * j] : 0.f;
                v[2 * j + 1] = hi >= least ? v[2 * j + 1] : 0.f;
            }
            store8(y + row[k] * a.y_ld + col[k], valid[k], y_whole, v);
        }
    }
}

template <class T>
void dropout(DropoutJob j, cudaStream_t s) {
    const bool one_row = !j.per_row && (j.rows == 1 || (j.x_ld == j.cols && j.y_ld == j.cols));
    if (one_row) {
        j.cols *= j.rows;
        j.x_ld = j.y_ld = (j.cols + 7) / 8 * 8;
        j.rows = 1;
    }
    const uint64_t per_row = (j.cols + 7) / 8, n = j.rows * per_row;
    auto go = [&](auto kernel) {
        launch_after(kernel, grid_for(n, kRowThreads * kDropoutVecs, 32), kRowThreads, 0, s, j, n, per_row, 65536.f / (float)(65536u - j.threshold),
                     rows_aligned<T>(j.x, j.x_ld), rows_aligned<T>(j.y, j.y_ld));
    };
    const bool eights = j.offset % 8 == 0 && (one_row || j.cols % 8 == 0);
    if (j.per_row) go(k_dropout<T, false, false, true>);
    else if (one_row && eights) go(k_dropout<T, true, true, false>);
    else if (one_row) go(k_dropout<T, true, false, false>);
    else go(k_dropout<T, false, false, false>);
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
