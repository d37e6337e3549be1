// C entry points of the token rows (declared in include/datago_b200.h): checks of the arguments, tensor maps, launches.  None of them
// allocates, waits or keeps anything (dg_product_status apart), so calls need no lock and can be captured.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "host.h"
#include "tokens.h"

using namespace dg;

// ---- how the work is dealt out ------------------------------------------------------------------------------------------
namespace dg {

ProductPlan plan_product(uint64_t m, uint64_t n, uint64_t k, bool b_by_column) {
    ProductPlan p{};
    if (m == 0 || n == 0) return p;
    constexpr uint32_t kPairs = kTokenSms / 2;
    const uint32_t groups = (uint32_t)scale_groups(k);
    p.tiles_m = (uint32_t)((m + kProductTileM - 1) / kProductTileM);
    // Column tiles of one width, as wide as can be (with two accumulators, or up to 256 columns with one), or narrower so that more SMs have one; the
    // contraction whole or in parts.  The cheapest in cycles, by what was measured: a group of 128 takes two cycles a column, but no less than
    // its bytes do at 39 a cycle and SM (that is 10 TB/s, where copies out of L2 end); a tile's sums 700 before and after it, or 150 where the
    // next tile hides them; parts a launch more, and their bytes twice.
    uint64_t best = ~0ull;
    for (uint64_t want = (n + kProductMaxTileN - 1) / kProductMaxTileN;; want *= 2) {
        for (const uint32_t widest : {kProductMaxTileN, kProductTwoSums}) {
            ProductPlan q = p;
            const uint64_t count = std::max<uint64_t>(want, (n + widest - 1) / widest);
            q.tile_n = (uint32_t)((n + count - 1) / count + 31) / 32 * 32;
            q.tiles_n = (uint32_t)((n + q.tile_n - 1) / q.tile_n);
            q.sums = q.tile_n <= kProductTwoSums ? 2 : 1;
            const uint64_t tiles = (uint64_t)q.tiles_m * q.tiles_n;
            const uint32_t b_bytes = (b_by_column ? 128 : q.tile_n / 2) * 128;
            // The tensor cores cut off what lies below their sums, and lose the more the longer a sum is (random terms over 116 groups 1.4e-6 of the
            // result, over 44 3e-7; beside one large term all small ones): no part is longer than kProductPartGroups (4096 x 4096 x
            // 131072 1.91 ms, in one part 1.52; 4096 x 1152 x 57600 285 us, in three parts 225).  More parts than that asks for, up to 16, where they
            // spread the work.
            const uint32_t least = (groups + kProductPartGroups - 1) / kProductPartGroups;
            for (uint32_t s = least; s == least || (s <= 16 && s * 8 <= groups); ++s) {
                q.split_groups = s == 1 ? groups : ((groups + s - 1) / s + 3) / 4 * 4;  // parts begin at multiples of four groups: the scales come in words
                q.splits = (groups + q.split_groups - 1) / q.split_groups;
                // a stays where its rows leave room for three slots of b and most pairs walk tiles of the same rows
                q.a_stays = q.splits == 1 && groups <= 2 * kProductSlots && groups * kProductABytes + 3 * 2 * b_bytes <= kProductRingBytes && tiles >= 2 * kPairs && q.tiles_n > 1;
                q.slots = std::min(kProductSlots, (kProductRingBytes - (q.a_stays ? groups * kProductABytes : 0)) / (2 * (b_bytes + (q.a_stays ? 0 : kProductABytes))));
                const uint64_t rounds = (tiles * q.splits + kPairs - 1) / kPairs, group = std::max(2 * q.tile_n, (b_bytes + (q.a_stays ? 0 : kProductABytes)) / 39);
                const uint64_t cost = rounds * q.split_groups * group + (q.sums == 2 ? 700 + (rounds - 1) * 150 : rounds * 700) + (q.splits > 1 ? 4000 + q.splits * m * n / 400 : 0);
                if (cost < best) {
                    best = cost;
                    p = q;
                }
            }
        }
        if (p.tiles_m * want * 2 > kPairs || n / want <= 32) break;
    }
    p.together = (uint32_t)std::min<uint64_t>(p.splits, std::max<uint64_t>(1, kProductPartsBytes / (4 * m * product_part_ld(n))));
    return p;
}

NormBackwardSplit norm_backward_split(uint64_t rows, uint64_t cols, uint64_t period, bool residual) {
    NormBackwardSplit d{};
    const uint64_t vecs = (cols + 7) / 8;
    const uint64_t each = vecs > 512 ? 2 : 1;  // vectors of eight columns that a thread owns
    d.row_threads = (uint32_t)((vecs + each - 1) / each + 31) / 32 * 32;
    d.cta_workers = std::max(1u, 256 / d.row_threads);
    const uint64_t ctas = (uint64_t)kTokenSms * std::max(1u, 480 / (d.row_threads * d.cta_workers)), workers = ctas * d.cta_workers;
    const uint64_t images = residual ? rows / period : 1;
    d.by_image = images > 1;
    d.parts = 1;
    // few residual rows: their images go to several workers, four at least to each
    if (d.by_image && period < workers) d.parts = (uint32_t)std::max<uint64_t>(1, std::min(images / 4, workers / period));
    const uint64_t units = d.by_image ? period * d.parts : (rows + kNormChunk - 1) / kNormChunk;
    d.ctas = (uint32_t)std::max<uint64_t>(1, std::min((units + d.cta_workers - 1) / d.cta_workers, ctas));
    return d;
}

}  // namespace dg

namespace {

int fail(int code, const char* fmt, ...) {
    char msg[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof msg, fmt, ap);
    va_end(ap);
    return dg_set_error(code, msg);
}

// The context's device while a call lasts.
struct OnDevice {
    int before = -1, device;
    cudaError_t error;
    explicit OnDevice(int d) : device(d) {
        error = cudaGetDevice(&before);
        if (error == cudaSuccess && before != d) error = cudaSetDevice(d);
    }
    ~OnDevice() {
        if (before >= 0 && before != device) cudaSetDevice(before);
    }
};

constexpr uint64_t kMostCols = (1ull << 31) - 1024, kMostRows = 1ull << 40, kMostElements = 1ull << 60;

int check_ctx(const dg_ctx* ctx) {
    if (!ctx) return fail(DG_E_INVALID, "ctx is NULL");
    if (ctx_device(ctx) == DG_DEVICE_NONE) return fail(DG_E_INVALID, "planning-only context: token rows need a CUDA device");
    return DG_OK;
}
uint64_t element(int32_t dtype) { return dtype == DG_F32 ? 4 : 2; }
int check_matrix(const dg_matrix* m, const char* name) {
    if (!m) return fail(DG_E_INVALID, "%s is NULL", name);
    if (m->dtype < DG_F32 || m->dtype > DG_F16) return fail(DG_E_INVALID, "%s: unknown dtype %d", name, (int)m->dtype);
    if (m->cols == 0 || m->cols > kMostCols || m->rows > kMostRows) return fail(DG_E_INVALID, "%s: %llu x %llu elements", name, (unsigned long long)m->rows, (unsigned long long)m->cols);
    if (m->ld < m->cols || m->ld > kMostElements / (m->rows + 1)) return fail(DG_E_INVALID, "%s: rows of %llu elements %llu apart", name, (unsigned long long)m->cols, (unsigned long long)m->ld);
    if (m->rows && !m->data) return fail(DG_E_INVALID, "%s: data is NULL", name);
    if ((uintptr_t)m->data % element(m->dtype)) return fail(DG_E_INVALID, "%s: data is not aligned to its elements", name);
    return DG_OK;
}
int check_rows8(const dg_rows8* r, const char* name) {
    if (!r) return fail(DG_E_INVALID, "%s is NULL", name);
    if (r->block != 1 && r->block != kScaleGroup) return fail(DG_E_INVALID, "%s: block is 1 or 128", name);
    if (r->cols == 0 || r->cols > kMostCols || r->rows > kMostRows) return fail(DG_E_INVALID, "%s: %llu x %llu elements", name, (unsigned long long)r->rows, (unsigned long long)r->cols);
    if (r->by_column > 1) return fail(DG_E_INVALID, "%s: by_column is 0 or 1", name);
    const uint64_t line = r->by_column ? r->rows : r->cols, lines = r->by_column ? r->cols : r->rows;
    if (r->ld < line || r->ld % 16 || r->ld > kMostElements / (lines + 1)) return fail(DG_E_INVALID, "%s: ld is a multiple of 16 and at least the %s", name, r->by_column ? "rows" : "cols");
    if (r->scale_ld < scale_groups(r->cols) || r->scale_ld % 4 || r->scale_ld > kMostElements / (r->rows + 1))
        return fail(DG_E_INVALID, "%s: scale_ld is a multiple of 4 and at least a byte per 128 columns", name);
    if (r->rows && (!r->values || !r->scales)) return fail(DG_E_INVALID, "%s: values or scales are NULL", name);
    if ((uintptr_t)r->values % 16 || (uintptr_t)r->scales % 4) return fail(DG_E_INVALID, "%s: values are 16-byte aligned, scales 4-byte", name);
    return DG_OK;
}
int check_like(const dg_matrix* m, const char* name, uint64_t rows, uint64_t cols, int32_t dtype) {
    if (int rc = check_matrix(m, name)) return rc;
    if (m->rows != rows || m->cols != cols) return fail(DG_E_INVALID, "%s: %llu x %llu elements, %llu x %llu wanted", name, (unsigned long long)m->rows, (unsigned long long)m->cols, (unsigned long long)rows, (unsigned long long)cols);
    if (m->dtype != dtype) return fail(DG_E_INVALID, "%s: another dtype than the input's", name);
    return DG_OK;
}
int check_rows8_like(const dg_rows8* r, const char* name, uint64_t rows, uint64_t cols) {
    if (int rc = check_rows8(r, name)) return rc;
    if (r->rows != rows || r->cols != cols) return fail(DG_E_INVALID, "%s: %llu x %llu elements, %llu x %llu wanted", name, (unsigned long long)r->rows, (unsigned long long)r->cols, (unsigned long long)rows, (unsigned long long)cols);
    return DG_OK;
}
int check_weight(const dg_matrix* w, uint64_t cols) {
    if (!w) return DG_OK;
    if (int rc = check_matrix(w, "weight")) return rc;
    if (w->rows != 1 || w->cols != cols) return fail(DG_E_INVALID, "weight: 1 x %llu elements wanted", (unsigned long long)cols);
    return DG_OK;
}
int check_floats(const float* p, const char* name) { return (uintptr_t)p % 4 ? fail(DG_E_INVALID, "%s is not aligned to its elements", name) : DG_OK; }
int check_workspace(const void* p, uint64_t bytes, uint64_t needed) {
    if (bytes < needed || (needed && !p)) return fail(DG_E_INVALID, "workspace of %llu bytes, %llu needed", (unsigned long long)bytes, (unsigned long long)needed);
    if (needed && (uintptr_t)p % 16) return fail(DG_E_INVALID, "workspace is not 16-byte aligned");
    return DG_OK;
}

// Where a matrix lies.  Two of them share memory unless their ranges are apart, or they are other columns of rows that are equally far apart (as a
// single row is from any).
struct Lies {
    uintptr_t at;
    uint64_t rows, width, pitch;  // bytes
};
Lies lies(const dg_matrix* m) { return {(uintptr_t)m->data, m->rows, m->cols * element(m->dtype), m->ld * element(m->dtype)}; }
Lies lies(const dg_rows8* r) { return r->by_column ? Lies{(uintptr_t)r->values, r->cols, r->rows, r->ld} : Lies{(uintptr_t)r->values, r->rows, r->cols, r->ld}; }
bool share(const Lies& a, const Lies& b) {
    if (!a.rows || !b.rows || !a.at || !b.at) return false;
    if (a.at + (a.rows - 1) * a.pitch + a.width <= b.at || b.at + (b.rows - 1) * b.pitch + b.width <= a.at) return false;
    if (a.rows > 1 && b.rows > 1 && a.pitch != b.pitch) return true;
    const uint64_t pitch = a.rows > 1 ? a.pitch : b.pitch, apart = (b.at % pitch + pitch - a.at % pitch) % pitch;  // from the columns of a to those of b
    return !(apart >= a.width && apart + b.width <= pitch);
}
// out may be in, where that is said of them, but not reach into it otherwise
template <class A, class B>
int check_apart(const A* out, const char* out_name, const B* in, const char* in_name, bool in_place = false) {
    if (!out || !in) return DG_OK;
    const Lies a = lies(out), b = lies(in);
    if (in_place && a.at == b.at && (a.pitch == b.pitch || a.rows <= 1)) return DG_OK;
    return share(a, b) ? fail(DG_E_INVALID, "%s overlaps %s", out_name, in_name) : DG_OK;
}

cudaStream_t stream_of(dg_ctx* ctx, void* stream) { return stream ? (cudaStream_t)stream : (cudaStream_t)dg_ctx_stream(ctx); }
// Runs `launch` (which returns a cudaError_t or nothing) on the context's device.
template <class F>
int launched(dg_ctx* ctx, F&& launch) {
    OnDevice on(ctx_device(ctx));
    if (on.error != cudaSuccess) return fail(DG_E_CUDA, "device %d: %s", ctx_device(ctx), cudaGetErrorString(on.error));
    launch();
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? DG_OK : fail(DG_E_CUDA, "launch: %s", cudaGetErrorString(e));
}

}  // namespace

extern "C" int dg_patch_rows(dg_ctx* ctx, void* stream, const uint8_t* pixels, uint32_t n, uint32_t h, uint32_t w, uint32_t channels,
                             uint32_t patch, const float* mean, const float* std, const dg_rows8* out8, const dg_matrix* out) {
    if (int rc = check_ctx(ctx)) return rc;
    if (!mean || !std || !out8 == !out) return fail(DG_E_INVALID, "mean and std, and one of out8 and out, are wanted");
    if (channels < 1 || channels > 4) return fail(DG_E_INVALID, "%u channels: 1 to 4 are wanted", channels);
    if (patch == 0 || patch > 4096 || h == 0 || w == 0 || h % patch || w % patch) return fail(DG_E_INVALID, "%u x %u pixels are no whole number of %u x %u patches", h, w, patch, patch);
    const uint64_t per_image = (uint64_t)(h / patch) * (w / patch), rows = n * per_image, cols = (uint64_t)patch * patch * channels;
    if ((uint64_t)patch * (patch * channels + 11) > 48 * 1024 - 24) return fail(DG_E_TOO_LARGE, "patches of %u x %u x %u: at most 48 KB", patch, patch, channels);
    if (per_image > (1ull << 27) / scale_groups(cols)) return fail(DG_E_TOO_LARGE, "%u x %u pixels are too many for one image", h, w);
    if (n > kMostCols) return fail(DG_E_TOO_LARGE, "%u images: at most %llu", n, (unsigned long long)kMostCols);  // launches add up to 2^30 images to a count of 32 bits
    if (n && !pixels) return fail(DG_E_INVALID, "pixels is NULL");
    if (out) {
        if (int rc = check_matrix(out, "out")) return rc;
        if (out->rows != rows || out->cols != cols) return fail(DG_E_INVALID, "out: %llu x %llu elements wanted", (unsigned long long)rows, (unsigned long long)cols);
    } else {
        if (int rc = check_rows8_like(out8, "out8", rows, cols)) return rc;
        if (out8->block != 1 || out8->by_column) return fail(DG_E_INVALID, "out8: patches have block 1 and are stored by row");
    }
    PatchJob j{pixels, n, h, w, channels, patch, {}, {}};
    for (uint32_t c = 0; c < channels; ++c) {
        if (!(std[c] > 0) || !std::isfinite(std[c]) || !std::isfinite(mean[c])) return fail(DG_E_INVALID, "channel %u: mean and std are finite, std above 0", c);
        j.gain[c] = (float)(1.0 / (255.0 * std[c]));
        j.shift[c] = (float)(-(double)mean[c] / std[c]);
        if (!std::isfinite(255 * j.gain[c]) || !std::isfinite(j.shift[c])) return fail(DG_E_INVALID, "channel %u: std is too small", c);
    }
    if (rows == 0) return DG_OK;
    return launched(ctx, [&] { launch_patch_rows(j, out8, out, stream_of(ctx, stream)); });
}

extern "C" int dg_quantize_rows(dg_ctx* ctx, void* stream, const dg_matrix* src, const dg_rows8* out) {
    if (int rc = check_ctx(ctx)) return rc;
    if (int rc = check_matrix(src, "src")) return rc;
    if (!out) return fail(DG_E_INVALID, "out is NULL");
    if (out->by_column && src->rows == 0) return fail(DG_E_INVALID, "the transpose of a matrix without rows has no columns");
    if (int rc = check_rows8_like(out, "out", out->by_column ? src->cols : src->rows, out->by_column ? src->rows : src->cols)) return rc;
    if (int rc = check_apart(out, "out", src, "src")) return rc;
    if (src->rows == 0) return DG_OK;
    return launched(ctx, [&] { launch_quantize_rows(*src, *out, stream_of(ctx, stream)); });
}

extern "C" uint64_t dg_product_workspace(dg_ctx* ctx, uint64_t m, uint64_t n, uint64_t k) {
    if (!ctx || m > kMostCols || n > kMostCols || k > kMostCols) return 0;
    return std::max(product_workspace(plan_product(m, n, k, false), m, n), product_workspace(plan_product(m, n, k, true), m, n));
}

extern "C" int dg_product(dg_ctx* ctx, void* stream, const dg_rows8* a, const dg_rows8* b, const dg_matrix* out, void* workspace,
                          uint64_t workspace_bytes) {
    if (int rc = check_ctx(ctx)) return rc;
    if (int rc = check_rows8(a, "a")) return rc;
    if (int rc = check_rows8(b, "b")) return rc;
    if (a->cols != b->cols) return fail(DG_E_INVALID, "a has %llu columns, b %llu", (unsigned long long)a->cols, (unsigned long long)b->cols);
    if (a->rows > kMostCols || b->rows == 0 || b->rows > kMostCols) return fail(DG_E_INVALID, "a has %llu rows, b %llu", (unsigned long long)a->rows, (unsigned long long)b->rows);
    if (int rc = check_matrix(out, "out")) return rc;
    if (out->rows != a->rows || out->cols != b->rows) return fail(DG_E_INVALID, "out: %llu x %llu elements wanted", (unsigned long long)a->rows, (unsigned long long)b->rows);
    for (const dg_rows8* in : {a, b})
        if (int rc = check_apart(out, "out", in, "an operand")) return rc;
    if (a->rows == 0) return DG_OK;
    ProductJob j{};
    j.plan = plan_product(a->rows, b->rows, a->cols, b->by_column != 0);
    if ((uint64_t)j.plan.tiles_m * j.plan.tiles_n * j.plan.together > kMostCols) return fail(DG_E_TOO_LARGE, "more tiles than a launch can count");
    if (int rc = check_workspace(workspace, workspace_bytes, dg_product_workspace(ctx, a->rows, b->rows, a->cols))) return rc;
    const auto encode = (CUresult(*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                     const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill))encode_tiled_entry();
    if (!encode) return fail(DG_E_CUDA, "the driver has no cuTensorMapEncodeTiled");
    auto map = [&](CUtensorMap* m, CUtensorMapDataType type, cuuint32_t dims, void* at, const cuuint64_t* dim, const cuuint64_t* pitch, const cuuint32_t* box,
                   CUtensorMapSwizzle swizzle) {
        const cuuint32_t step[3] = {1, 1, 1};
        return encode(m, type, dims, at, dim, pitch, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    // lines of bytes (rows, or columns); a copy brings 128 bytes of them, what lies outside the matrix as zeros
    auto operand = [&](CUtensorMap* m, const dg_rows8& r, uint32_t rows) {
        const cuuint64_t dim[2] = {r.by_column ? r.rows : r.cols, r.by_column ? r.cols : r.rows}, pitch[1] = {r.ld};
        const cuuint32_t box[2] = {128, r.by_column ? 128 : rows};
        return map(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, r.values, dim, pitch, box, CU_TENSOR_MAP_SWIZZLE_128B);
    };
    if (!operand(&j.a, *a, kProductTileM / 2) || !operand(&j.b, *b, j.plan.tile_n / 2)) return fail(DG_E_CUDA, "cuTensorMapEncodeTiled rejected an operand");
    {  // the output, or the parts of a launch; rows that do not start at multiples of 16 bytes are stored without a map.  A map stores whole sixteens of
       // bytes, also where its rows end inside one: it has the columns of whole ones only.
        const bool split = j.plan.splits > 1;
        void* const at = split ? workspace : out->data;
        const int32_t dtype = split ? (int32_t)DG_F32 : out->dtype;
        const uint64_t ld = (split ? product_part_ld(b->rows) : out->ld) * element(dtype), cols = split ? product_part_ld(b->rows) : b->rows - b->rows % (16 / element(dtype));
        const cuuint64_t dim[3] = {cols, a->rows, j.plan.together}, pitch[2] = {ld, ld * a->rows};
        const cuuint32_t box[3] = {(cuuint32_t)(64 / element(dtype)), 32, 1};
        const CUtensorMapDataType types[3] = {CU_TENSOR_MAP_DATA_TYPE_FLOAT32, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, CU_TENSOR_MAP_DATA_TYPE_FLOAT16};
        if (cols && ((uintptr_t)at | ld) % 16 == 0 && pitch[1] < 1ull << 40 && map(&j.out_map, types[dtype], 3, at, dim, pitch, box, CU_TENSOR_MAP_SWIZZLE_64B))
            j.map_cols = std::min<uint64_t>(cols, b->rows);
    }
    j.a_by_column = a->by_column != 0; j.b_by_column = b->by_column != 0;
    j.a_scales = a->scales; j.b_scales = b->scales;
    j.a_scale_ld = a->scale_ld; j.b_scale_ld = b->scale_ld;
    j.a_block = a->block; j.b_block = b->block;
    j.m = a->rows; j.n = b->rows; j.k = a->cols;
    j.out = out->data; j.ld = out->ld; j.dtype = out->dtype;
    j.parts = (float*)workspace;
    OnDevice on(ctx_device(ctx));
    if (on.error != cudaSuccess) return fail(DG_E_CUDA, "device %d: %s", ctx_device(ctx), cudaGetErrorString(on.error));
    const cudaError_t e = launch_product(j, stream_of(ctx, stream));
    return e == cudaSuccess ? DG_OK : fail(DG_E_CUDA, "launch: %s", cudaGetErrorString(e));
}

extern "C" int dg_product_status(dg_ctx* ctx, void* stream) {
    if (int rc = check_ctx(ctx)) return rc;
    OnDevice on(ctx_device(ctx));
    unsigned int count = 0;
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    if (on.error == cudaSuccess && cudaStreamIsCapturing(stream_of(ctx, stream), &capture) == cudaSuccess && capture != cudaStreamCaptureStatusNone)
        return fail(DG_E_INVALID, "the stream is being captured");
    const cudaError_t e = on.error != cudaSuccess ? on.error : product_gave_up(&count, stream_of(ctx, stream));
    if (e != cudaSuccess) return fail(DG_E_CUDA, "%s", cudaGetErrorString(e));
    count = ctx_products_unreported(ctx, count);
    return count ? fail(DG_E_SYNC_LIMIT, "%u CTAs of products gave up waiting for a copy", count) : DG_OK;
}

extern "C" int dg_rms_norm(dg_ctx* ctx, void* stream, const dg_matrix* x, const dg_matrix* residual, const dg_matrix* weight, float eps,
                           const dg_matrix* sum, const dg_matrix* y, const dg_rows8* y8, float* rstd) {
    if (int rc = check_ctx(ctx)) return rc;
    if (int rc = check_matrix(x, "x")) return rc;
    if (x->cols > kNormMaxCols) return fail(DG_E_TOO_LARGE, "rows of %llu elements: at most %llu", (unsigned long long)x->cols, (unsigned long long)kNormMaxCols);
    if (residual) {
        if (int rc = check_matrix(residual, "residual")) return rc;
        if (residual->cols != x->cols || residual->dtype != x->dtype) return fail(DG_E_INVALID, "residual: the columns and dtype of x are wanted");
        if (residual->rows == 0 || x->rows % residual->rows || residual->rows >> 32) return fail(DG_E_INVALID, "residual: %llu rows do not divide %llu", (unsigned long long)residual->rows, (unsigned long long)x->rows);
    }
    if (int rc = check_weight(weight, x->cols)) return rc;
    if (!(eps >= 0) || !std::isfinite(eps)) return fail(DG_E_INVALID, "eps is finite and not below 0");
    if (sum) {
        if (int rc = check_like(sum, "sum", x->rows, x->cols, x->dtype)) return rc;
    }
    if (y) if (int rc = check_like(y, "y", x->rows, x->cols, x->dtype)) return rc;
    if (y8) {
        if (int rc = check_rows8_like(y8, "y8", x->rows, x->cols)) return rc;
        if (y8->block != 1 || y8->by_column) return fail(DG_E_INVALID, "y8: a norm's rows have block 1 and are stored by row");
    }
    if (int rc = check_floats(rstd, "rstd")) return rc;
    if (!sum && !y && !y8 && !rstd) return fail(DG_E_INVALID, "no output is wanted");
    if (int rc = check_apart(sum, "sum", x, "x", true)) return rc;
    if (int rc = check_apart(y, "y", sum, "sum")) return rc;
    if (int rc = check_apart(y8, "y8", sum, "sum")) return rc;
    if (int rc = check_apart(y, "y", y8, "y8")) return rc;
    for (const dg_matrix* in : {x, residual, weight}) {
        if (int rc = in == x ? DG_OK : check_apart(sum, "sum", in, "an input")) return rc;
        if (int rc = check_apart(y, "y", in, "an input")) return rc;
        if (int rc = check_apart(y8, "y8", in, "an input")) return rc;
    }
    if (x->rows == 0) return DG_OK;
    NormJob j{};
    j.rows = x->rows; j.cols = (uint32_t)x->cols; j.dtype = x->dtype; j.eps = eps;
    j.x = x->data; j.x_ld = x->ld;
    if (residual) { j.residual = residual->data; j.residual_ld = residual->ld; j.residual_rows = (uint32_t)residual->rows; }
    if (weight) { j.weight = weight->data; j.weight_dtype = weight->dtype; }
    if (sum) { j.sum = sum->data; j.sum_ld = sum->ld; }
    if (y) { j.y = y->data; j.y_ld = y->ld; }
    if (y8) j.y8 = *y8;
    j.rstd = rstd;
    return launched(ctx, [&] { launch_rms_norm(j, stream_of(ctx, stream)); });
}

extern "C" uint64_t dg_rms_norm_backward_workspace(dg_ctx* ctx, uint64_t rows, uint64_t cols, uint64_t residual_rows) {
    if (!ctx || rows == 0 || cols == 0 || cols > kNormMaxCols || rows > kMostRows) return 0;
    // a call without dresidual ignores residual_rows and deals the rows out otherwise
    const uint64_t without = norm_backward_workspace(norm_backward_split(rows, cols, rows, false), cols, rows);
    if (!residual_rows || rows % residual_rows) return without;
    return std::max(without, norm_backward_workspace(norm_backward_split(rows, cols, residual_rows, true), cols, residual_rows));
}

extern "C" int dg_rms_norm_backward(dg_ctx* ctx, void* stream, const dg_matrix* dy, const dg_matrix* h, const float* rstd, const dg_matrix* weight,
                                    const dg_matrix* dsum, const dg_matrix* dx, float* dresidual, uint64_t residual_rows, float* dweight,
                                    void* workspace, uint64_t workspace_bytes) {
    if (int rc = check_ctx(ctx)) return rc;
    if (int rc = check_matrix(dy, "dy")) return rc;
    if (dy->cols > kNormMaxCols) return fail(DG_E_TOO_LARGE, "rows of %llu elements: at most %llu", (unsigned long long)dy->cols, (unsigned long long)kNormMaxCols);
    if (int rc = check_like(h, "h", dy->rows, dy->cols, dy->dtype)) return rc;
    if (int rc = check_weight(weight, dy->cols)) return rc;
    if (dsum) if (int rc = check_like(dsum, "dsum", dy->rows, dy->cols, dy->dtype)) return rc;
    if (dx) {
        if (int rc = check_like(dx, "dx", dy->rows, dy->cols, dy->dtype)) return rc;
        for (const dg_matrix* in : {dy, dsum})
            if (int rc = check_apart(dx, "dx", in, "a gradient", true)) return rc;
        for (const dg_matrix* in : {h, weight})
            if (int rc = check_apart(dx, "dx", in, "h or weight")) return rc;
    }
    if (dy->rows && !rstd) return fail(DG_E_INVALID, "rstd is NULL");
    if (!dx && !dresidual && !dweight) return fail(DG_E_INVALID, "no output is wanted");
    for (const float* p : {rstd, (const float*)dresidual, (const float*)dweight})
        if (int rc = check_floats(p, "rstd, dresidual or dweight")) return rc;
    if (dresidual && (residual_rows == 0 || dy->rows % residual_rows || residual_rows > kMostRows))
        return fail(DG_E_INVALID, "%llu residual rows do not divide %llu", (unsigned long long)residual_rows, (unsigned long long)dy->rows);
    const uint64_t period = dresidual ? residual_rows : dy->rows;
    NormBackwardJob j{};
    if (dy->rows) {
        j.split = norm_backward_split(dy->rows, dy->cols, period, dresidual != nullptr);
        if (int rc = check_workspace(workspace, workspace_bytes, norm_backward_workspace(j.split, dy->cols, period))) return rc;
    }
    j.rows = dy->rows; j.period = period; j.cols = (uint32_t)dy->cols; j.dtype = dy->dtype;
    j.dy = dy->data; j.dy_ld = dy->ld; j.h = h->data; j.h_ld = h->ld; j.rstd = rstd;
    if (weight) { j.weight = weight->data; j.weight_dtype = weight->dtype; }
    if (dsum) { j.dsum = dsum->data; j.dsum_ld = dsum->ld; }
    if (dx) { j.dx = dx->data; j.dx_ld = dx->ld; }
    j.dresidual = dresidual; j.dweight = dweight;
    return launched(ctx, [&] { launch_rms_norm_backward(j, (float*)workspace, stream_of(ctx, stream)); });
}

extern "C" int dg_dropout(dg_ctx* ctx, void* stream, const dg_matrix* x, double p, uint64_t seed, uint64_t offset, int per_row, const dg_matrix* y) {
    if (int rc = check_ctx(ctx)) return rc;
    if (int rc = check_matrix(x, "x")) return rc;
    if (int rc = check_like(y, "y", x->rows, x->cols, x->dtype)) return rc;
    if (int rc = check_apart(y, "y", x, "x", true)) return rc;
    const double t = p >= 0 && p < 1 ? std::floor(p * 65536 + 0.5) : 65536;
    if (t > 65535) return fail(DG_E_INVALID, "p is in [0, 1) and at most 65535 / 65536");
    const uint64_t indices = x->rows * (per_row ? 1 : x->cols);
    if (indices && offset + (indices - 1) < offset) return fail(DG_E_INVALID, "offset: the indices pass 2^64");
    if (x->rows == 0) return DG_OK;
    const DropoutJob j{x->data, y->data, x->rows, x->cols, x->ld, y->ld, seed, offset, (uint32_t)t, x->dtype, per_row != 0};
    return launched(ctx, [&] { launch_dropout(j, stream_of(ctx, stream)); });
}
