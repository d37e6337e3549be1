// Launch interface between the token entry points (tokens.cu) and their kernels.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include "../../include/datago_b200.h"

namespace dg {

constexpr uint32_t kScaleGroup = 128;  // columns of 8-bit rows that share a scale
inline uint64_t scale_groups(uint64_t cols) { return (cols + kScaleGroup - 1) / kScaleGroup; }

constexpr uint32_t kTokenSms = 148;    // of a B200

// ---- 8-bit rows (kernels_tokens.cu) ---------------------------------------------------------------------------------
struct PatchJob {
    const uint8_t* pixels;
    uint32_t n, h, w, channels, patch;
    float gain[4], shift[4];  // value = pixel * gain + shift
};
void launch_patch_rows(const PatchJob& job, const dg_rows8* out8, const dg_matrix* out, cudaStream_t s);
void launch_quantize_rows(const dg_matrix& src, const dg_rows8& out, cudaStream_t s);

// ---- norm (kernels_tokens.cu) -----------------------------------------------------------------------------------------
constexpr uint64_t kNormMaxCols = 16384;
struct NormJob {
    uint64_t rows;
    uint32_t cols, residual_rows;
    int32_t dtype, weight_dtype;
    const void *x, *residual, *weight;
    uint64_t x_ld, residual_ld, sum_ld, y_ld;
    void *sum, *y;
    dg_rows8 y8;  // values NULL: none
    float* rstd;
    float eps;
};
void launch_rms_norm(const NormJob& job, cudaStream_t s);

// How the rows of the backward pass are dealt out: row_threads threads work on a row, cta_workers rows of threads make a CTA.
constexpr uint32_t kNormChunk = 16;  // neighbouring rows that a worker takes at a time, where no images share a residual row
struct NormBackwardSplit {
    uint32_t row_threads, cta_workers, ctas;
    uint32_t parts;  // that the images of a residual row are split into
    bool by_image;   // images share residual rows, and their gradient is wanted
};
NormBackwardSplit norm_backward_split(uint64_t rows, uint64_t cols, uint64_t period, bool residual);
inline uint64_t norm_backward_workspace(const NormBackwardSplit& d, uint64_t cols, uint64_t period) {
    return 4 * cols * ((uint64_t)d.ctas * d.cta_workers + (d.parts > 1 ? d.parts * period : 0));
}
struct NormBackwardJob {
    uint64_t rows, period;   // period: rows of dresidual
    uint32_t cols;
    int32_t dtype, weight_dtype;
    const void *dy, *h, *weight, *dsum;
    const float* rstd;
    uint64_t dy_ld, h_ld, dsum_ld, dx_ld;
    void* dx;
    float *dresidual, *dweight;
    NormBackwardSplit split;
};
void launch_rms_norm_backward(const NormBackwardJob& job, float* workspace, cudaStream_t s);

// ---- dropout (kernels_tokens.cu) ----------------------------------------------------------------------------------------
struct DropoutJob {
    const void* x;
    void* y;
    uint64_t rows, cols, x_ld, y_ld, seed, offset;
    uint32_t threshold;  // of 65536
    int32_t dtype;
    bool per_row;
};
void launch_dropout(const DropoutJob& job, cudaStream_t s);

// ---- product (kernels_product.cu) ------------------------------------------------------------------------------------------
// Tiles of 256 x at most 256; up to 224 columns a tile's sums leave tensor memory while the next tile's are made.
constexpr uint32_t kProductTileM = 256, kProductMaxTileN = 256, kProductTwoSums = 224;
constexpr uint32_t kProductPartGroups = 64;              // of a part of the contraction, at most
constexpr uint64_t kProductPartsBytes = 512ull << 20;    // of the workspace for parts that are made together (one part may be larger)
constexpr uint32_t kProductRingBytes = 192 * 1024, kProductABytes = kProductTileM / 2 * 128, kProductSlots = 6;
struct ProductPlan {
    uint32_t tile_n;           // columns of an output tile, a multiple of 32
    uint32_t tiles_m, tiles_n;
    uint32_t splits, split_groups;  // the contraction is cut into `splits` parts of split_groups groups of 128
    uint32_t together;              // parts of a launch: all, or as many as the workspace has room for beside the sum of those before them
    uint32_t sums;                  // accumulators
    uint32_t slots;                 // of 256 columns each, of the ring of b, and of a unless it stays
    bool a_stays;                   // all groups of a row of tiles have room
};
ProductPlan plan_product(uint64_t m, uint64_t n, uint64_t k, bool b_by_column);
inline uint64_t product_part_ld(uint64_t n) { return (n + 3) / 4 * 4; }
inline uint64_t product_workspace(const ProductPlan& p, uint64_t m, uint64_t n) {
    return p.splits > 1 ? (uint64_t)(p.together + (p.together < p.splits)) * m * product_part_ld(n) * 4 : 0;
}
struct ProductJob {
    // boxes of 128 bytes x 128 (a), tile_n / 2 (b) or, of an operand by column, 128 lines, 128-byte swizzle; of 64 bytes x 32 rows x 1 part, 64-byte swizzle
    CUtensorMap a, b, out_map;
    const uint8_t *a_scales, *b_scales;
    uint64_t a_scale_ld, b_scale_ld, m, n, k, ld;
    uint32_t a_block, b_block;
    bool a_by_column, b_by_column;
    uint64_t map_cols;  // columns that leave through out_map; 0: none
    void* out;
    int32_t dtype;
    float* parts;
    ProductPlan plan;
    uint32_t first_group;  // of the parts of a launch
};
cudaError_t launch_product(const ProductJob& job, cudaStream_t s);
cudaError_t product_gave_up(unsigned int* count, cudaStream_t s);  // waits for the stream; CTAs on the current device since the process began

}  // namespace dg
