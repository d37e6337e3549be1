// Stand-ins for the kernels of the token rows, for tests of their entry points (csrc/tokens.cpp) without a GPU: a launch is counted.
#include "../datago_b200/csrc/tokens.h"

static int launches = 0;
static unsigned int gave_up = 0;

extern "C" {
int fake_launches() { int n = launches; launches = 0; return n; }
void fake_gave_up(unsigned int n) { gave_up = n; }
void fake_product_plan(uint64_t m, uint64_t n, uint64_t k, int b_by_column, uint32_t out[8]) {
    const dg::ProductPlan p = dg::plan_product(m, n, k, b_by_column != 0);
    const uint32_t v[8] = {p.tile_n, p.tiles_m, p.tiles_n, p.splits, p.split_groups, p.sums, p.slots, p.a_stays};
    for (int i = 0; i < 8; ++i) out[i] = v[i];
}
void fake_backward_split(uint64_t rows, uint64_t cols, uint64_t period, int residual, uint32_t out[2]) {
    const dg::NormBackwardSplit d = dg::norm_backward_split(rows, cols, period, residual != 0);
    out[0] = d.ctas * d.cta_workers;
    out[1] = d.parts;
}
}

namespace dg {
void launch_patch_rows(const PatchJob&, const dg_rows8*, const dg_matrix*, cudaStream_t) { ++launches; }
void launch_quantize_rows(const dg_matrix&, const dg_rows8&, cudaStream_t) { ++launches; }
void launch_rms_norm(const NormJob&, cudaStream_t) { ++launches; }
void launch_rms_norm_backward(const NormBackwardJob&, float*, cudaStream_t) { ++launches; }
void launch_dropout(const DropoutJob&, cudaStream_t) { ++launches; }
cudaError_t launch_product(const ProductJob&, cudaStream_t) { ++launches; return cudaSuccess; }
cudaError_t product_gave_up(unsigned int* count, cudaStream_t) { *count = gave_up; gave_up = 0; return cudaSuccess; }
}  // namespace dg
