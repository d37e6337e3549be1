// Stand-ins for the kernels of the token rows (see fake_tokens.cpp): launches are counted, the products that gave up stay counted, as they do on a
// device.
#include "../datago_b200/csrc/tokens.h"

static int launches = 0;
static unsigned int gave_up = 0;

extern "C" {
int fake_launches() { int n = launches; launches = 0; return n; }
void fake_gave_up(unsigned int more) { gave_up += more; }
void fake_product_plan(uint64_t m, uint64_t n, uint64_t k, int b_by_column, uint64_t out[6]) {
    const dg::ProductPlan p = dg::plan_product(m, n, k, b_by_column != 0);
    const uint64_t v[6] = {p.splits, p.split_groups, p.together, (uint64_t)p.tiles_m * p.tiles_n, p.slots, p.a_stays};
    for (int i = 0; i < 6; ++i) out[i] = v[i];
}
}

namespace dg {
void launch_patch_rows(const PatchJob&, const dg_rows8*, const dg_matrix*, cudaStream_t) { ++launches; }
void launch_quantize_rows(const dg_matrix&, const dg_rows8&, cudaStream_t) { ++launches; }
void launch_rms_norm(const NormJob&, cudaStream_t) { ++launches; }
void launch_rms_norm_backward(const NormBackwardJob&, float*, cudaStream_t) { ++launches; }
void launch_dropout(const DropoutJob&, cudaStream_t) { ++launches; }
cudaError_t launch_product(const ProductJob&, cudaStream_t) { ++launches; return cudaSuccess; }
cudaError_t product_gave_up(unsigned int* count, cudaStream_t) { *count = gave_up; return cudaSuccess; }
}  // namespace dg
