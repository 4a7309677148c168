#include "skn_paged_prompt.cuh"

cudaError_t skn_paged_prompt(__half, const skn_paged *pc, const PagedAttn &p) {
    return pc->spec.head_dim == 64 ? prompt_launch<__half, 64>(pc, p) : prompt_launch<__half, 128>(pc, p);
}
