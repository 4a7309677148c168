#include "skn_paged_prompt.cuh"

cudaError_t skn_paged_prompt(__nv_bfloat16, const skn_paged *pc, const PagedAttn &p) {
    return pc->spec.head_dim == 64 ? prompt_launch<__nv_bfloat16, 64>(pc, p) : prompt_launch<__nv_bfloat16, 128>(pc, p);
}
