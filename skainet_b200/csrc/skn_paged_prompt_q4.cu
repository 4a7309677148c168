#include "skn_paged_prompt.cuh"

cudaError_t skn_paged_prompt(skn_q4, const skn_paged *pc, const PagedAttn &p) {
    return pc->spec.head_dim == 64 ? prompt_launch<skn_q4, 64>(pc, p) : prompt_launch<skn_q4, 128>(pc, p);
}
