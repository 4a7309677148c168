#include "skn_paged_attn.cuh"

cudaError_t skn_paged_attn_bf16(const skn_paged *pc, int32_t io, PagedAttn &p) { return attn_by_type<__nv_bfloat16>(pc, io, p); }
