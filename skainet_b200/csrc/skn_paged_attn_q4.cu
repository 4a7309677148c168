#include "skn_paged_attn.cuh"

cudaError_t skn_paged_attn_q4(const skn_paged *pc, int32_t io, PagedAttn &p) { return attn_by_type<skn_q4>(pc, io, p); }
