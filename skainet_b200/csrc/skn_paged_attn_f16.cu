#include "skn_paged_attn.cuh"

cudaError_t skn_paged_attn_f16(const skn_paged *pc, int32_t io, PagedAttn &p) { return attn_by_type<__half>(pc, io, p); }
