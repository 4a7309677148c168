// Attention over the paged KV cache: tensor maps, workspace and the choice of the kernel.
#include "skn_paged_prompt.cuh"

// ---- launches ---------------------------------------------------------------------------------------------------------------
static cudaError_t encode(CUtensorMap *map, CUtensorMapDataType type, int rank, void *base, const cuuint64_t *dim, const cuuint64_t *stride, const cuuint32_t *box,
                          CUtensorMapSwizzle swizzle) {
    skn_encode_tiled_fn fn = nullptr;
    const cudaError_t e = skn_tmap_encoder(&fn);
    if (e != cudaSuccess) return e;
    const cuuint32_t one[3] = {1, 1, 1};
    const CUresult r = fn(map, type, (cuuint32_t)rank, base, dim, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t skn_paged_attn_prepare(skn_paged *pc) {
    const skn_paged_spec &s = pc->spec;
    const int D = s.head_dim, P = s.page_tokens;
    cudaError_t e = cudaSuccess;
    for (int i = 0; i < 2 && e == cudaSuccess; ++i) {
        uint8_t *pool = i ? pc->v : pc->k;
        const cuuint64_t heads = (cuuint64_t)s.n_pages * s.n_kv_heads;
        if (s.kv_dtype != SKN_KV_Q4_0) {
            // 16 rows, each half of 128 bytes by itself: [D / 64][16][64], swizzled
            const cuuint64_t dim[3] = {64, heads * P, (cuuint64_t)D / 64}, stride[2] = {(cuuint64_t)D * 2, 128};
            const cuuint32_t box[3] = {64, 16, (cuuint32_t)D / 64};
            e = encode(&pc->map[i], CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, pool, dim, stride, box, CU_TENSOR_MAP_SWIZZLE_128B);
            const cuuint32_t whole[3] = {64, (cuuint32_t)P, 1};
            if (e == cudaSuccess) e = encode(&pc->wide[i], CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, pool, dim, stride, whole, CU_TENSOR_MAP_SWIZZLE_128B);
        } else {
            // quants of 16 rows (wide: up to 32), in words: [D / 32][rows][4]; scales [rows][D / 32], two to a word
            for (int w = 0; w < 2 && e == cudaSuccess; ++w) {
                const cuuint32_t rows = w && P > 16 ? 32 : 16;
                CUtensorMap *to = w ? pc->wide : pc->map;
                const cuuint64_t dim[3] = {(cuuint64_t)P * 4, (cuuint64_t)D / 32, heads}, stride[2] = {(cuuint64_t)P * 16, (cuuint64_t)pc->head_bytes};
                const cuuint32_t box[3] = {rows * 4, (cuuint32_t)D / 32, 1};
                e = encode(&to[i], CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, pool, dim, stride, box, CU_TENSOR_MAP_SWIZZLE_NONE);
                const cuuint64_t sdim[2] = {(cuuint64_t)P * D / 64, heads}, sstride[1] = {(cuuint64_t)pc->head_bytes};
                const cuuint32_t sbox[2] = {rows * (cuuint32_t)D / 64, 1};
                if (e == cudaSuccess) e = encode(&to[2 + i], CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, pool + (size_t)P * D / 2, sdim, sstride, sbox, CU_TENSOR_MAP_SWIZZLE_NONE);
            }
        }
    }
    pc->n_parts = 4 * pc->ctx->sm_count;
    const size_t row = (D + 4) * sizeof(float), decode_rows = (size_t)2 * pc->ctx->sm_count * SKN_PAGED_PART_ROWS, prompt_rows = (size_t)2 * pc->ctx->sm_count * PP_ROWS;
    const size_t tickets = paged_ticket_bytes(pc);
    pc->prompt_parts = (int64_t)(prompt_rows * (D + 4));
    if (e == cudaSuccess) e = cudaMalloc((void **)&pc->d_parts, (decode_rows + prompt_rows) * row);
    if (e == cudaSuccess) e = cudaMalloc((void **)&pc->d_tickets, tickets);
    if (e == cudaSuccess) e = cudaMemsetAsync(pc->d_tickets, 0, tickets, pc->ctx->stream);
    return e;
}

int32_t skn_paged_attn_launch(skn_paged *pc, const skn_paged_batch *batch, int32_t io, const void *q, int64_t q_stride, int32_t n_q_heads, float scale,
                              int32_t window, int32_t sinks, void *out, int64_t out_stride) {
    PagedAttn p = {};
    p.st = paged_step(pc, batch);
    p.k_pool = pc->k; p.v_pool = pc->v;
    p.q = q; p.out = out;
    p.q_stride = q_stride; p.out_stride = out_stride;
    p.group = n_q_heads / pc->spec.n_kv_heads;
    // a window that reaches back over any table's tokens is none
    p.window = window >= (int64_t)batch->max_pages * pc->spec.page_tokens ? 0 : window;
    p.sinks = p.window ? sinks : 0;
    p.scale = scale * PAGED_LOG2E;
    p.parts = pc->d_parts;
    p.tickets = pc->d_tickets;
    SKN_CUDA(pc->ctx, pc->spec.kv_dtype == SKN_KV_F16    ? skn_paged_attn_f16(pc, io, p)
                      : pc->spec.kv_dtype == SKN_KV_BF16 ? skn_paged_attn_bf16(pc, io, p)
                                                         : skn_paged_attn_q4(pc, io, p));
    return SKN_OK;
}
