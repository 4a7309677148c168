// Attention over the paged KV cache.
#include "skn_paged.cuh"

#include <math.h>

// One row (a token's query head) at a time, straight from the definition: a CTA takes the row's visible keys 128 at a time, a thread per key
// for the scores and a thread per dimension for the sum of values, with a running maximum and sum.  Nothing of a key that the row
// does not see is read.
constexpr int PLAIN_THREADS = 128;

template <class CT, int D, class IO>
__global__ void __launch_bounds__(PLAIN_THREADS) skn_paged_plain_kernel(const PagedStep st, const uint8_t *k_pool, const uint8_t *v_pool, const IO *q, int64_t q_stride,
                                                                       int group, float scale, int window, int sinks, IO *out, int64_t out_stride) {
    __shared__ float qs[D], ps[PLAIN_THREADS], red[8];
    __shared__ const uint8_t *at[PLAIN_THREADS];
    const int head = blockIdx.y, s = blockIdx.z, tid = threadIdx.x;
    const PagedSeq sq = paged_seq(st, s);
    for (int t = blockIdx.x; t < sq.n; t += gridDim.x) {
        const int pos = sq.len - sq.n + t;
        IO *o = out + (int64_t)(sq.first + t) * out_stride + head * D;
        __syncthreads();
        if (tid < D / 8) {
            float x[8];
            io_load8(q + (int64_t)(sq.first + t) * q_stride + head * D + 8 * tid, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) qs[8 * tid + i] = x[i];
        }
        __syncthreads();
        float m = -INFINITY, l = 0.f, acc = 0.f;
        const int lo = window ? max(0, pos - window + 1) : 0, first = min(sinks, lo);      // visible: 0 .. first - 1 and lo .. pos
        const int n = pos < 0 ? 0 : first + pos + 1 - lo;
        for (int b = 0; b < n; b += PLAIN_THREADS) {
            const int i = b + tid, p = i < first ? i : lo + i - first;
            float z = -INFINITY;
            const uint8_t *row = nullptr;
            if (i < n) {
                const int page = paged_page(st, s, p), r = p & ((1 << st.page_shift) - 1);
                if (page >= 0) {
                    const int64_t base = paged_at(st, page, head / group);
                    float dot[8] = {};                  // eight short sums: 16 roundings each, not 128
                    for (int c = 0; c < D / 8; ++c) {
                        float x[8];
                        paged_load8<D>(reinterpret_cast<const CT *>(k_pool + base), st.page_shift, r, c, x);
#pragma unroll
                        for (int j = 0; j < 8; ++j) dot[j] = fmaf(x[j], qs[8 * c + j], dot[j]);
                    }
                    z = (((dot[0] + dot[1]) + (dot[2] + dot[3])) + ((dot[4] + dot[5]) + (dot[6] + dot[7]))) * scale;
                    row = v_pool + base;
                }
            }
            at[tid] = row;
            float top = z;
#pragma unroll
            for (int o2 = 16; o2; o2 >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o2));
            if ((tid & 31) == 0) red[tid >> 5] = top;
            __syncthreads();
            top = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
            const float base = top == -INFINITY ? 0.f : top, fix = expf(m - base);
            const float w = row ? expf(z - base) : 0.f;
            ps[tid] = w;
            float sum = w;
#pragma unroll
            for (int o2 = 16; o2; o2 >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o2);
            if ((tid & 31) == 0) red[4 + (tid >> 5)] = sum;
            __syncthreads();
            l = l * fix + red[4] + red[5] + red[6] + red[7];
            acc *= fix;
            m = top;
            if (tid < D) {
                const int here = min(PLAIN_THREADS, n - b);
                for (int j = 0; j < here; ++j) {
                    if (!at[j]) continue;
                    const int pj = b + j < first ? b + j : lo + b + j - first;
                    float x[8];
                    paged_load8<D>(reinterpret_cast<const CT *>(at[j]), st.page_shift, pj & ((1 << st.page_shift) - 1), tid >> 3, x);
                    float v = x[0];
#pragma unroll
                    for (int e = 1; e < 8; ++e) v = (tid & 7) == e ? x[e] : v;
                    acc = fmaf(ps[j], v, acc);
                }
            }
            __syncthreads();
        }
        if (tid < D) ps[tid] = n > 0 ? acc / l : 0.f;      // (a NaN among the visible scores reaches l)
        __syncthreads();
        if (tid < D / 8) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = ps[8 * tid + i];
            io_store8(o + 8 * tid, x);
        }
    }
}

template <class CT, int D, class IO>
static cudaError_t plain_launch(const skn_paged *pc, const PagedStep &st, const void *q, int64_t q_stride, int n_q_heads, float scale, int window, int sinks, void *out,
                                int64_t out_stride) {
    const dim3 grid((unsigned)(st.max_new < 4096 ? st.max_new : 4096), (unsigned)n_q_heads, (unsigned)st.n_seqs);
    skn_paged_plain_kernel<CT, D, IO><<<grid, PLAIN_THREADS, 0, pc->ctx->stream>>>(st, pc->k, pc->v, static_cast<const IO *>(q), q_stride,
                                                                                   n_q_heads / pc->spec.n_kv_heads, scale, window, sinks, static_cast<IO *>(out), out_stride);
    return cudaGetLastError();
}
template <class CT, int D> static cudaError_t plain_by_io(int32_t io, const skn_paged *pc, const PagedStep &st, const void *q, int64_t qs, int nq, float sc, int w, int si, void *o, int64_t os) {
    return io == SKN_KV_F32 ? plain_launch<CT, D, float>(pc, st, q, qs, nq, sc, w, si, o, os) : plain_launch<CT, D, __nv_bfloat16>(pc, st, q, qs, nq, sc, w, si, o, os);
}
template <class CT> static cudaError_t plain_by_dim(int32_t io, const skn_paged *pc, const PagedStep &st, const void *q, int64_t qs, int nq, float sc, int w, int si, void *o, int64_t os) {
    return pc->spec.head_dim == 64 ? plain_by_io<CT, 64>(io, pc, st, q, qs, nq, sc, w, si, o, os) : plain_by_io<CT, 128>(io, pc, st, q, qs, nq, sc, w, si, o, os);
}

int32_t skn_paged_attn_launch(skn_paged *pc, const skn_paged_batch *batch, int32_t io, const void *q, int64_t q_stride, int32_t n_q_heads, float scale,
                              int32_t window, int32_t sinks, void *out, int64_t out_stride) {
    const PagedStep st = paged_step(pc, batch);
    auto *by = pc->spec.kv_dtype == SKN_KV_F16 ? plain_by_dim<__half> : pc->spec.kv_dtype == SKN_KV_BF16 ? plain_by_dim<__nv_bfloat16> : plain_by_dim<skn_q4>;
    SKN_CUDA(pc->ctx, by(io, pc, st, q, q_stride, n_q_heads, scale, window, sinks, out, out_stride));
    return SKN_OK;
}
