// The paged KV cache: what its translation units share (skn_paged.cu: pools, append, gather, host forms; skn_paged_attn.cu: attention).
#pragma once
#include "skn_internal.cuh"

#include <cuda.h>
#include <type_traits>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#define SKN_MAGIC_PAGED 0x736b6e70u   // 'sknp'

struct skn_paged {
    uint32_t magic;
    skn_ctx *ctx;
    skn_paged_spec spec;
    int page_shift;              // page_tokens = 1 << page_shift
    bool owns;                   // the pools are this cache's
    uint8_t *k, *v;
    int64_t head_bytes;          // one page of one head
    int64_t pool_bytes;
    double *d_turns;             // [rot_dims / 2] half turns per position
    // Attention's workspace (skn_paged_attn.cu): tensor maps of the pools and, for rows whose keys several CTAs share, their partial results
    CUtensorMap map[4];          // K, V; of Q4_0 their quants, then their scales
    CUtensorMap wide[4];         // the same in larger boxes (prompts): whole pages of half rows; of Q4_0 up to 32 rows
    int n_parts;                 // CTAs that share a launch's work, at most
    float *d_parts;              // prompts: blocks of rows of two segments per SM; then (from prompt_parts on) decoding, two per CTA: [rows of a CTA's segment][head_dim + 4]:
    int64_t prompt_parts;        // output, maximum, sum
    unsigned *d_tickets;         // [2][2 n_parts], zero between launches (a launch that gave up: from the report of it on, skn_paged.cu)
    skn_paged *next;             // of all caches
};
constexpr int SKN_PAGED_PART_ROWS = 32;
constexpr int PAGED_MAX_HEADS = 256;         // kv heads
constexpr float PAGED_LOG2E = 1.4426950408889634f;        // scores are formed in base 2

// A step as the kernels see it
struct PagedStep {
    const int32_t *table, *starts, *lens;
    int32_t n_seqs, n_tokens, max_new, max_pages;
    int32_t heads, page_shift, n_pages;
    int64_t head_bytes;
    int32_t *status;
};
static inline PagedStep paged_step(const skn_paged *pc, const skn_paged_batch *b) {
    // (no sequence has more rows than the step: a bound that says nothing makes no larger grid)
    return PagedStep{b->page_table, b->token_start, b->lengths, b->n_seqs, b->n_tokens, b->max_new < b->n_tokens ? b->max_new : b->n_tokens, b->max_pages,
                     pc->spec.n_kv_heads, pc->page_shift, pc->spec.n_pages, pc->head_bytes, pc->ctx->d_status};
}

#ifdef __CUDACC__
// One sequence of the step.  What the caller's arrays say of it is checked here, once per kernel: a sequence that does not fit the
// step or its page table has no rows (and is reported).
struct PagedSeq { int first, n, len; };
__device__ __forceinline__ PagedSeq paged_seq(const PagedStep &st, int s) {
    const int a = st.starts[s], b = st.starts[s + 1], len = st.lens[s];
    PagedSeq q = {a, b - a, len};
    if (a < 0 || b < a || b > st.n_tokens || b - a > st.max_new || len < 0 || (int64_t)len > ((int64_t)st.max_pages << st.page_shift)) {
        *st.status = SKN_ERR_ARG;
        q.n = 0;
    }
    return q;
}
// page of a position that lies in the table; -1 (and a report) where the table holds none
__device__ __forceinline__ int paged_page(const PagedStep &st, int s, int pos) {
    const int page = st.table[(int64_t)s * st.max_pages + (pos >> st.page_shift)];
    if ((unsigned)page < (unsigned)st.n_pages) return page;
    *st.status = SKN_ERR_ARG;
    return -1;
}
__device__ __forceinline__ int64_t paged_at(const PagedStep &st, int page, int head) { return ((int64_t)page * st.heads + head) * st.head_bytes; }

// rows of fp32 or bf16, eight elements at a time
__device__ __forceinline__ void io_load8(const float *p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void io_load8(const __nv_bfloat16 *p, float (&x)[8]) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ uint32_t io_pack(__nv_bfloat16, float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t io_pack(__half, float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void io_store8(float *p, const float (&x)[8]) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
template <class T> __device__ __forceinline__ void io_store8(T *p, const float (&x)[8]) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(io_pack(T(), x[0], x[1]), io_pack(T(), x[2], x[3]), io_pack(T(), x[4], x[5]), io_pack(T(), x[6], x[7]));
}

// Cached rows.  `at`: a page of one head; dims 8 c .. 8 c + 7 of its row r, D = head_dim
struct skn_q4 { uint8_t b; };
template <int D> __device__ __forceinline__ void paged_load8(const __nv_bfloat16 *at, int, int r, int c, float (&x)[8]) { io_load8(at + r * D + 8 * c, x); }
template <int D> __device__ __forceinline__ void paged_load8(const __half *at, int, int r, int c, float (&x)[8]) {
    const uint4 u = *reinterpret_cast<const uint4 *>(at + r * D + 8 * c);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
template <int D> __device__ __forceinline__ void paged_load8(const skn_q4 *at, int page_shift, int r, int c, float (&x)[8]) {
    const uint8_t *p = reinterpret_cast<const uint8_t *>(at);
    const uint2 u = *reinterpret_cast<const uint2 *>(p + ((((c >> 2) << page_shift) + r) << 4) + ((c & 1) << 3));
    const float d = __half2float(*reinterpret_cast<const __half *>(p + ((D / 2) << page_shift) + (r * (D / 32) + (c >> 2)) * 2));
    const int sh = (c & 2) << 1;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)((int)((((i < 4 ? u.x : u.y) >> (8 * (i & 3) + sh)) & 15u)) - 8) * d;
}
// one dimension
template <int D, class CT> __device__ __forceinline__ float paged_load1(const CT *at, int page_shift, int r, int d) {
    if constexpr (std::is_same<CT, __nv_bfloat16>::value) return __bfloat162float(at[r * D + d]);
    else if constexpr (std::is_same<CT, __half>::value) return __half2float(at[r * D + d]);
    else {
        const uint8_t *p = reinterpret_cast<const uint8_t *>(at);
        const int q = p[((((d >> 5) << page_shift) + r) << 4) + (d & 15)] >> (d & 16 ? 4 : 0) & 15;
        return (float)(q - 8) * __half2float(*reinterpret_cast<const __half *>(p + ((D / 2) << page_shift) + (r * (D / 32) + (d >> 5)) * 2));
    }
}

// a kernel's largest dynamic shared memory, once per kernel and device (`done`: a bit each; setting it twice does no harm, but two contexts share the
// setting: it is the most that any cache asks for)
template <class K> static cudaError_t paged_attributes(K *kern, size_t smem, int device, uint64_t *done) {
    if (device < 64 && __atomic_load_n(done, __ATOMIC_RELAXED) >> device & 1) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess && device < 64) __atomic_fetch_or(done, (uint64_t)1 << device, __ATOMIC_RELAXED);
    return e;
}
#endif

static inline size_t paged_ticket_bytes(const skn_paged *pc) { return (size_t)4 * pc->n_parts * sizeof(unsigned); }

bool skn_paged_ok(const skn_paged *pc);
cudaError_t skn_paged_attn_prepare(skn_paged *pc);
// attention over `batch` (device arrays) on the context's stream; arguments checked by the caller
int32_t skn_paged_attn_launch(skn_paged *pc, const skn_paged_batch *batch, int32_t io, const void *q, int64_t q_stride, int32_t n_q_heads, float scale,
                              int32_t window, int32_t sinks, void *out, int64_t out_stride);
