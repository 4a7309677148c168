// Paged KV cache: pools, append with rotation, gather, and the host-pointer forms.
#include "skn_paged.cuh"

#include <math.h>
#include <pthread.h>
#include <new>

// ---- append -------------------------------------------------------------------------------------------------------------
// A CTA takes one token.  Where it goes is looked up and the sines and cosines of its position are formed once, in shared memory (in 64 bits: the angle of
// a far position, and keys that land next to a border of the cache's rounding; queries too: with fp32 sines they are off by 3.8e-8 instead of their own rounding's
// 2.5e-8, and six prompts of 7500 tokens in bf16 take 36.5 us instead of 37.5); its threads take 16 dimensions of a head at a time, eight and the
// eight they turn with, so that the rotation may happen in place.  The rows are requested a unit ahead, the first before all that.
// Bound by HBM from a few thousand tokens on.  8192 tokens of 32 + 2 x 8 heads of 128, all of them turned: bf16 rows and cache 37.5 us (5.4 TB/s), fp32 rows and
// a cache of 4 bits 62.7 us (5.5 TB/s); with requests behind the sines 96 us for the first; with four tokens to a CTA of 256 threads 41.4 and 68.3 us, no faster
// for any smaller step (512 tokens 8.6 us instead of 8.1).  Alone, a token is 3 us of latency.

// sequence of row i: the last one that starts at or before it (-1: none).  Every warp counts the starts for itself: 32 of them at even distances, then
// those between two of these.  (One after the other, 32 at a time, they are a chain of loads as long as the batch.)
__device__ __forceinline__ int paged_find(const PagedStep &st, int i) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = st.n_seqs + 1;                     // starts before lo are at or before i, from hi on they are not
    while (lo < hi) {
        const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step - 1;
        const int n = __popc(__ballot_sync(0xffffffffu, at < hi && st.starts[at] <= i));
        hi = min(hi, lo + (n + 1) * step - 1);
        lo = min(hi, lo + n * step);
    }
    return lo - 1 < st.n_seqs ? lo - 1 : -1;
}

// q of one value: x * fp32(1 / d) + 8.5 in 64 bits, cut off.  The sum with one rounding in fp32 is off by 2^-21 at most, so that 64 bits are
// needed within 2^-18 of a whole number only.
__device__ __forceinline__ uint32_t q4_of(float x, float inv) {
    const float t = fmaf(x, inv, 8.5f);
    int q = (int)t;
    const float f = t - (float)q;
    if (f < 0x1p-18f || f > 1.f - 0x1p-18f) q = (int)__dadd_rn(__dmul_rn((double)x, (double)inv), 8.5);
    return (uint32_t)(q < 0 ? 0 : q > 15 ? 15 : q);
}
// Eight dims of a 32-dim block in each of four neighbouring lanes (all of them here): quants and scale to the page
template <int D> __device__ __forceinline__ void q4_store(uint8_t *page, int page_shift, int row, int block, int quarter, const float (&x)[8]) {
    const int lane = threadIdx.x & 31;
    const unsigned mask = 0xFu << (lane & 28);
    float m = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) m = fabsf(x[i]) > fabsf(m) ? x[i] : m;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {              // of equals the one in the lower lane
        const float y = __shfl_xor_sync(mask, m, o);
        m = fabsf(y) > fabsf(m) || (fabsf(y) == fabsf(m) && (lane & o)) ? y : m;
    }
    const float d = m / -8.f, inv = d != 0.f ? 1.f / d : 0.f;
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        lo |= q4_of(x[i], inv) << (8 * i);
        hi |= q4_of(x[4 + i], inv) << (8 * i);
    }
    const uint32_t lo2 = __shfl_down_sync(mask, lo, 2, 4), hi2 = __shfl_down_sync(mask, hi, 2, 4);
    if (quarter < 2) *reinterpret_cast<uint2 *>(page + (((block << page_shift) + row) << 4) + 8 * quarter) = make_uint2(lo | (lo2 << 4), hi | (hi2 << 4));
    if (quarter == 0) *reinterpret_cast<__half *>(page + ((D / 2) << page_shift) + (row * (D / 32) + block) * 2) = __float2half_rn(d);
}

struct PagedRows {                                     // rows of the step's tokens
    const void *k, *v, *q;
    void *q_out;
    int64_t k_stride, v_stride, q_stride, q_out_stride;
    int q_heads, rot, halves;
    const double *turns;
    uint8_t *k_pool, *v_pool;
};

// Row ranges that go back: the search above may miss every row of such a sequence, so each CTA looks at some by itself, with a warp that does not search
__device__ __forceinline__ void paged_order(const PagedStep &st) {
    for (int s = blockIdx.x * 32 + (threadIdx.x & 31); s < st.n_seqs; s += gridDim.x * 32)
        if (st.starts[s] > st.starts[s + 1]) *st.status = SKN_ERR_ARG;
}

struct PagedPlace { int pos, page, row; };             // of a token: its position (negative: nowhere), page (negative: none) and row of the page
// by a whole warp
__device__ __forceinline__ PagedPlace paged_place(const PagedStep &st, int i) {
    PagedPlace at = {-1, -1, 0};
    const int s = i < st.n_tokens ? paged_find(st, i) : -1;
    if (s < 0) return at;
    const PagedSeq q = paged_seq(st, s);
    if (i < q.first || i >= q.first + q.n) return at;
    at.pos = q.len - q.n + i - q.first;
    if (at.pos >= 0) {
        at.page = paged_page(st, s, at.pos);
        at.row = at.pos & ((1 << st.page_shift) - 1);
    }
    return at;
}

// eight dimensions and the eight they turn with, in 64 bits; c: the unit of 16.  Pair 8 c + i lies at [i][c]: the units of a
// head are neighbouring lanes (at [8 c + i] they met in the same banks: with four tokens to a CTA 8192 of them took 52 us instead of 43)
template <int UNITS> __device__ __forceinline__ void paged_turn(float (&x)[8], float (&y)[8], const double2 *turn, int c, bool halves) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (halves) {
            const double2 t = turn[j * UNITS + c];
            const double a = x[j], b = y[j];
            x[j] = (float)(a * t.x - b * t.y);
            y[j] = (float)(a * t.y + b * t.x);
        } else if (!(j & 1)) {
            const double2 t = turn[(j >> 1) * UNITS + c], w = turn[(4 + (j >> 1)) * UNITS + c];
            const double x0 = x[j], x1 = x[j + 1], y0 = y[j], y1 = y[j + 1];
            x[j] = (float)(x0 * t.x - x1 * t.y);
            x[j + 1] = (float)(x0 * t.y + x1 * t.x);
            y[j] = (float)(y0 * w.x - y1 * w.y);
            y[j + 1] = (float)(y0 * w.y + y1 * w.x);
        }
    }
}

// eight elements as they lie in memory
template <class IO> struct IoRow8 {
    float f[8];
    __device__ __forceinline__ void load(const IO *p) { io_load8(p, f); }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = f[i];
    }
};
template <> struct IoRow8<__nv_bfloat16> {
    uint4 u;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { u = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
};

template <class CT, int D, class IO>
__global__ void __launch_bounds__(128, 8) skn_paged_append_kernel(const PagedStep st, const PagedRows r) {
    constexpr bool Q4 = sizeof(CT) == 1;
    constexpr int THREADS = 128, UNITS = D / 16;
    extern __shared__ float staged[];                  // Q4: the rotated keys, [heads][D]
    __shared__ double2 turn[D / 2];
    __shared__ PagedPlace place;
    const int tid = threadIdx.x, n_units = (r.q_heads + (Q4 ? 1 : 2) * st.heads) * UNITS;
    const int64_t t = blockIdx.x;
    // where a unit's 16 dimensions are: head < 0: of the queries; from st.heads on: of the values
    auto find = [&](int u, int &head, int &c, int &a, int &b) {
        head = u / UNITS - r.q_heads;
        c = u % UNITS;
        const bool turned = 16 * c < r.rot && head < st.heads;
        a = turned && r.halves ? c : 2 * c;
        b = turned && r.halves ? c + r.rot / 16 : 2 * c + 1;
        return turned;
    };
    IoRow8<IO> x, y;
    auto request = [&](int u) {
        if (u < n_units) {
            int head, c, a, b;
            find(u, head, c, a, b);
            const IO *src = head < 0            ? static_cast<const IO *>(r.q) + t * r.q_stride + (head + r.q_heads) * D
                            : head < st.heads ? static_cast<const IO *>(r.k) + t * r.k_stride + head * D
                                              : static_cast<const IO *>(r.v) + t * r.v_stride + (head - st.heads) * D;
            x.load(src + 8 * a);
            y.load(src + 8 * b);
        }
    };
    request(tid);
    if (tid < 32) {
        const PagedPlace found = paged_place(st, blockIdx.x);
        if (tid == 0) place = found;
    } else if (tid < 64) paged_order(st);
    __syncthreads();
    const PagedPlace at = place;
    if (at.pos < 0) return;
    for (int i = tid; i < r.rot / 2; i += THREADS) {
        double2 x;
        sincospi((double)at.pos * r.turns[i], &x.y, &x.x);
        turn[(i & 7) * UNITS + (i >> 3)] = x;
    }
    __syncthreads();
    for (int u = tid; u < n_units; u += THREADS) {
        int head, c, a, b;
        const bool turned = find(u, head, c, a, b);
        float xf[8], yf[8];
        x.get(xf);
        y.get(yf);
        request(u + THREADS);
        if (head >= 0 && at.page < 0) continue;
        if (turned) paged_turn<UNITS>(xf, yf, turn, c, r.halves);
        if (head < 0) {
            IO *to = static_cast<IO *>(r.q_out) + t * r.q_out_stride + (head + r.q_heads) * D;
            io_store8(to + 8 * a, xf);
            io_store8(to + 8 * b, yf);
        } else if constexpr (Q4) {
            io_store8(staged + head * D + 8 * a, xf);
            io_store8(staged + head * D + 8 * b, yf);
        } else {
            CT *to = reinterpret_cast<CT *>(head < st.heads ? r.k_pool + paged_at(st, at.page, head) : r.v_pool + paged_at(st, at.page, head - st.heads)) + at.row * D;
            io_store8(to + 8 * a, xf);
            io_store8(to + 8 * b, yf);
        }
    }
    if constexpr (Q4) {
        __syncthreads();
        // four neighbouring lanes per block of 32 dims; the bound is a multiple of four, so they stay together
        if (at.page < 0) return;
        for (int u = tid; u < 2 * st.heads * (D / 8); u += THREADS) {
            const int head = u / (D / 8), c = u % (D / 8);
            float z[8];
            if (head < st.heads) io_load8(staged + head * D + 8 * c, z);
            else io_load8(static_cast<const IO *>(r.v) + t * r.v_stride + (head - st.heads) * D + 8 * c, z);
            uint8_t *to = head < st.heads ? r.k_pool + paged_at(st, at.page, head) : r.v_pool + paged_at(st, at.page, head - st.heads);
            q4_store<D>(to, st.page_shift, at.row, c >> 2, c & 3, z);
        }
    }
}

// ---- gather ---------------------------------------------------------------------------------------------------------------
// A CTA takes one token here too: 8192 of 2 x 8 heads of 128 to fp32 rows from bf16 21.6 us (4.7 TB/s), from 4 bits 20.7 us (3.7 TB/s: the look-up and the loads of a token
// follow one another)
template <class CT, int D, class IO>
__global__ void __launch_bounds__(256) skn_paged_gather_kernel(const PagedStep st, const uint8_t *k_pool, const uint8_t *v_pool, IO *k_out, IO *v_out) {
    __shared__ PagedPlace place;
    if (threadIdx.x < 32) {
        const PagedPlace found = paged_place(st, blockIdx.x);
        if (threadIdx.x == 0) place = found;
    } else if (threadIdx.x < 64) paged_order(st);
    __syncthreads();
    const PagedPlace at = place;
    if (at.page < 0) return;
    for (int u = threadIdx.x; u < 2 * st.heads * (D / 8); u += 256) {
        const int head = u / (D / 8), c = u % (D / 8);
        const bool is_v = head >= st.heads;
        const int h = is_v ? head - st.heads : head;
        float x[8];
        paged_load8<D>(reinterpret_cast<const CT *>((is_v ? v_pool : k_pool) + paged_at(st, at.page, h)), st.page_shift, at.row, c, x);
        io_store8((is_v ? v_out : k_out) + ((int64_t)blockIdx.x * st.heads + h) * D + 8 * c, x);
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------
bool skn_paged_ok(const skn_paged *pc) { return pc && pc->magic == SKN_MAGIC_PAGED && skn_ctx_ok(pc->ctx); }

static int32_t check_spec(skn_ctx *ctx, const skn_paged_spec *s) {
    if (!s) return skn_fail(ctx, SKN_ERR_ARG, "NULL specification");
    if (s->kv_dtype != SKN_KV_F16 && s->kv_dtype != SKN_KV_BF16 && s->kv_dtype != SKN_KV_Q4_0)
        return skn_fail(ctx, SKN_ERR_TYPE, "a paged cache holds fp16, bf16 or Q4_0, not element type %d", s->kv_dtype);
    if (s->n_kv_heads < 1 || s->n_kv_heads > PAGED_MAX_HEADS || s->n_pages < 1) return skn_fail(ctx, SKN_ERR_ARG, "pages and heads (at most %d) must be positive", PAGED_MAX_HEADS);
    if (s->head_dim != 64 && s->head_dim != 128) return skn_fail(ctx, SKN_ERR_SHAPE, "head_dim must be 64 or 128 (got %d)", s->head_dim);
    if (s->page_tokens != 16 && s->page_tokens != 32 && s->page_tokens != 64 && s->page_tokens != 128)
        return skn_fail(ctx, SKN_ERR_SHAPE, "a page holds 16, 32, 64 or 128 tokens, not %d", s->page_tokens);
    if (s->rot_dims < 0 || s->rot_dims > s->head_dim || s->rot_dims % 16)
        return skn_fail(ctx, SKN_ERR_SHAPE, "rot_dims must be a multiple of 16 up to head_dim (got %d)", s->rot_dims);
    if (s->rot_pairs != SKN_ROT_ADJACENT && s->rot_pairs != SKN_ROT_HALVES) return skn_fail(ctx, SKN_ERR_ARG, "unknown pairing %d", s->rot_pairs);
    if (s->rot_dims && !(s->rot_base > 0 && isfinite(s->rot_base))) return skn_fail(ctx, SKN_ERR_ARG, "rot_base must be positive");
    return SKN_OK;
}
static int64_t page_head_bytes(const skn_paged_spec *s) {
    return (int64_t)s->page_tokens * (s->kv_dtype == SKN_KV_Q4_0 ? s->head_dim / 2 + s->head_dim / 16 : 2 * s->head_dim);
}
static int64_t pool_bytes_of(const skn_paged_spec *s) { return page_head_bytes(s) * s->n_kv_heads * s->n_pages; }

// the parts of a step that the host can see; SKN_OK with *nothing where there is no row
static int32_t check_batch(skn_ctx *ctx, const skn_paged_batch *b, bool *nothing, bool host = false) {
    if (!b) return skn_fail(ctx, SKN_ERR_ARG, "NULL batch");
    if (b->n_seqs < 0 || b->n_tokens < 0 || b->max_new < 0 || b->max_pages < 0) return skn_fail(ctx, SKN_ERR_ARG, "negative count in the batch");
    *nothing = b->n_seqs == 0 || b->n_tokens == 0 || (b->max_new == 0 && !host);
    if (*nothing) return SKN_OK;
    if (b->n_tokens > (1 << 24)) return skn_fail(ctx, SKN_ERR_SHAPE, "%d rows in a step; 2^24 at most", b->n_tokens);
    if (b->n_seqs > 65535) return skn_fail(ctx, SKN_ERR_SHAPE, "%d sequences in a step; 65535 at most", b->n_seqs);
    if (b->max_pages > (1 << 23)) return skn_fail(ctx, SKN_ERR_SHAPE, "%d pages a sequence; 2^23 at most", b->max_pages);
    if (!b->token_start || !b->lengths || (!b->page_table && b->max_pages)) return skn_fail(ctx, SKN_ERR_ARG, "NULL array in the batch");
    return SKN_OK;
}
static int32_t check_rows(skn_ctx *ctx, const char *what, const void *p, int64_t stride, int64_t width, int32_t io) {
    const int per = io == SKN_KV_F32 ? 4 : 8;
    if (!p) return skn_fail(ctx, SKN_ERR_ARG, "%s is NULL", what);
    if (((uintptr_t)p & 15) || stride % per) return skn_fail(ctx, SKN_ERR_ALIGN, "%s: rows must be 16-byte aligned", what);
    if (stride < width) return skn_fail(ctx, SKN_ERR_SHAPE, "%s: rows of %lld elements are %lld apart", what, (long long)width, (long long)stride);
    return SKN_OK;
}
// whether rows of a and b meet in memory (side by side in wider rows of one length they do not)
static bool rows_meet(int64_t n, int32_t io, const void *a, int64_t a_stride, int64_t a_width, const void *b, int64_t b_stride, int64_t b_width) {
    const int64_t size = io == SKN_KV_F32 ? 4 : 2;
    const uintptr_t p = (uintptr_t)a, q = (uintptr_t)b;
    if (p >= q + ((n - 1) * b_stride + b_width) * size || q >= p + ((n - 1) * a_stride + a_width) * size) return false;
    if (a_stride != b_stride) return true;
    const int64_t row = a_stride * size, behind = q >= p ? (int64_t)((q - p) % (uintptr_t)row) : (row - (int64_t)((p - q) % (uintptr_t)row)) % row;
    return behind < a_width * size || behind + b_width * size > row;
}
static int32_t check_heads(skn_ctx *ctx, const skn_paged *pc, int32_t n_q_heads) {
    if (n_q_heads < 1 || n_q_heads % pc->spec.n_kv_heads) return skn_fail(ctx, SKN_ERR_SHAPE, "Shapes do not align.");
    if (n_q_heads / pc->spec.n_kv_heads > 64) return skn_fail(ctx, SKN_ERR_SHAPE, "%d query heads per kv head; 64 at most", n_q_heads / pc->spec.n_kv_heads);
    return SKN_OK;
}
static int32_t check_mask(skn_ctx *ctx, float scale, int32_t window, int32_t sinks) {
    if (window < 0 || sinks < 0) return skn_fail(ctx, SKN_ERR_ARG, "negative window or sinks");
    if (!isfinite(scale * PAGED_LOG2E)) return skn_fail(ctx, SKN_ERR_ARG, "a scale of %g: times log2(e) it is no number", scale);
    return SKN_OK;
}
static int32_t check_io(skn_ctx *ctx, int32_t io) {
    if (io != SKN_KV_F32 && io != SKN_KV_BF16) return skn_fail(ctx, SKN_ERR_TYPE, "rows are fp32 or bf16, not element type %d", io);
    return SKN_OK;
}

template <class CT, int D, class IO> static cudaError_t append_launch(const PagedStep &st, const PagedRows &r, int device, cudaStream_t stream) {
    const size_t smem = sizeof(CT) == 1 ? (size_t)st.heads * D * sizeof(float) : 0;
    auto *kern = skn_paged_append_kernel<CT, D, IO>;
    if (smem > 32000) {
        static uint64_t done = 0;
        const cudaError_t e = paged_attributes(kern, (size_t)PAGED_MAX_HEADS * D * sizeof(float), device, &done);
        if (e != cudaSuccess) return e;
    }
    kern<<<st.n_tokens, 128, smem, stream>>>(st, r);
    return cudaGetLastError();
}
template <class CT, int D, class IO> static cudaError_t gather_launch(const PagedStep &st, const skn_paged *pc, void *k, void *v, cudaStream_t stream) {
    skn_paged_gather_kernel<CT, D, IO><<<st.n_tokens, 256, 0, stream>>>(st, pc->k, pc->v, static_cast<IO *>(k), static_cast<IO *>(v));
    return cudaGetLastError();
}
#define PAGED_BY_IO(fn, CT, D, ...) (io == SKN_KV_F32 ? fn<CT, D, float>(__VA_ARGS__) : fn<CT, D, __nv_bfloat16>(__VA_ARGS__))
#define PAGED_BY_DIM(fn, CT, ...) (pc->spec.head_dim == 64 ? PAGED_BY_IO(fn, CT, 64, __VA_ARGS__) : PAGED_BY_IO(fn, CT, 128, __VA_ARGS__))
#define PAGED_BY_TYPE(fn, ...)                                                                   \
    (pc->spec.kv_dtype == SKN_KV_F16    ? PAGED_BY_DIM(fn, __half, __VA_ARGS__)                   \
     : pc->spec.kv_dtype == SKN_KV_BF16 ? PAGED_BY_DIM(fn, __nv_bfloat16, __VA_ARGS__)            \
                                        : PAGED_BY_DIM(fn, skn_q4, __VA_ARGS__))

static int32_t append_run(skn_paged *pc, const skn_paged_batch *b, int32_t io, const PagedRows &r) {
    SKN_CUDA(pc->ctx, PAGED_BY_TYPE(append_launch, paged_step(pc, b), r, pc->ctx->device, pc->ctx->stream));
    return SKN_OK;
}

// ---- host-pointer forms: the step's arrays are checked here, so a mistake is answered before anything has run -----------------------
enum { NEED_ROWS, NEED_SEEN };
// What a step reads of the tables: the pages of its rows' positions (NEED_ROWS), or of all that their queries see.  once: no row is written twice.
static int32_t check_tables(skn_paged *pc, const skn_paged_batch *b, int need, int32_t window, int32_t sinks, bool once) {
    skn_ctx *ctx = pc->ctx;
    const int P = pc->spec.page_tokens;
    uint8_t *taken = nullptr;
    if (once) {
        taken = new (std::nothrow) uint8_t[((size_t)pc->spec.n_pages * P + 7) / 8]();
        if (!taken) return skn_fail(ctx, SKN_ERR_OOM, "host allocation failed");
    }
    int32_t rc = SKN_OK;
    for (int s = 0; s < b->n_seqs && rc == SKN_OK; ++s) {
        const int64_t a = b->token_start[s], e = b->token_start[s + 1], len = b->lengths[s];
        if (a < 0 || e < a || e > b->n_tokens || e - a > b->max_new || len < 0) {
            rc = skn_fail(ctx, SKN_ERR_ARG, "sequence %d: rows %lld to %lld of %d, length %lld", s, (long long)a, (long long)e, b->n_tokens, (long long)len);
            break;
        }
        if (e == a) continue;
        if (len > (int64_t)b->max_pages * P) {
            rc = skn_fail(ctx, SKN_ERR_SHAPE, "sequence %d: %lld tokens in %d pages of %d", s, (long long)len, b->max_pages, P);
            break;
        }
        const int64_t first = len - (e - a) > 0 ? len - (e - a) : 0;      // position of the first row that is no padding
        const int64_t from = need == NEED_ROWS ? first : !window ? 0 : first - window + 1 > 0 ? first - window + 1 : 0;
        for (int64_t p = 0; p < len; p += P) {
            const int64_t last = p + P < len ? p + P : len;
            if (last <= from && !(need == NEED_SEEN && window && p < sinks)) continue;
            const int page = b->page_table[(int64_t)s * b->max_pages + p / P];
            if (page < 0 || page >= pc->spec.n_pages) {
                rc = skn_fail(ctx, SKN_ERR_ARG, "sequence %d: page %d of position %lld is none of %d", s, page, (long long)p, pc->spec.n_pages);
                break;
            }
            for (int64_t t = p > first ? p : first; once && t < last; ++t) {
                const size_t at = (size_t)page * P + (t - p);
                if (taken[at >> 3] >> (at & 7) & 1) {
                    rc = skn_fail(ctx, SKN_ERR_ARG, "sequence %d: row %d of page %d is written twice", s, (int)(t - p), page);
                    break;
                }
                taken[at >> 3] |= (uint8_t)(1 << (at & 7));
            }
            if (rc) break;
        }
    }
    delete[] taken;
    return rc;
}

struct HostStep {                                       // the step's arrays and rows on the device, in the context's scratch
    skn_paged_batch b;
    float *rows[4];
};
// n_rows arrays of width[i] floats per token, those with a host pointer filled; the outputs start as what the caller's hold
static int32_t stage_step(skn_paged *pc, const skn_paged_batch *b, int n_rows, const int64_t *width, const float *const *host, HostStep *h) {
    skn_ctx *ctx = pc->ctx;
    const size_t n_table = (size_t)b->n_seqs * b->max_pages;
    const size_t ints = (n_table + 2 * (size_t)b->n_seqs + 1 + 63) / 64 * 64;
    size_t bytes = ints * 4;
    for (int i = 0; i < n_rows; ++i) bytes += (size_t)b->n_tokens * width[i] * 4;
    const int32_t rc = skn_stage_reserve(ctx, &ctx->d_scratch, &ctx->d_scratch_bytes, bytes);
    if (rc) return rc;
    int32_t *d = static_cast<int32_t *>(ctx->d_scratch);
    h->b = *b;
    h->b.page_table = d;
    h->b.token_start = d + n_table;
    h->b.lengths = d + n_table + b->n_seqs + 1;
    if (n_table) SKN_CUDA(ctx, cudaMemcpyAsync(d, b->page_table, n_table * 4, cudaMemcpyHostToDevice, ctx->stream));
    SKN_CUDA(ctx, cudaMemcpyAsync(d + n_table, b->token_start, (b->n_seqs + 1) * 4, cudaMemcpyHostToDevice, ctx->stream));
    SKN_CUDA(ctx, cudaMemcpyAsync(d + n_table + b->n_seqs + 1, b->lengths, b->n_seqs * 4, cudaMemcpyHostToDevice, ctx->stream));
    float *at = reinterpret_cast<float *>(d + ints);
    for (int i = 0; i < n_rows; ++i) {
        h->rows[i] = at;
        if (host[i]) SKN_CUDA(ctx, cudaMemcpyAsync(at, host[i], (size_t)b->n_tokens * width[i] * 4, cudaMemcpyHostToDevice, ctx->stream));
        at += (size_t)b->n_tokens * width[i];
    }
    return SKN_OK;
}
static int32_t enter_host(skn_paged *pc, const skn_paged_batch *b, bool *nothing) {
    const int32_t rc = check_batch(pc->ctx, b, nothing, true);
    if (rc || *nothing) return rc;
    SKN_CUDA(pc->ctx, cudaSetDevice(pc->ctx->device));
    return SKN_OK;
}

// ---- after a wait that ran out ------------------------------------------------------------------------------------------------------
// A prompt kernel that gives up leaves some of its joins' counters above zero, and the next launch, a captured one too, would join too early.  So
// a report of the status, which every caller gets before it can trust a result again, zeroes the counters of the context's caches.
static pthread_mutex_t caches_lock = PTHREAD_MUTEX_INITIALIZER;
static skn_paged *caches;
static void tickets_back(skn_ctx *ctx) {
    pthread_mutex_lock(&caches_lock);
    cudaDeviceSynchronize();                            // (graphs may run on other streams than the context's)
    for (skn_paged *pc = caches; pc; pc = pc->next)
        if (pc->ctx == ctx) cudaMemsetAsync(pc->d_tickets, 0, paged_ticket_bytes(pc), ctx->stream);
    pthread_mutex_unlock(&caches_lock);
}
static void caches_add(skn_paged *pc) {
    pthread_mutex_lock(&caches_lock);
    pc->next = caches;
    caches = pc;
    pthread_mutex_unlock(&caches_lock);
    pc->ctx->after_failure = tickets_back;
}
static void caches_remove(const skn_paged *pc) {
    pthread_mutex_lock(&caches_lock);
    for (skn_paged **at = &caches; *at; at = &(*at)->next)
        if (*at == pc) {
            *at = pc->next;
            break;
        }
    pthread_mutex_unlock(&caches_lock);
}

extern "C" {

int32_t skn_paged_pool_bytes(const skn_paged_spec *spec, int64_t *bytes) {
    const int32_t rc = check_spec(nullptr, spec);
    if (rc) return rc;
    if (!bytes) return skn_fail(nullptr, SKN_ERR_ARG, "bytes is NULL");
    *bytes = pool_bytes_of(spec);
    return SKN_OK;
}

int32_t skn_paged_create(skn_ctx *ctx, const skn_paged_spec *spec, void *k_pool_dev, void *v_pool_dev, skn_paged **out) {
    if (!skn_ctx_ok(ctx)) return skn_fail(nullptr, SKN_ERR_BAD_HANDLE, "bad context handle");
    SKN_ENTER(ctx);
    if (!out) return skn_fail(ctx, SKN_ERR_ARG, "out is NULL");
    *out = nullptr;
    const int32_t rc = check_spec(ctx, spec);
    if (rc) return rc;
    if ((int64_t)spec->n_pages * spec->n_kv_heads * spec->page_tokens > INT32_MAX)
        return skn_fail(ctx, SKN_ERR_SHAPE, "%d pages of %d tokens and %d heads are more than 2^31 rows", spec->n_pages, spec->page_tokens, spec->n_kv_heads);
    if (!k_pool_dev != !v_pool_dev) return skn_fail(ctx, SKN_ERR_ARG, "one pool is NULL");
    if (((uintptr_t)k_pool_dev | (uintptr_t)v_pool_dev) & 15) return skn_fail(ctx, SKN_ERR_ALIGN, "pools must be 16-byte aligned");
    const uintptr_t ka = (uintptr_t)k_pool_dev, va = (uintptr_t)v_pool_dev;
    if (k_pool_dev && (ka < va ? va - ka : ka - va) < (uintptr_t)pool_bytes_of(spec)) return skn_fail(ctx, SKN_ERR_ARG, "one pool lies over the other");
    skn_paged *pc = new (std::nothrow) skn_paged();
    if (!pc) return skn_fail(ctx, SKN_ERR_OOM, "host allocation failed");
    pc->magic = SKN_MAGIC_PAGED;
    pc->ctx = ctx;
    pc->spec = *spec;
    for (pc->page_shift = 4; (1 << pc->page_shift) < spec->page_tokens;) ++pc->page_shift;
    pc->head_bytes = page_head_bytes(spec);
    pc->pool_bytes = pool_bytes_of(spec);
    pc->owns = !k_pool_dev;
    pc->k = static_cast<uint8_t *>(k_pool_dev);
    pc->v = static_cast<uint8_t *>(v_pool_dev);
    double turns[64];
    for (int i = 0; i < spec->rot_dims / 2; ++i) turns[i] = pow(spec->rot_base, -2.0 * i / spec->rot_dims) / 3.14159265358979323846;
    cudaError_t e = cudaSetDevice(ctx->device);
    if (pc->owns) {
        if (e == cudaSuccess) e = cudaMalloc((void **)&pc->k, pc->pool_bytes);
        if (e == cudaSuccess) e = cudaMalloc((void **)&pc->v, pc->pool_bytes);
        if (e == cudaSuccess) e = cudaMemsetAsync(pc->k, 0, pc->pool_bytes, ctx->stream);
        if (e == cudaSuccess) e = cudaMemsetAsync(pc->v, 0, pc->pool_bytes, ctx->stream);
    }
    if (e == cudaSuccess) e = cudaMalloc((void **)&pc->d_turns, sizeof(turns));
    if (e == cudaSuccess) e = cudaMemcpyAsync(pc->d_turns, turns, sizeof(turns), cudaMemcpyHostToDevice, ctx->stream);
    if (e == cudaSuccess) e = skn_paged_attn_prepare(pc);
    if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);
    if (e != cudaSuccess) {
        skn_paged_destroy(pc);
        return skn_check_cuda(ctx, e, "paged cache allocation");
    }
    caches_add(pc);
    *out = pc;
    return SKN_OK;
}

int32_t skn_paged_destroy(skn_paged *pc) {
    if (!pc || pc->magic != SKN_MAGIC_PAGED) return skn_fail(nullptr, SKN_ERR_BAD_HANDLE, "bad paged cache handle");
    caches_remove(pc);
    if (skn_ctx_ok(pc->ctx)) {
        cudaSetDevice(pc->ctx->device);
        cudaStreamSynchronize(pc->ctx->stream);
    }
    if (pc->owns) {
        if (pc->k) cudaFree(pc->k);
        if (pc->v) cudaFree(pc->v);
    }
    if (pc->d_turns) cudaFree(pc->d_turns);
    if (pc->d_parts) cudaFree(pc->d_parts);
    if (pc->d_tickets) cudaFree(pc->d_tickets);
    pc->magic = 0;
    delete pc;
    return SKN_OK;
}

int32_t skn_paged_info(const skn_paged *pc, void **k_pool_dev, void **v_pool_dev, int64_t *pool_bytes) {
    if (!skn_paged_ok(pc)) return skn_fail(nullptr, SKN_ERR_BAD_HANDLE, "bad paged cache handle");
    if (k_pool_dev) *k_pool_dev = pc->k;
    if (v_pool_dev) *v_pool_dev = pc->v;
    if (pool_bytes) *pool_bytes = pc->pool_bytes;
    return SKN_OK;
}

int32_t skn_paged_append_dev(skn_paged *pc, const skn_paged_batch *batch, int32_t io, const void *k_dev, int64_t k_stride, const void *v_dev,
                             int64_t v_stride, const void *q_dev, int64_t q_stride, int32_t n_q_heads, void *q_out_dev, int64_t q_out_stride) {
    if (!skn_paged_ok(pc)) return skn_fail(nullptr, SKN_ERR_BAD_HANDLE, "bad paged cache handle");
    skn_ctx *ctx = pc->ctx;
    SKN_ENTER(ctx);
    bool nothing;
    int32_t rc = check_io(ctx, io);
    if (rc || (rc = check_batch(ctx, batch, &nothing)) || nothing) return rc;
    const int64_t w = (int64_t)pc->spec.n_kv_heads * pc->spec.head_dim;
    if ((rc = check_rows(ctx, "k", k_dev, k_stride, w, io)) || (rc = check_rows(ctx, "v", v_dev, v_stride, w, io))) return rc;
    if (q_dev) {
        const int64_t wq = (int64_t)n_q_heads * pc->spec.head_dim;
        if ((rc = check_heads(ctx, pc, n_q_heads)) || (rc = check_rows(ctx, "q", q_dev, q_stride, wq, io)) ||
            (rc = check_rows(ctx, "q_out", q_out_dev, q_out_stride, wq, io)))
            return rc;
        // tokens are turned side by side: only a row's own place may be written to
        const int32_t n = batch->n_tokens;
        if ((q_out_dev != q_dev || (q_out_stride != q_stride && n > 1)) && rows_meet(n, io, q_dev, q_stride, wq, q_out_dev, q_out_stride, wq))
            return skn_fail(ctx, SKN_ERR_ARG, "q_out lies over q, but is not q");
        if (rows_meet(n, io, k_dev, k_stride, w, q_out_dev, q_out_stride, wq) || rows_meet(n, io, v_dev, v_stride, w, q_out_dev, q_out_stride, wq))
            return skn_fail(ctx, SKN_ERR_ARG, "q_out lies over k or v");
    }
    SKN_CUDA(ctx, cudaSetDevice(ctx->device));
    return append_run(pc, batch, io, PagedRows{k_dev, v_dev, q_dev, q_out_dev, k_stride, v_stride, q_stride, q_out_stride, q_dev ? n_q_heads : 0,
                                               pc->spec.rot_dims, pc->spec.rot_pairs == SKN_ROT_HALVES, pc->d_turns, pc->k, pc->v});
}

int32_t skn_paged_append(skn_paged *pc, const skn_paged_batch *batch, const float *k_host, const float *v_host, const float *q_host,
                         int32_t n_q_heads, float *q_out_host) {
    if (!skn_paged_ok(pc)) return skn_fail(nullptr, SKN_ERR_BAD_HANDLE, "bad paged cache handle");
    skn_ctx *ctx = pc->ctx;
    SKN_ENTER(ctx);
    bool nothing;
    int32_t rc = enter_host(pc, batch, &nothing);
    if (rc || nothing) return rc;
    if (!k_host || !v_host || !q_host != !q_out_host) return skn_fail(ctx, SKN_ERR_ARG, "NULL argument");
    if (q_host && (rc = check_heads(ctx, pc, n_q_heads))) return rc;
    if ((rc = check_tables(pc, batch, NEED_ROWS, 0, 0, true)) || batch->max_new == 0) return rc;
    const int64_t w = (int64_t)pc->spec.n_kv_heads * pc->spec.head_dim, wq = q_host ? (int64_t)n_q_heads * pc->spec.head_dim : 0;
    const int64_t width[4] = {w, w, wq, wq};
    const float *host[4] = {k_host, v_host, q_host, q_out_host};
    HostStep h;
    if ((rc = stage_step(pc, batch, 4, width, host, &h))) return rc;
    if ((rc = append_run(pc, &h.b, SKN_KV_F32, PagedRows{h.rows[0], h.rows[1], h.rows[2], h.rows[3], w, w, wq, wq, q_host ? n_q_heads : 0,
                                                         pc->spec.rot_dims, pc->spec.rot_pairs == SKN_ROT_HALVES, pc->d_turns, pc->k, pc->v})))
        return rc;
    const skn_result r = {q_out_host, h.rows[3], (size_t)batch->n_tokens * wq * 4};
    return skn_sync_results(ctx, &r, q_host ? 1 : 0);
}

int32_t skn_paged_gather_dev(skn_paged *pc, const skn_paged_batch *batch, int32_t io, void *k_out_dev, void *v_out_dev) {
    if (!skn_paged_ok(pc)) return skn_fail(nullptr, SKN_ERR_BAD_HANDLE, "bad paged cache handle");
    skn_ctx *ctx = pc->ctx;
    SKN_ENTER(ctx);
    bool nothing;
    int32_t rc = check_io(ctx, io);
    if (rc || (rc = check_batch(ctx, batch, &nothing)) || nothing) return rc;
    if ((rc = check_rows(ctx, "k_out", k_out_dev, 16, 0, io)) || (rc = check_rows(ctx, "v_out", v_out_dev, 16, 0, io))) return rc;
    const int64_t w = (int64_t)pc->spec.n_kv_heads * pc->spec.head_dim;
    if (rows_meet(batch->n_tokens, io, k_out_dev, w, w, v_out_dev, w, w)) return skn_fail(ctx, SKN_ERR_ARG, "k_out lies over v_out");
    SKN_CUDA(ctx, cudaSetDevice(ctx->device));
    SKN_CUDA(ctx, PAGED_BY_TYPE(gather_launch, paged_step(pc, batch), pc, k_out_dev, v_out_dev, ctx->stream));
    return SKN_OK;
}

int32_t skn_paged_gather(skn_paged *pc, const skn_paged_batch *batch, float *k_out_host, float *v_out_host) {
    if (!skn_paged_ok(pc)) return skn_fail(nullptr, SKN_ERR_BAD_HANDLE, "bad paged cache handle");
    skn_ctx *ctx = pc->ctx;
    SKN_ENTER(ctx);
    bool nothing;
    int32_t rc = enter_host(pc, batch, &nothing);
    if (rc || nothing) return rc;
    if (!k_out_host || !v_out_host) return skn_fail(ctx, SKN_ERR_ARG, "NULL argument");
    if ((rc = check_tables(pc, batch, NEED_ROWS, 0, 0, false)) || batch->max_new == 0) return rc;
    const int64_t w = (int64_t)pc->spec.n_kv_heads * pc->spec.head_dim;
    const int64_t width[2] = {w, w};
    const float *host[2] = {k_out_host, v_out_host};
    HostStep h;
    if ((rc = stage_step(pc, batch, 2, width, host, &h))) return rc;
    const int32_t io = SKN_KV_F32;
    SKN_CUDA(ctx, PAGED_BY_TYPE(gather_launch, paged_step(pc, &h.b), pc, h.rows[0], h.rows[1], ctx->stream));
    const size_t bytes = (size_t)batch->n_tokens * w * 4;
    const skn_result r[2] = {{k_out_host, h.rows[0], bytes}, {v_out_host, h.rows[1], bytes}};
    return skn_sync_results(ctx, r, 2);
}

int32_t skn_paged_attn_dev(skn_paged *pc, const skn_paged_batch *batch, int32_t io, const void *q_dev, int64_t q_stride, int32_t n_q_heads,
                           float scale, int32_t window, int32_t sinks, void *out_dev, int64_t out_stride) {
    if (!skn_paged_ok(pc)) return skn_fail(nullptr, SKN_ERR_BAD_HANDLE, "bad paged cache handle");
    skn_ctx *ctx = pc->ctx;
    SKN_ENTER(ctx);
    bool nothing;
    int32_t rc = check_io(ctx, io);
    if (rc || (rc = check_batch(ctx, batch, &nothing)) || (rc = check_heads(ctx, pc, n_q_heads))) return rc;
    if ((rc = check_mask(ctx, scale, window, sinks))) return rc;
    if (nothing) return SKN_OK;
    const int64_t wq = (int64_t)n_q_heads * pc->spec.head_dim;
    if ((rc = check_rows(ctx, "q", q_dev, q_stride, wq, io)) || (rc = check_rows(ctx, "out", out_dev, out_stride, wq, io))) return rc;
    // outputs are written while other rows' queries are still to be read, and a query is asked for again where a result is not finite
    if (rows_meet(batch->n_tokens, io, q_dev, q_stride, wq, out_dev, out_stride, wq)) return skn_fail(ctx, SKN_ERR_ARG, "out lies over q");
    SKN_CUDA(ctx, cudaSetDevice(ctx->device));
    return skn_paged_attn_launch(pc, batch, io, q_dev, q_stride, n_q_heads, scale, window, window ? sinks : 0, out_dev, out_stride);
}

int32_t skn_paged_attn(skn_paged *pc, const skn_paged_batch *batch, const float *q_host, int32_t n_q_heads, float scale, int32_t window,
                       int32_t sinks, float *out_host) {
    if (!skn_paged_ok(pc)) return skn_fail(nullptr, SKN_ERR_BAD_HANDLE, "bad paged cache handle");
    skn_ctx *ctx = pc->ctx;
    SKN_ENTER(ctx);
    bool nothing;
    int32_t rc = enter_host(pc, batch, &nothing);
    if (rc || (rc = check_heads(ctx, pc, n_q_heads))) return rc;
    if ((rc = check_mask(ctx, scale, window, sinks))) return rc;
    if (nothing) return SKN_OK;
    if (!q_host || !out_host) return skn_fail(ctx, SKN_ERR_ARG, "NULL argument");
    if ((rc = check_tables(pc, batch, NEED_SEEN, window, sinks, false)) || batch->max_new == 0) return rc;
    const int64_t wq = (int64_t)n_q_heads * pc->spec.head_dim;
    const int64_t width[2] = {wq, wq};
    const float *host[2] = {q_host, out_host};
    HostStep h;
    if ((rc = stage_step(pc, batch, 2, width, host, &h))) return rc;
    if ((rc = skn_paged_attn_launch(pc, &h.b, SKN_KV_F32, h.rows[0], wq, n_q_heads, scale, window, window ? sinks : 0, h.rows[1], wq))) return rc;
    const skn_result r = {out_host, h.rows[1], (size_t)batch->n_tokens * wq * 4};
    return skn_sync_results(ctx, &r, 1);
}

}  // extern "C"
