// Attention over the paged KV cache: rows of few tokens (decoding), and every row of fp32.  A translation unit per cache type.
//
// Work.  A segment is a sequence's new rows (up to 8 NB of them: tokens x query heads of one kv head) over the keys that some of them sees,
// in units of 16 (fp16, bf16) or 32 (Q4_0) keys.  The units of all segments form one line, which the CTAs share out evenly, so that a batch of
// unequal lengths keeps every SM at work to the end; a segment that lies in several CTAs leaves partial results (maximum, sum,
// unnormalised output), which the last of them to finish joins in order.
//
// A unit.  Each of a CTA's warps (four for up to eight rows, else eight) takes every fourth or eighth unit through a ring of its own, filled by TMA.  S^T = K q^T with mma.sync (m16n8k16: 16 keys
// x 8 rows): keys are the operand of 16 so that up to eight query heads waste nothing.  Scores go through one running maximum per row that
// moves only when a weight would exceed 2^SLACK (one vote a unit instead of six shuffles).  Weights are transposed by movmatrix into the second
// operand of O^T = V^T p^T.  A product takes operands of one type, the cache's (Q4_0: fp16).  fp32 rows: queries and weights as sums of two fp16 (fp16 and Q4_0 caches) or three
// bf16 terms.  bf16 rows: queries in one term, weights in one of fp16, whose rounding an output's own hides (relative errors of 1.66e-3 either way), or in two of bf16: with one
// 2.2e-3, 48 sequences with a window of 4096 133 us instead of 134.
// The tensor cores cut their sums off instead of rounding them, so for these rows the small terms have an accumulator of their own, the large ones
// two for the scores, and a unit's output is formed from zero and added in fp32.
//
// Q4_0.  K: a nibble masked out of a word is an fp16 subnormal, q 2^-24 (or 16 q 2^-24), which the tensor cores multiply exactly, so quants need
// no conversion; one accumulator per block of 32 dims starts at -8 sum q and is scaled by the key's d.  V: weights are multiplied by the
// key's d of the block, in fp16 relative to a power of two 2^E that follows the largest d, and meet q - 8 (one packed instruction for two): with
// the 8 taken off at the end, a dimension of zeros would come out as the rounding of two large sums.
//
// Infinities and NaN.  Scores of hidden keys are replaced, not added to.  A hidden row of V meets a weight of zero, and zero times infinity is no
// zero: in units with hidden keys, rows that nobody sees are cleared if they are not finite.  Whatever else goes wrong with such values
// (a key that some rows see and others do not; an infinity that meets the two terms of a weight) leaves a result that is not finite,
// and a segment with one is computed again straight from the definition (paged_redo).
//
// 16-bit caches are bound by HBM: 16 sequences of 8192 tokens, 32 / 8 heads of 128, fp16 pages 97 us for fp32 rows and 95 us for bf16 ones (5.5 and 5.7 TB/s, 0.86 of a copy's
// rate), bf16 pages 99 and 96, 48 sequences with a window of 4096 134 us (6.0 TB/s).  Q4_0: 64 sequences of 16384, bf16 rows, 393 us (3.1 TB/s; 60 % of the
// issue slots, the ALU pipe at 57 %: masks, permutes and conversions of V; neither is at its end), 16 of 8192 71 us, with fp32 rows, two terms of everything, 103.  One sequence
// of 100 tokens is 8 us of latency, 1024 of one's 4100 20 us in a graph.  Shares smaller than the CTAs that run at a time (twice as many) cost 95 -> 101 us: every share has a beginning.
#pragma once
#include "skn_paged.cuh"
#include "skn_mma.cuh"
#include "skn_tc.cuh"

#include <math.h>

// Sequences whose work is shared out: as many as have room for their places in shared memory; a step of more takes a CTA per segment.  That is the room's border, not one of
// speed: 300 sequences of 1000 tokens each take 195 us shared out and 183 as CTAs, 510 of 500 and one of 32768 198 us, 600 and that one (as CTAs) 558.
constexpr int PA_MAX_SEQS = 512;
constexpr float PA_NONE = -3.402823466e38f;  // running maximum before the first score: the lowest number, so that no score is below it

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d = a b + c
__device__ __forceinline__ void mma_f16_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %10, %11};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ float pa_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// a b from zero
template <class CT> __device__ __forceinline__ void mma_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<CT, __nv_bfloat16>::value) mma_bf16_first(d, a, b0, b1);
    else mma_f16_from(d, a, b0, b1, 0.f, 0.f);
}
template <class CT> __device__ __forceinline__ void mma_as(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<CT, __nv_bfloat16>::value) mma_bf16(c, a, b0, b1);
    else mma_f16(c, a, b0, b1);
}
// o += a b, b in NT terms, small ones first; fp32 rows: from zero, and then added
template <class CT, bool EX, int NT> __device__ __forceinline__ void pa_add(float (&o)[4], const uint32_t (&a)[4], const uint32_t (&b)[NT][2]) {
    if constexpr (EX) {
        float x[4];
        mma_zero<CT>(x, a, b[NT - 1][0], b[NT - 1][1]);
#pragma unroll
        for (int n = NT - 2; n >= 0; --n) mma_as<CT>(x, a, b[n][0], b[n][1]);
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] += x[c];
    } else {
#pragma unroll
        for (int n = NT - 1; n >= 0; --n) mma_as<CT>(o, a, b[n][0], b[n][1]);
    }
}
__device__ __forceinline__ uint32_t movm(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// two values -> NT packed terms of the product's type
template <class CT, int NT> __device__ __forceinline__ void terms_of(float x, float y, uint32_t (&w)[NT]) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        if constexpr (std::is_same<CT, __nv_bfloat16>::value) {
            w[i] = pack_bf16(x, y);
            if (i + 1 < NT) less_bf16(x, y, w[i]);
        } else {
            w[i] = pack_f16(x, y);
            if (i + 1 < NT) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                x -= f.x;
                y -= f.y;
            }
        }
    }
}
__device__ __forceinline__ void tma_3d(void *dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(skn_smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(skn_smem_u32(bar))
                 : "memory");
}

struct PagedAttn {
    PagedStep st;
    const uint8_t *k_pool, *v_pool;
    const void *q;
    void *out;
    int64_t q_stride, out_stride;
    int group, window, sinks;
    float scale;                  // times log2(e)
    int direct;                   // a CTA per segment: no sharing (rows in blocks of 8 NB)
    int above, upto;              // sequences of other numbers of rows (tokens x group) are left to another launch
    int split;                    // ... which follows this one, or is this one: it begins while that one ends
    float *parts;
    unsigned *tickets;
};

// The keys that a segment's rows see, as units: 0 .. a - 1 (first tokens), then from unit a + gap on
struct PagedSpan { int units, a, gap; };
__device__ __forceinline__ PagedSpan paged_span(const PagedAttn &p, int pmin, int pmax, int unit) {
    const int lo = p.window ? max(0, max(0, pmin) - p.window + 1) : 0;
    const int a = (min(p.sinks, lo) + unit - 1) / unit, b = lo / unit;
    PagedSpan s = {(pmax + unit) / unit, 0, 0};
    if (pmax < 0) s.units = 1;                       // rows without a key still have an output
    if (p.window && b > a) {
        s.a = a;
        s.gap = b - a;
        s.units -= s.gap;
    }
    return s;
}
__device__ __forceinline__ bool paged_sees(const PagedAttn &p, int key, int pos) {
    return key <= pos && (!p.window || key > pos - p.window || key < p.sinks);
}

// A sequence's rows for this launch
__device__ __forceinline__ PagedSeq paged_mine(const PagedAttn &p, int s) {
    PagedSeq q = paged_seq(p.st, s);
    const int rows = q.n * p.group;                  // (at most 2^30)
    if (rows <= p.above || rows > p.upto) q.n = 0;
    return q;
}

struct PagedSegment {
    int seq, head, first, rows, row0;     // its rows of the step: token first + r / group, query head head * group + r % group, r = row0 ..
    int n, len;                           // of the sequence
    PagedSpan span;
    int u0, u1;                           // this CTA's units
    int c0, n_parts, slot;                // CTAs that have some of it: c0 .. c0 + n_parts - 1
};

// a / b of numbers that are not negative (a division in 64 bits takes several hundred cycles, and a launch of few units is some thousands)
__device__ __forceinline__ long long paged_div(long long a, long long b) {
    return (a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}
// Where a CTA leaves its part of a segment that others share: a CTA ends in at most one such segment and begins in at most one
__device__ __forceinline__ int paged_slot(const PagedSegment &g, int cta) { return 2 * cta + (cta == g.c0); }

// A segment from the definition, eight rows at a time: a thread per key for the scores, then a thread per dimension (and part of the keys) for the outputs
// (THREADS of them, which `bar` brings together).  put(row, maximum (base 2), sum, this thread's dimension of the unnormalised output).
// Eight rows share every load: 256 rows take 3.3 us a key.
constexpr int PA_REDO = 8;
template <int D, int THREADS> struct alignas(16) PagedScratch {
    float q[D][PA_REDO], w[THREADS][PA_REDO], red[THREADS / 32][PA_REDO];
    int page[THREADS];
    uint8_t row[THREADS], seen[THREADS];                 // of its page; a bit per row of queries
};
template <class CT, int D, int THREADS, class IO, class Bar, class Put>
__device__ __noinline__ void paged_redo(const PagedAttn &p, const PagedSegment &g, int unit, PagedScratch<D, THREADS> &sc, Bar bar, Put put) {
    const int tid = threadIdx.x, dim = tid % D;
    for (int r0 = 0; r0 < g.rows; r0 += PA_REDO) {
        bar();
        for (int i = tid; i < PA_REDO * (D / 8); i += THREADS) {
            const int k = i / (D / 8), c = i % (D / 8), R = g.row0 + r0 + k;
            float x[8] = {};
            if (r0 + k < g.rows) io_load8(static_cast<const IO *>(p.q) + (int64_t)(g.first + R / p.group) * p.q_stride + (g.head * p.group + R % p.group) * D + 8 * c, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) sc.q[8 * c + e][k] = x[e];
        }
        bar();
        float m[PA_REDO], l[PA_REDO], acc[PA_REDO];
#pragma unroll
        for (int k = 0; k < PA_REDO; ++k) {
            m[k] = PA_NONE;
            l[k] = acc[k] = 0.f;
        }
        for (int b = g.u0 * unit; b < g.u1 * unit; b += THREADS) {
            auto key_of = [&](int i) { const int u = i / unit; return (u < g.span.a ? u : u + g.span.gap) * unit + i % unit; };
            const int key = key_of(b + tid);
            uint32_t seen = 0;
            if (b + tid < g.u1 * unit)
#pragma unroll
                for (int k = 0; k < PA_REDO; ++k)
                    seen |= (uint32_t)(r0 + k < g.rows && paged_sees(p, key, g.len - g.n + (g.row0 + r0 + k) / p.group)) << k;
            float z[PA_REDO] = {};
            if (seen) {
                const int page = paged_page(p.st, g.seq, key), row = key & ((1 << p.st.page_shift) - 1);
                if (page >= 0) {
                    const CT *at = reinterpret_cast<const CT *>(p.k_pool + paged_at(p.st, page, g.head));
#pragma unroll 4
                    for (int c = 0; c < D / 8; ++c) {
                        float x[8], y[PA_REDO] = {};
                        paged_load8<D>(at, p.st.page_shift, row, c, x);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            float qs[PA_REDO];
                            io_load8(sc.q[8 * c + e], qs);
#pragma unroll
                            for (int k = 0; k < PA_REDO; ++k) y[k] = fmaf(x[e], qs[k], y[k]);
                        }
#pragma unroll
                        for (int k = 0; k < PA_REDO; ++k) z[k] += y[k];
                    }
                } else seen = 0;
                sc.page[tid] = page;
                sc.row[tid] = (uint8_t)row;
            }
            sc.seen[tid] = (uint8_t)seen;
#pragma unroll
            for (int k = 0; k < PA_REDO; ++k) {
                z[k] = seen >> k & 1 ? z[k] * p.scale : -INFINITY;
                float top = z[k];
#pragma unroll
                for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                if ((tid & 31) == 0) sc.red[tid >> 5][k] = top;
            }
            bar();
            float fix[PA_REDO];
#pragma unroll
            for (int k = 0; k < PA_REDO; ++k) {
                float top = m[k];
#pragma unroll
                for (int w = 0; w < THREADS / 32; ++w) top = fmaxf(top, sc.red[w][k]);
                fix[k] = exp2f(m[k] - top);
                z[k] = seen >> k & 1 ? exp2f(z[k] - top) : 0.f;
                sc.w[tid][k] = z[k];
                m[k] = top;
            }
            bar();
#pragma unroll
            for (int k = 0; k < PA_REDO; ++k) {
#pragma unroll
                for (int o = 16; o; o >>= 1) z[k] += __shfl_xor_sync(0xffffffffu, z[k], o);
                if ((tid & 31) == 0) sc.red[tid >> 5][k] = z[k];
            }
            bar();
#pragma unroll
            for (int k = 0; k < PA_REDO; ++k) {
                l[k] *= fix[k];
                acc[k] *= fix[k];
#pragma unroll
                for (int w = 0; w < THREADS / 32; ++w) l[k] += sc.red[w][k];
            }
            const int end = min(THREADS, g.u1 * unit - b);
            for (int j0 = tid / D; j0 < end; j0 += 8 * (THREADS / D)) {      // eight rows of V on their way at once; one that is hidden is not touched
                uint32_t which[8];
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int j = j0 + e * (THREADS / D);
                    which[e] = j < end ? sc.seen[j] : 0;
                    v[e] = 0.f;
                    if (which[e])
                        v[e] = paged_load1<D>(reinterpret_cast<const CT *>(p.v_pool + paged_at(p.st, sc.page[j], g.head)), p.st.page_shift, sc.row[j], dim);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (!which[e]) continue;
                    float ws[PA_REDO];
                    io_load8(sc.w[j0 + e * (THREADS / D)], ws);
#pragma unroll
                    for (int k = 0; k < PA_REDO; ++k)
                        if (which[e] >> k & 1) acc[k] = fmaf(ws[k], v[e], acc[k]);
                }
            }
            bar();
        }
        // the parts of the keys
#pragma unroll
        for (int k = 0; k < PA_REDO; ++k) sc.w[tid][k] = acc[k];
        bar();
#pragma unroll
        for (int k = 0; k < PA_REDO; ++k) {
            acc[k] = 0.f;
#pragma unroll
            for (int part = 0; part < THREADS / D; ++part) acc[k] += sc.w[part * D + dim][k];
            if (r0 + k < g.rows) put(r0 + k, m[k], l[k], acc[k]);
        }
    }
    bar();
}

// four dimensions of a segment's row to the output
template <class IO> __device__ __forceinline__ void paged_out4(const PagedAttn &p, const PagedSegment &g, int r, int d, int dims, float4 x, float sum) {
    const int t = (g.row0 + r) / p.group;
    IO *to = static_cast<IO *>(p.out) + (int64_t)(g.first + t) * p.out_stride + (g.head * p.group + (g.row0 + r) % p.group) * dims + d;
    // (no weight: zero for a row that sees nothing; a row at a position sees itself, so all of its scores were minus infinity, and 0 / 0 is NaN)
    if (sum == 0.f && g.len - g.n + t < 0) x = make_float4(0.f, 0.f, 0.f, 0.f);
    else if (sum == 0.f) x = make_float4(NAN, NAN, NAN, NAN);
    else x = make_float4(x.x / sum, x.y / sum, x.z / sum, x.w / sum);
    if constexpr (sizeof(IO) == 4) *reinterpret_cast<float4 *>(to) = x;
    else *reinterpret_cast<uint2 *>(to) = make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
}

template <class CT, int D, int NB, bool EX> struct PaTraits {
    static constexpr bool Q4 = sizeof(CT) == 1, BF = std::is_same<CT, __nv_bfloat16>::value;
    static constexpr int UNIT = Q4 ? 32 : 16;
    static constexpr int NT = EX ? (BF ? 3 : 2) : 1;                              // ... of a query
    static constexpr int WT = EX ? NT : BF ? 2 : 1;                               // terms of a weight
    // A CTA of eight warps per SM; one row block of eight: CTAs of four, two per SM (Q4_0: four), so that one's queries, pages and results are under way
    // while another computes (64 sequences of 300 tokens 36.9 -> 26.6 us, 16 of 8192 95 -> 96)
    static constexpr int WARPS = NB == 1 ? 4 : 8, THREADS = 32 * WARPS;
    static constexpr int ROW = Q4 ? D / 2 + D / 16 : 2 * D;
    static constexpr int HALF = (16 * ROW + 127) / 128 * 128;                     // 16 rows, where TMA may put them
    static constexpr int TILE = UNIT / 16 * HALF, STAGE = 2 * TILE;               // K, then V
    // the rings of an SM: about 190 KB of 16-bit rows; of 4 bits 148 KB (D = 128)
    static constexpr int STAGES = Q4 ? (D == 128 ? 2 : 4) : D == 128 ? (NB == 4 ? 2 : 3) : 6;
    static constexpr int PER_SM = NB > 1 ? 1 : Q4 ? 4 : 2;
    static constexpr int ROWS = 8 * NB;
    // Weights reach 2^SLACK before the maximum moves.  In fp16 they are lifted to 2^15 at most, so that a weight of 2^-24 - 15 + SLACK of its row's largest is
    // the last one there; fp32 rows, whose second term ends there too, pay for a smaller SLACK with more moves
    static constexpr int SLACK = EX ? 1 : 4;
    static constexpr int LIFT = BF ? 0 : EX ? 14 : 11;                            // exponent; the maximum that weights are taken from is that much less
    static constexpr int V_UP = EX ? 12 : 7;                                      // Q4_0: the largest d, times 2^lift, is 2^V_UP .. 2^(V_UP + 1) when the lift is set
    static constexpr bool Q_SMEM = NB > 1 || (Q4 && EX);                          // query fragments in shared memory instead of registers
    static constexpr int KS = D / 16;
    static constexpr int RING = WARPS * STAGES * STAGE;
    static constexpr int COMB = WARPS * ROWS * (D + 4) * 4;                     // lies over the ring between segments
    static constexpr int BODY = (RING > COMB ? RING : COMB);
    static constexpr int Q_BYTES = Q_SMEM ? NT * NB * KS * 32 * 8 : 0;
    static constexpr size_t SMEM = 1024 + BODY + Q_BYTES;
    static_assert(ROWS * (D + 4) * 4 % 16 == 0 && ROWS * (D + 4) * 4 + sizeof(PagedScratch<D, THREADS>) <= BODY, "what a segment is computed again in lies over the ring too");
};

template <class CT, int D, int NB, bool EX>
__global__ void __launch_bounds__((PaTraits<CT, D, NB, EX>::THREADS), (PaTraits<CT, D, NB, EX>::PER_SM))
skn_paged_attn_kernel(const __grid_constant__ PagedAttn p, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                      const __grid_constant__ CUtensorMap mks, const __grid_constant__ CUtensorMap mvs) {
    using T = PaTraits<CT, D, NB, EX>;
    using IO = typename std::conditional<EX, float, __nv_bfloat16>::type;
    constexpr int UNIT = T::UNIT, NT = T::NT, WT = T::WT, KS = T::KS, STAGES = T::STAGES, ROWS = T::ROWS, NBLK = D / 32, WARPS = T::WARPS, THREADS = T::THREADS;
    extern __shared__ uint8_t raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    uint2 *qf = reinterpret_cast<uint2 *>(ring + T::BODY);
    __shared__ uint64_t full[WARPS * STAGES];
    __shared__ long long before[PA_MAX_SEQS + 1];
    __shared__ int seq_first[PA_MAX_SEQS], seq_n[PA_MAX_SEQS], seq_len[PA_MAX_SEQS];
    __shared__ float wml[WARPS][2 * ROWS], rml[2 * ROWS];
    __shared__ long long wsum_s[WARPS];
    __shared__ int flags[2];                   // [0] a result is not finite, [1] a wait ran out
    __shared__ unsigned ticket;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
    const PagedStep &st = p.st;

    if (tid < WARPS * STAGES) skn_mbar_init(&full[tid], 1);
    if (tid < 2) flags[tid] = 0;
    skn_fence_mbar_init();

    // ---- the line of units -----------------------------------------------------------------------------------------------
    long long u = 0, u_end = 1, total = 1;
    int n_cta = 1;
    if (!p.direct) {
        long long run = 0;
        for (int b = 0; b < st.n_seqs; b += THREADS) {
            const int s = b + tid;
            long long x = 0;
            if (s < st.n_seqs) {
                const PagedSeq sq = paged_mine(p, s);
                seq_first[s] = sq.first;
                seq_n[s] = sq.n;
                seq_len[s] = sq.len;
                if (sq.n > 0) x = paged_span(p, sq.len - sq.n, sq.len - 1, UNIT).units + (1LL << 40);      // and one segment a head
            }
            long long inc = x;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += y;
            }
            if (lane == 31) wsum_s[warp] = inc;
            __syncthreads();
            long long base = run;
            for (int w = 0; w < WARPS; ++w) {
                if (w < warp) base += wsum_s[w];
                run += wsum_s[w];
            }
            if (s < st.n_seqs) before[s] = ((base + inc - x) & ((1LL << 40) - 1)) * st.heads;
            __syncthreads();
        }
        total = (run & ((1LL << 40) - 1)) * st.heads;
        if (total == 0) {
            if (p.split) skn_pdl_wait();
            return;
        }
        // fewer CTAs where each would get less than a unit per warp; short segments get one each (nothing to join: 100 tokens of one sequence 18.5 -> 9.2 us)
        const long long segments = (run >> 40) * st.heads;
        const long long want = total <= 2 * WARPS * segments ? segments : (total + WARPS - 1) / WARPS;
        n_cta = want < (long long)gridDim.x ? (int)want : (int)gridDim.x;
        if ((int)blockIdx.x >= n_cta) {
            if (p.split) skn_pdl_wait();
            return;
        }
        u = paged_div(total * blockIdx.x, n_cta);
        u_end = paged_div(total * (blockIdx.x + 1), n_cta);
    } else __syncthreads();

    int stage = 0, parity = 0;                 // of the warp's next unit
    int s_at = 0;
    while (u < u_end) {
        // ---- which segment ------------------------------------------------------------------------------------------------
        PagedSegment g;
        if (p.direct) {
            g.seq = blockIdx.z;
            g.head = blockIdx.y;
            const PagedSeq sq = paged_mine(p, g.seq);
            g.n = sq.n; g.len = sq.len; g.first = sq.first;
            const int n_blocks = (sq.n * p.group + ROWS - 1) / ROWS;
            const int rb = n_blocks - 1 - (int)blockIdx.x;              // the longest rows first
            if (rb < 0) {
                if (p.split) skn_pdl_wait();
                return;
            }
            g.row0 = rb * ROWS;
            g.rows = min(ROWS, sq.n * p.group - g.row0);
            g.span = paged_span(p, sq.len - sq.n + g.row0 / p.group, sq.len - sq.n + (g.row0 + g.rows - 1) / p.group, UNIT);
            g.u0 = 0; g.u1 = g.span.units;
            g.n_parts = 1; g.c0 = 0; g.slot = 0;
            u = u_end;
        } else {
            int lo = s_at, hi = st.n_seqs - 1;                          // the last sequence that begins at or before u and has units
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (before[mid] <= u) lo = mid; else hi = mid - 1;
            }
            s_at = g.seq = lo;
            g.n = seq_n[lo]; g.len = seq_len[lo]; g.first = seq_first[lo];
            g.row0 = 0; g.rows = g.n * p.group;
            g.span = paged_span(p, g.len - g.n, g.len - 1, UNIT);
            const long long off = u - before[lo];
            g.head = (int)paged_div(off, g.span.units);
            g.u0 = (int)(off - (long long)g.head * g.span.units);
            const long long left = u_end - u;
            g.u1 = left < g.span.units - g.u0 ? g.u0 + (int)left : g.span.units;
            g.c0 = (int)blockIdx.x;
            g.n_parts = 1;
            if (g.u0 > 0 || g.u1 < g.span.units) {
                const long long a = u - g.u0;
                g.c0 = (int)paged_div((a + 1) * n_cta - 1, total);
                g.n_parts = (int)paged_div((a + g.span.units) * n_cta - 1, total) - g.c0 + 1;
            }
            g.slot = paged_slot(g, (int)blockIdx.x);
            u += g.u1 - g.u0;
        }
        const int pmin = g.len - g.n + g.row0 / p.group, pmax = g.len - g.n + (g.row0 + g.rows - 1) / p.group;
        const int n_mine = (g.u1 - g.u0 - warp + WARPS - 1) / WARPS;         // units g.u0 + warp + WARPS j

        // ---- queries, on their way while the pages are looked up: this lane's part of row g8 of each block of eight ---------------
        // 16-bit caches: dims 16 k + 2 t, + 1, + 8, + 9.  Q4_0: of block k / 2, its lower (k even) or upper 16: 4 t, + 2, + 1, + 3
        float x[NB][KS][4];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int r = 8 * nb + g8, t = (g.row0 + r) / p.group;
            const IO *q = static_cast<const IO *>(p.q) + (int64_t)(g.first + t) * p.q_stride + (g.head * p.group + (g.row0 + r) % p.group) * D;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                float a[4] = {};
                if (r < g.rows) {
                    if constexpr (EX && T::Q4) {
                        const float4 y = *reinterpret_cast<const float4 *>(q + 16 * k + 4 * t4);
                        a[0] = y.x; a[1] = y.z; a[2] = y.y; a[3] = y.w;
                    } else if constexpr (EX) {
                        const float2 y = *reinterpret_cast<const float2 *>(q + 16 * k + 2 * t4), z = *reinterpret_cast<const float2 *>(q + 16 * k + 8 + 2 * t4);
                        a[0] = y.x; a[1] = y.y; a[2] = z.x; a[3] = z.y;
                    } else if constexpr (T::Q4) {
                        const uint2 y = *reinterpret_cast<const uint2 *>(q + 16 * k + 4 * t4);
                        a[0] = __uint_as_float(y.x << 16); a[1] = __uint_as_float(y.y << 16);
                        a[2] = __uint_as_float(y.x & 0xFFFF0000u); a[3] = __uint_as_float(y.y & 0xFFFF0000u);
                    } else {
                        const uint32_t y = *reinterpret_cast<const uint32_t *>(q + 16 * k + 2 * t4), z = *reinterpret_cast<const uint32_t *>(q + 16 * k + 8 + 2 * t4);
                        a[0] = __uint_as_float(y << 16); a[1] = __uint_as_float(y & 0xFFFF0000u);
                        a[2] = __uint_as_float(z << 16); a[3] = __uint_as_float(z & 0xFFFF0000u);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) x[nb][k][i] = a[i];
            }
        }

        // ---- loads of the warp's units: lane j of `pages` holds the pages of unit j (mod 32) ---------------------------------
        int page0 = -1, page1 = -1;
        auto key_of = [&](int j) {
            const int i = g.u0 + warp + WARPS * j;
            return (i < g.span.a ? i : i + g.span.gap) * UNIT;
        };
        const int seen_from = p.window ? max(0, max(0, pmin) - p.window + 1) : 0;
        auto needed = [&](int k) { return k <= pmax && (k + 15 >= seen_from || k < p.sinks); };     // some row sees some of 16 keys
        auto look_up = [&](int j0) {               // pages of units j0 .. j0 + 31; the table is asked for none that nobody needs
            const int j = j0 + lane;
            page0 = page1 = -1;
            if (j < n_mine) {
                const int k = key_of(j);
                if (needed(k)) page0 = paged_page(st, g.seq, k);
                if (T::Q4) {
                    if (needed(k + 16)) page1 = st.page_shift > 4 && page0 >= 0 ? page0 : paged_page(st, g.seq, k + 16);
                }
            }
        };
        look_up(0);
        uint8_t *const mine = ring + warp * STAGES * T::STAGE;
        uint32_t there = 0;                        // two bits a stage: which 16 keys of its unit have a page
        auto issue = [&](int j, int at) {          // a lane per box of 16 rows: K and V, Q4_0: quants and scales of both halves
            const int pg0 = __shfl_sync(0xffffffffu, page0, j & 31), pg1 = T::Q4 ? __shfl_sync(0xffffffffu, page1, j & 31) : -1;
            there = (there & ~(3u << (2 * at))) | ((uint32_t)(pg0 >= 0) << (2 * at)) | ((uint32_t)(pg1 >= 0) << (2 * at + 1));
            uint64_t *bar = &full[warp * STAGES + at];
            const int row = key_of(j) & ((1 << st.page_shift) - 1);
            uint8_t *const to = mine + at * T::STAGE + (lane & 1) * T::TILE;
            if (lane == 0) {
                const int n = (pg0 >= 0) + (pg1 >= 0);
                if (n) skn_mbar_expect_tx(bar, n * 32 * T::ROW);
                else skn_mbar_arrive(bar);
            }
            __syncwarp();
            if constexpr (!T::Q4) {
                if (lane < 2 && pg0 >= 0) tma_3d(to, lane ? &mv : &mk, 0, ((pg0 * st.heads + g.head) << st.page_shift) + row, 0, bar);
            } else {
                // quants [D / 32][16][16 bytes], then scales [16][D / 32]
                const int h = (lane >> 2) & 1, pg = h ? pg1 : pg0, z = pg * st.heads + g.head, r = (row + 16 * h) & ((1 << st.page_shift) - 1);
                if (lane < 8 && pg >= 0) {
                    if (lane & 2) tc_tma_load_2d(to + h * T::HALF + 16 * (D / 2), lane & 1 ? &mvs : &mks, r * (D / 64), z, bar);
                    else tma_3d(to + h * T::HALF, lane & 1 ? &mv : &mk, r * 4, 0, z, bar);
                }
            }
        };
        const bool dead = flags[1] != 0;
        int issued = dead ? n_mine : 0;
        for (int i = 0; i < STAGES && issued < n_mine; ++i, ++issued) issue(issued, (stage + i) % STAGES);

        // ---- fragments of the second operand: fp16 products take queries times a power of two that brings a row's largest to 2^14 .. 2^15 ---
        uint32_t qr[T::Q_SMEM ? 1 : NT][T::Q_SMEM ? 1 : NB][KS][2];
        float cs[NB][2];                           // factor of the scores of rows 2 t4, 2 t4 + 1
        float bias[T::Q4 ? NB : 1][T::Q4 ? NBLK : 1][2];
        int pos[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            float f = 1.f;
            if constexpr (!T::BF) {
                float top = 0.f;
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(x[nb][k][i]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                int e = 14 - ((int)(__float_as_uint(top) >> 23) - 127);
                e = top > 0.f && top < INFINITY ? max(-120, min(120, e)) : 0;
                const float up = __uint_as_float((uint32_t)(127 + e) << 23);
                f = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[nb][k][i] *= up;
            }
            float bs[T::Q4 ? NBLK : 1];
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                if constexpr (T::Q4) {
                    const float sum = (x[nb][k][0] + x[nb][k][1]) + (x[nb][k][2] + x[nb][k][3]);
                    if (k & 1) bs[k >> 1] += sum; else bs[k >> 1] = sum;
                    if (!EX && (k & 1)) {           // the upper nibble stands 16 times higher
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[nb][k][i] *= 0.0625f;
                    }
                }
                uint32_t a[NT], b[NT];
                terms_of<CT, NT>(x[nb][k][0], x[nb][k][1], a);
                terms_of<CT, NT>(x[nb][k][2], x[nb][k][3], b);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if constexpr (T::Q_SMEM) {
                        if (warp == 0) qf[((n * NB + nb) * KS + k) * 32 + lane] = make_uint2(a[n], b[n]);
                    } else {
                        qr[n][nb][k][0] = a[n];
                        qr[n][nb][k][1] = b[n];
                    }
                }
            }
            f *= p.scale;
            if constexpr (T::Q4 && !EX) f *= 16777216.f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int src = 4 * (2 * t4 + c);
                cs[nb][c] = __shfl_sync(0xffffffffu, f, src);
                if (!(fabsf(cs[nb][c]) < INFINITY)) flags[0] = 1;       // scores of minus infinity would look like hidden keys': the segment is computed again
                const int rc = 8 * nb + 2 * t4 + c;
                pos[nb][c] = rc < g.rows ? g.len - g.n + (g.row0 + rc) / p.group : -1;
                if constexpr (T::Q4) {
#pragma unroll
                    for (int b = 0; b < NBLK; ++b) {
                        float s = bs[b];
                        s += __shfl_xor_sync(0xffffffffu, s, 1);
                        s += __shfl_xor_sync(0xffffffffu, s, 2);
                        bias[nb][b][c] = __shfl_sync(0xffffffffu, s, src) * (-8.f / 16777216.f);
                    }
                }
            }
        }
        if constexpr (T::Q_SMEM) __syncthreads();

        // ---- the units ------------------------------------------------------------------------------------------------------
        float o[D / 16][NB][4], m[NB][2], most[NB][2], l[NB][2];
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[i][nb][c] = 0.f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                m[nb][c] = 0.f;
                most[nb][c] = -INFINITY;
                l[nb][c] = 0.f;
            }
        int lift = T::Q4 ? 0 : T::LIFT;            // m: the maximum less this; most: exponent of the largest weight before it moves
        __half2 vlim = __floats2half2_rn(0.f, 0.f); // Q4_0: the largest |d| that the lift takes
        for (int j = 0; j < n_mine && !dead; ++j) {
            const int kbase = key_of(j);
            bool gone = false;
            {
                uint64_t *bar = &full[warp * STAGES + stage];
                if (!tc_wait_warp(bar, parity, lane)) gone = true;
            }
            if (gone) {
                if (lane == 0) {
                    *st.status = SKN_ERR_TIMEOUT;
                    flags[1] = 1;
                }
                for (; j < issued; ++j) {          // what is on its way lands before its place is used again
                    tc_wait_warp(&full[warp * STAGES + stage], parity, lane);
                    if (++stage == STAGES) {
                        stage = 0;
                        parity ^= 1;
                    }
                }
                break;
            }
            const bool has0 = there >> (2 * stage) & 1, has1 = !T::Q4 || (there >> (2 * stage + 1) & 1);
            uint8_t *kt = mine + stage * T::STAGE, *vt = kt + T::TILE;
            const bool whole = kbase + UNIT - 1 <= pmin && has0 && has1 && (!p.window || kbase > pmax - p.window || kbase + UNIT <= p.sinks);
            if constexpr (!T::Q4) {
                if (!whole) {                      // rows of V that are not finite: cleared if nobody sees them
                    const int r = lane & 15, key = kbase + r;
                    const uint32_t base = skn_smem_u32(vt) + r * 128;
                    bool odd = false, some = false;
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        const int cc = (lane >> 4) * (D / 16) + c;
                        const uint4 v = tc_lds128(base + (cc >> 3) * 2048 + (((cc & 7) ^ (r & 7)) << 4));
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                        constexpr uint32_t EXP = T::BF ? 0x7F80u : 0x7C00u;
#pragma unroll
                        for (int i = 0; i < 4; ++i) odd |= (w[i] & EXP) == EXP || (w[i] & (EXP << 16)) == (EXP << 16);
                    }
                    odd |= __shfl_xor_sync(0xffffffffu, (int)odd, 16) != 0;      // (every lane takes part)
                    for (int t = g.row0 / p.group; t <= (g.row0 + g.rows - 1) / p.group; ++t) some |= has0 && paged_sees(p, key, g.len - g.n + t);
                    if (odd && !some) {
#pragma unroll 1
                        for (int c = 0; c < D / 16; ++c) {
                            const int cc = (lane >> 4) * (D / 16) + c;
                            *reinterpret_cast<uint4 *>(vt + r * 128 + (cc >> 3) * 2048 + (((cc & 7) ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
                        }
                        skn_fence_proxy_async();
                    }
                    __syncwarp();
                }
            }
#pragma unroll
            for (int sub = 0; sub < UNIT / 16; ++sub) {
                const int key0 = kbase + 16 * sub;
                const bool hidden_page = !(sub ? has1 : has0);
                float s[NB][4];
                // ---- scores ------------------------------------------------------------------------------------------------
                const uint8_t *vq = nullptr;       // Q4_0: this half's rows of V
                float dv[2][T::Q4 ? NBLK : 1];
                __half2 dtop = vlim;
                if constexpr (T::Q4) {
                    const uint8_t *kq = kt + sub * T::HALF, *kd = kq + 16 * (D / 2), *vd = vt + sub * T::HALF + 16 * (D / 2);
                    vq = vt + sub * T::HALF;
                    float dk[2][NBLK];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t wk[NBLK / 2], wv[NBLK / 2];
                        if constexpr (D == 128) {
                            const uint2 a = *reinterpret_cast<const uint2 *>(kd + (g8 + 8 * h) * 8), b = *reinterpret_cast<const uint2 *>(vd + (g8 + 8 * h) * 8);
                            wk[0] = a.x; wk[1] = a.y; wv[0] = b.x; wv[1] = b.y;
                        } else {
                            wk[0] = *reinterpret_cast<const uint32_t *>(kd + (g8 + 8 * h) * 4);
                            wv[0] = *reinterpret_cast<const uint32_t *>(vd + (g8 + 8 * h) * 4);
                        }
#pragma unroll
                        for (int b = 0; b < NBLK / 2; ++b) {
                            const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&wk[b]));
                            const __half2 hv = *reinterpret_cast<const __half2 *>(&wv[b]);
                            const float2 c = __half22float2(hv);
                            dk[h][2 * b] = a.x; dk[h][2 * b + 1] = a.y;
                            dv[h][2 * b] = c.x; dv[h][2 * b + 1] = c.y;
                            dtop = __hmax2_nan(dtop, __habs2(hv));
                        }
                    }
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int c = 0; c < 4; ++c) s[nb][c] = 0.f;
#pragma unroll
                    for (int b = 0; b < NBLK; ++b) {
                        const uint32_t w0 = *reinterpret_cast<const uint32_t *>(kq + b * 256 + g8 * 16 + t4 * 4);
                        const uint32_t w1 = *reinterpret_cast<const uint32_t *>(kq + b * 256 + (g8 + 8) * 16 + t4 * 4);
                        uint32_t lo[4] = {w0 & 0x000F000Fu, w1 & 0x000F000Fu, (w0 >> 8) & 0x000F000Fu, (w1 >> 8) & 0x000F000Fu};
                        uint32_t hi[4] = {w0 & 0x00F000F0u, w1 & 0x00F000F0u, (w0 >> 8) & 0x00F000F0u, (w1 >> 8) & 0x00F000F0u};
                        if constexpr (EX) {        // q - 8 itself: no large sums that cancel
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                lo[i] |= 0x64006400u;
                                hi[i] |= 0x64006400u;
                                const __half2 x = __hadd2(*reinterpret_cast<const __half2 *>(&lo[i]), __float2half2_rn(-1032.f));
                                const __half2 y = __hfma2(*reinterpret_cast<const __half2 *>(&hi[i]), __float2half2_rn(0.0625f), __float2half2_rn(-72.f));
                                lo[i] = *reinterpret_cast<const uint32_t *>(&x);
                                hi[i] = *reinterpret_cast<const uint32_t *>(&y);
                            }
                        }
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            float acc[4], small[4];
#pragma unroll
                            for (int n = NT - 1; n >= 0; --n) {
                                uint2 f0, f1;
                                if constexpr (T::Q_SMEM) {
                                    f0 = qf[((n * NB + nb) * KS + 2 * b) * 32 + lane];
                                    f1 = qf[((n * NB + nb) * KS + 2 * b + 1) * 32 + lane];
                                } else {
                                    f0 = make_uint2(qr[n][nb][2 * b][0], qr[n][nb][2 * b][1]);
                                    f1 = make_uint2(qr[n][nb][2 * b + 1][0], qr[n][nb][2 * b + 1][1]);
                                }
                                if constexpr (EX) {
                                    mma_f16_from(n ? small : acc, lo, f0.x, f0.y, 0.f, 0.f);
                                    mma_f16(n ? small : acc, hi, f1.x, f1.y);
                                } else {
                                    mma_f16_from(acc, lo, f0.x, f0.y, bias[nb][b][0], bias[nb][b][1]);
                                    mma_f16(acc, hi, f1.x, f1.y);
                                }
                            }
                            if constexpr (EX) {
#pragma unroll
                                for (int c = 0; c < 4; ++c) acc[c] += small[c];
                            }
                            s[nb][0] = fmaf(acc[0], dk[0][b], s[nb][0]);
                            s[nb][1] = fmaf(acc[1], dk[0][b], s[nb][1]);
                            s[nb][2] = fmaf(acc[2], dk[1][b], s[nb][2]);
                            s[nb][3] = fmaf(acc[3], dk[1][b], s[nb][3]);
                        }
                    }
                } else {
                    const int row = (lane & 7) + (lane & 8);
                    const uint32_t base = skn_smem_u32(kt) + row * 128;
                    float odd[EX ? NB : 1][4], small[EX ? NB : 1][4];
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        const int c = 2 * k + (lane >> 4);
                        uint32_t a[4];
                        ldsm4(a, base + (c >> 3) * 2048 + (((c & 7) ^ (row & 7)) << 4));
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                            for (int n = NT - 1; n >= 0; --n) {
                                uint2 f;
                                if constexpr (T::Q_SMEM) f = qf[((n * NB + nb) * KS + k) * 32 + lane];
                                else f = make_uint2(qr[n][nb][k][0], qr[n][nb][k][1]);
                                if constexpr (EX) {
                                    float (&to)[4] = n ? small[nb] : k & 1 ? odd[nb] : s[nb];
                                    if (n ? k == 0 && n == NT - 1 : k < 2) mma_zero<CT>(to, a, f.x, f.y);
                                    else mma_as<CT>(to, a, f.x, f.y);
                                } else if (k == 0) mma_zero<CT>(s[nb], a, f.x, f.y);
                                else mma_as<CT>(s[nb], a, f.x, f.y);
                            }
                    }
                    if constexpr (EX) {
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                            for (int c = 0; c < 4; ++c) s[nb][c] = (s[nb][c] + odd[nb][c]) + small[nb][c];
                    }
                }
                // ---- weights -----------------------------------------------------------------------------------------------
                bool move = false;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        s[nb][c] = fmaf(s[nb][c], cs[nb][c & 1], -m[nb][c & 1]);
                        if (!whole && (hidden_page || !paged_sees(p, key0 + g8 + 8 * (c >> 1), pos[nb][c & 1]))) s[nb][c] = -INFINITY;
                        move |= s[nb][c] > most[nb][c & 1];
                    }
                if constexpr (T::Q4) move |= !__hble2(dtop, vlim);
                if (__any_sync(0xffffffffu, move)) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float top = fmaxf(s[nb][c], s[nb][c + 2]);
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                            // the row's maximum, `lift` above m, moves by so much (the first one either way)
                            const bool begun = most[nb][c] > -INFINITY;
                            const float by = begun ? fmaxf(top - (float)lift, 0.f) : top > -INFINITY ? top - (float)lift : 0.f, fix = begun ? pa_ex2(-by) : 1.f;
                            if (top > -INFINITY) most[nb][c] = (float)(lift + T::SLACK);
                            s[nb][c] -= by;
                            s[nb][c + 2] -= by;
                            m[nb][c] += by;
                            l[nb][c] *= fix;
#pragma unroll
                            for (int i = 0; i < D / 16; ++i) {
                                o[i][nb][c] *= fix;
                                o[i][nb][c + 2] *= fix;
                            }
                        }
                    if constexpr (T::Q4) {
                        // scales of V: those of keys that nobody sees count for nothing; the largest of the others decides E
                        float top = 0.f;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int key = key0 + g8 + 8 * h;
                            bool some = false;
                            for (int t = g.row0 / p.group; t <= (g.row0 + g.rows - 1) / p.group; ++t) some |= !hidden_page && paged_sees(p, key, g.len - g.n + t);
#pragma unroll
                            for (int b = 0; b < NBLK; ++b) {
                                if (!some) dv[h][b] = 0.f;
                                if (fabsf(dv[h][b]) < INFINITY) top = fmaxf(top, fabsf(dv[h][b]));
                            }
                        }
#pragma unroll
                        for (int o2 = 1; o2 < 32; o2 <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o2));
                        if (top > __half2float(__low2half(vlim))) {
                            // up to 2^LIFT: weights stay within 2^15
                            const int fresh = T::V_UP + 127 - (int)(__float_as_uint(top) >> 23), by = fresh - lift;
                            const float fix = __uint_as_float((uint32_t)(127 + by) << 23);
                            lift = fresh;
                            vlim = __float2half2_rn(fminf(__uint_as_float((uint32_t)(127 + T::LIFT - fresh) << 23), 65504.f));
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                                for (int c = 0; c < 2; ++c) {
                                    m[nb][c] -= (float)by;
                                    l[nb][c] *= fix;
                                    s[nb][c] += (float)by;
                                    s[nb][c + 2] += (float)by;
                                    most[nb][c] += (float)by;            // (minus infinity stays)
                                }
#pragma unroll
                                for (int i = 0; i < D / 16; ++i)
#pragma unroll
                                    for (int c = 0; c < 4; ++c) o[i][nb][c] *= fix;
                            }
                        }
                    }
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        s[nb][c] = pa_ex2(s[nb][c]);
                        l[nb][c & 1] += s[nb][c];
                    }
                // ---- values ------------------------------------------------------------------------------------------------
                if constexpr (T::Q4) {
                    // 1024 + q or 1024 + 16 q in fp16, then q - 8: exact, so that a value of zero adds nothing
                    const uint32_t mask = g8 & 4 ? 0x00F000F0u : 0x000F000Fu;
                    const __half2 vmul = __float2half2_rn(g8 & 4 ? 0.0625f : 1.f), vadd = __float2half2_rn(g8 & 4 ? -72.f : -1032.f);
                    auto less8 = [&](uint32_t x) {
                        const uint32_t y = (x & mask) | 0x64006400u;
                        const __half2 z = __hfma2(*reinterpret_cast<const __half2 *>(&y), vmul, vadd);
                        return *reinterpret_cast<const uint32_t *>(&z);
                    };
#pragma unroll
                    for (int b = 0; b < NBLK; ++b) {
                        uint32_t pb[NB][NT][2];
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            const float w0 = s[nb][0] * dv[0][b], w1 = s[nb][1] * dv[0][b], w2 = s[nb][2] * dv[1][b], w3 = s[nb][3] * dv[1][b];
                            uint32_t a[NT], c[NT];
                            terms_of<CT, NT>(w0, w1, a);
                            terms_of<CT, NT>(w2, w3, c);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                pb[nb][n][0] = movm(a[n]);
                                pb[nb][n][1] = movm(c[n]);
                            }
                        }
                        const uint8_t *at = vq + b * 256 + 2 * t4 * 16 + (g8 & 3) * 4;
                        const uint32_t x0 = *reinterpret_cast<const uint32_t *>(at), x1 = *reinterpret_cast<const uint32_t *>(at + 16);
                        const uint32_t x2 = *reinterpret_cast<const uint32_t *>(at + 128), x3 = *reinterpret_cast<const uint32_t *>(at + 144);
                        const uint32_t lo = __byte_perm(x0, x1, 0x5410), lo2 = __byte_perm(x2, x3, 0x5410), hi = __byte_perm(x0, x1, 0x7632), hi2 = __byte_perm(x2, x3, 0x7632);
                        const uint32_t a0[4] = {less8(lo), less8(lo >> 8), less8(lo2), less8(lo2 >> 8)};
                        const uint32_t a1[4] = {less8(hi), less8(hi >> 8), less8(hi2), less8(hi2 >> 8)};
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            pa_add<CT, EX, NT>(o[2 * b][nb], a0, pb[nb]);
                            pa_add<CT, EX, NT>(o[2 * b + 1][nb], a1, pb[nb]);
                        }
                    }
                } else {
                    uint32_t pb[NB][WT][2];
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        uint32_t a[WT], c[WT];
                        terms_of<CT, WT>(s[nb][0], s[nb][1], a);
                        terms_of<CT, WT>(s[nb][2], s[nb][3], c);
#pragma unroll
                        for (int n = 0; n < WT; ++n) {
                            pb[nb][n][0] = movm(a[n]);
                            pb[nb][n][1] = movm(c[n]);
                        }
                    }
                    const int row = (lane & 7) + ((lane & 16) >> 1);
                    const uint32_t base = skn_smem_u32(vt) + row * 128;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        const int c = 2 * i + ((lane >> 3) & 1);
                        uint32_t a[4];
                        ldsm4t(a, base + (c >> 3) * 2048 + (((c & 7) ^ (row & 7)) << 4));
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) pa_add<CT, EX, WT>(o[i][nb], a, pb[nb]);
                    }
                }
            }
            __syncwarp();                          // the stage is read
            if (issued < n_mine) {
                if ((issued & 31) == 0) look_up(issued);
                issue(issued, stage);
                ++issued;
            }
            if (++stage == STAGES) {
                stage = 0;
                parity ^= 1;
            }
        }
        // ---- the warps' results -----------------------------------------------------------------------------------------------
        __syncthreads();                           // every ring is empty: the results lie over them
        float *comb = reinterpret_cast<float *>(ring);
        {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float x = l[nb][c];
                    x += __shfl_xor_sync(0xffffffffu, x, 4);
                    x += __shfl_xor_sync(0xffffffffu, x, 8);
                    x += __shfl_xor_sync(0xffffffffu, x, 16);
                    const int r = 8 * nb + 2 * t4 + c;
                    if (g8 == 0) {
                        wml[warp][2 * r] = m[nb][c];
                        wml[warp][2 * r + 1] = x;
                    }
                    float *to = comb + (warp * ROWS + r) * (D + 4);
                    if constexpr (T::Q4) {
#pragma unroll
                        for (int b = 0; b < NBLK; ++b)
#pragma unroll
                            for (int i = 0; i < 2; ++i)
                                *reinterpret_cast<float2 *>(to + 32 * b + 4 * (g8 & 3) + 16 * (g8 >> 2) + 2 * i) = make_float2(o[2 * b + i][nb][c], o[2 * b + i][nb][c + 2]);
                    } else {
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) {
                            to[16 * i + g8] = o[i][nb][c];
                            to[16 * i + g8 + 8] = o[i][nb][c + 2];
                        }
                    }
                }
            __syncthreads();
            // maximum, sum and output of all warps, out or to the other CTAs of the segment
            if (tid < ROWS) {
                float top = PA_NONE;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) top = fmaxf(top, wml[w][2 * tid + 1] != 0.f ? wml[w][2 * tid] : PA_NONE);
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) {
                    const float f = wml[w][2 * tid + 1] != 0.f ? exp2f(wml[w][2 * tid] - top) : 0.f;
                    sum += wml[w][2 * tid + 1] * f;
                    wml[w][2 * tid] = f;
                }
                rml[2 * tid] = top;
                rml[2 * tid + 1] = sum;
            }
            __syncthreads();
        }
        float *const part = p.parts + (int64_t)g.slot * ROWS * (D + 4);
        auto put4 = [&](int r, int d, float4 x, float m, float sum) {       // four dimensions of a row's result
            if (g.n_parts > 1) {
                *reinterpret_cast<float4 *>(part + r * (D + 4) + d) = x;
                if (d == 0) *reinterpret_cast<float2 *>(part + r * (D + 4) + D) = make_float2(m, sum);
            } else
                paged_out4<IO>(p, g, r, d, D, x, sum);
        };
        for (int i = tid; i < g.rows * (D / 4); i += THREADS) {
            const int r = i / (D / 4), d = i % (D / 4) * 4;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float f = wml[w][2 * r];
                const float4 y = *reinterpret_cast<const float4 *>(comb + (w * ROWS + r) * (D + 4) + d);
                if (f != 0.f) { x.x = fmaf(y.x, f, x.x); x.y = fmaf(y.y, f, x.y); x.z = fmaf(y.z, f, x.z); x.w = fmaf(y.w, f, x.w); }
            }
            const float sum = rml[2 * r + 1], all = (x.x + x.y) + (x.z + x.w) + sum;
            if (!(fabsf(all) < INFINITY)) flags[0] = 1;             // (a sum of finite values that overflows is computed again for nothing)
            put4(r, d, x, rml[2 * r], sum);
        }
        if (g.n_parts > 1) __threadfence();
        __syncthreads();
        if (flags[0]) {
            const PagedSegment seg = g;            // (a copy: the address of the one that the loops use is not taken)
            paged_redo<CT, D, THREADS, IO>(p, seg, UNIT, *reinterpret_cast<PagedScratch<D, THREADS> *>(ring + ROWS * (D + 4) * 4), [] { __syncthreads(); }, [=](int r, float rm, float rl, float acc) {
                if (tid < D) comb[r * (D + 4) + tid] = acc;
                if (tid == 0) {
                    comb[r * (D + 4) + D] = rm;
                    comb[r * (D + 4) + D + 1] = rl;
                }
            });
            for (int i = tid; i < g.rows * (D / 4); i += THREADS) {
                const int r = i / (D / 4), d = i % (D / 4) * 4;
                put4(r, d, *reinterpret_cast<const float4 *>(comb + r * (D + 4) + d), comb[r * (D + 4) + D], comb[r * (D + 4) + D + 1]);
            }
            if (tid == 0) flags[0] = 0;
            __threadfence();
            __syncthreads();
        }
        // ---- the last CTA of a segment joins what all of them left ------------------------------------------------------------------
        if (g.n_parts > 1) {
            if (tid == 0) ticket = atomicInc(&p.tickets[paged_slot(g, g.c0)], (unsigned)g.n_parts - 1);
            __syncthreads();
            if (ticket == (unsigned)g.n_parts - 1) {
                __threadfence();
                for (int i = tid; i < g.rows * (D / 4); i += THREADS) {
                    const int r = i / (D / 4), d = i % (D / 4) * 4;
                    float top = PA_NONE, sum = 0.f;
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int k = 0; k < g.n_parts; k += 8) {        // eight parts' loads on their way at once
                        float2 ml[8];
                        float4 y[8];
#pragma unroll
                        for (int b = 0; b < 8; ++b) {
                            const float *from = p.parts + ((int64_t)paged_slot(g, g.c0 + min(k + b, g.n_parts - 1)) * ROWS + r) * (D + 4);
                            ml[b] = __ldcg(reinterpret_cast<const float2 *>(from + D));
                            y[b] = __ldcg(reinterpret_cast<const float4 *>(from + d));
                        }
                        float high = top;
#pragma unroll
                        for (int b = 0; b < 8; ++b)
                            if (k + b < g.n_parts && ml[b].y != 0.f) high = fmaxf(high, ml[b].x);
                        const float fix = exp2f(top - high);
                        top = high;
                        sum *= fix;
                        x.x *= fix; x.y *= fix; x.z *= fix; x.w *= fix;
#pragma unroll
                        for (int b = 0; b < 8; ++b) {
                            if (k + b >= g.n_parts || ml[b].y == 0.f) continue;
                            const float f = exp2f(ml[b].x - top);
                            sum = fmaf(ml[b].y, f, sum);
                            x.x = fmaf(y[b].x, f, x.x); x.y = fmaf(y[b].y, f, x.y); x.z = fmaf(y[b].z, f, x.z); x.w = fmaf(y[b].w, f, x.w);
                        }
                    }
                    paged_out4<IO>(p, g, r, d, D, x, sum);
                }
            }
        }
        skn_fence_proxy_async();                   // the rings were written to as results
        __syncthreads();
    }
    if (p.split) skn_pdl_wait();               // (whoever waits for this launch waits for the one before)
}

// ---- launches ---------------------------------------------------------------------------------------------------------------
template <class CT, int D, int NB, bool EX> static cudaError_t attn_launch(const skn_paged *pc, const PagedAttn &p) {
    using T = PaTraits<CT, D, NB, EX>;
    auto *kern = skn_paged_attn_kernel<CT, D, NB, EX>;
    static uint64_t done = 0;
    const cudaError_t e = paged_attributes(kern, T::SMEM, pc->ctx->device, &done);
    if (e != cudaSuccess) return e;
    const int64_t rows = (int64_t)p.st.max_new * p.group, most = rows < p.upto ? rows : p.upto;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = p.direct ? dim3((unsigned)((most + T::ROWS - 1) / T::ROWS), (unsigned)p.st.heads, (unsigned)p.st.n_seqs) : dim3((unsigned)(T::PER_SM * pc->ctx->sm_count));
    cfg.blockDim = dim3(T::THREADS);
    cfg.dynamicSmemBytes = T::SMEM;
    cfg.stream = pc->ctx->stream;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = p.split ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, p, pc->map[0], pc->map[1], pc->map[2], pc->map[3]);
}
// bf16 rows of prompts (skn_paged_prompt.cuh); the first argument names the cache type
cudaError_t skn_paged_prompt(__half, const skn_paged *pc, const PagedAttn &p);
cudaError_t skn_paged_prompt(__nv_bfloat16, const skn_paged *pc, const PagedAttn &p);
cudaError_t skn_paged_prompt(skn_q4, const skn_paged *pc, const PagedAttn &p);

// Up to 32 rows a sequence: shared out with the keys.  More: blocks of rows, bf16 on tcgen05, fp32 a CTA each; then the sequences of a step that
// have few (the rows of one token or a little more: decoding beside prompts) follow in a launch of their own, which begins while the first one ends.
// (512 tokens of a prompt beside 256 sequences of 2048 decoding, bf16, 32 / 8 heads of 128: 356 us; all of them as blocks of 256 rows 643; both on their own
// 30 and 329.)  Where the two kernels meet, fp16 pages, 4 query heads per kv head: 8 tokens (32 rows) here and 9 there, behind 512 cached ones 20.6
// and 23.0 us, 4096: 41.0 and 34.9, 16384: 51.4 and 59.8; 32 sequences of 2048 88.7 and 90.6.
template <class CT, int D, bool EX> static cudaError_t attn_by_rows(const skn_paged *pc, PagedAttn &p) {
    int64_t rows = (int64_t)p.st.max_new * p.group;
    p.above = 0;
    p.upto = INT32_MAX;
    if (rows > SKN_PAGED_PART_ROWS) {
        const bool more = p.st.n_seqs > 1;
        const int few = p.group <= 8 ? 8 : p.group <= 16 ? 16 : SKN_PAGED_PART_ROWS;
        if (more) p.above = few;
        p.direct = 1;
        if (!EX) p.split = more;
        const cudaError_t e = EX ? attn_launch<CT, D, 4, EX>(pc, p) : skn_paged_prompt(CT(), pc, p);
        if (e != cudaSuccess || !more) return e;
        p.above = 0;
        p.upto = few;
        p.parts = pc->d_parts + pc->prompt_parts;
        p.tickets = pc->d_tickets + 2 * pc->n_parts;
    }
    p.direct = p.st.n_seqs > PA_MAX_SEQS;
    if (rows > p.upto) rows = p.upto;
    return rows <= 8 ? attn_launch<CT, D, 1, EX>(pc, p) : rows <= 16 ? attn_launch<CT, D, 2, EX>(pc, p) : attn_launch<CT, D, 4, EX>(pc, p);
}
template <class CT> static cudaError_t attn_by_type(const skn_paged *pc, int32_t io, PagedAttn &p) {
    if (pc->spec.head_dim == 64) return io == SKN_KV_F32 ? attn_by_rows<CT, 64, true>(pc, p) : attn_by_rows<CT, 64, false>(pc, p);
    return io == SKN_KV_F32 ? attn_by_rows<CT, 128, true>(pc, p) : attn_by_rows<CT, 128, false>(pc, p);
}

cudaError_t skn_paged_attn_f16(const skn_paged *pc, int32_t io, PagedAttn &p);
cudaError_t skn_paged_attn_bf16(const skn_paged *pc, int32_t io, PagedAttn &p);
cudaError_t skn_paged_attn_q4(const skn_paged *pc, int32_t io, PagedAttn &p);
