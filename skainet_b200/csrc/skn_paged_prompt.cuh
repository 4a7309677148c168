// Attention of prompts over the paged KV cache: bf16 rows, more of them per kv head than the kernel of skn_paged_attn.cuh takes at a time.
//
// 256 rows (tokens x query heads of one kv head) in two tiles of 128 against 128 keys at a time, on tcgen05: S = Q K^T and O += P V with S, O and P in tensor
// memory (P in 16 bits over its own S: the first operand of the second product), Q, K and V in shared memory with 128-byte swizzle, V
// as the transposed second operand.  A product takes operands of one type, so P is fp16, over bf16 caches bf16: relative errors of 2.1e-3 instead of the 1.64e-3 of an output's own
// rounding.  In two terms it would be 1.64e-3, and a prompt of 8192 tokens 851 us instead of 581, prompts of 129 to 3000 under a window, heads of 64, 126 instead of 89.  A thread of the two softmax warpgroups owns a row: its maximum and sum need no exchange.  The maximum moves only
// when a weight would exceed 2^SLACK; O is then scaled where it is, by the same threads.  While one tile's softmax runs, the tensor cores work
// on the other tile.  Weights are handed over in halves (of 64 keys); in quarters the waits cost more than the earlier start gives (a prompt of 8192
// tokens 534 -> 585 us).  One warp issues the MMAs, one the TMA loads (a box per page, or 128 rows of larger ones).  Q4_0: a warpgroup turns quants
// into fp16 (q - 8) d between the two.
//
// Work is shared out as in skn_paged_attn.cuh: the units (128 keys of a block of rows) of all blocks form one line, one contiguous share for each CTA;
// blocks that lie in several shares are joined by the last of their CTAs to finish.  One warp walks the line for all the others (each for itself
// held its state in registers, which the softmax warps had to spill: 544 -> 512 us; the kernel of Q4_0, at 128 registers, still spills 140 bytes).
//
// Hidden rows of V (behind the last key that the block sees, before its window, on pages that were given back) are cleared in shared memory before the
// product: a warp does it in the few units that have some.  A result that is not finite is computed again from the definition.  Q4_0: fp16 holds
// (q - 8) d up to 65504, so |d| below 2^13.  A larger one would leave minus infinity for some scores, which looks like a hidden key's, so blocks with such a scale become NaN:
// whoever sees them is computed again.
//
// Bound by the chain of a tile (scores, softmax, products, each waiting for the one before) at about half of what the exponentials and the products
// would each take alone.  32 / 8 heads of 128, bf16: a prompt of 8192 tokens 495 us (1110 TFLOP/s, 0.66 of the measured burst), 512 tokens behind 16383 cached
// ones 145 us (960), in 4 bits 182 us; heads of 64: 113 us (615 TFLOP/s: as many exponentials for half the products).  64 tokens alone: 15 us, of which
// 7 before the first product (launch, the line, the first segment, queries).
#pragma once
#include "skn_paged_attn.cuh"

constexpr int PP_ROWS = 256, PP_KEYS = 128;
// units that a block's start and end are worth on the line (2: a prompt of 8192 tokens 705 us, 3: 593, 4: 512, 6: 507, 9: 519; 16 of 1024: 331, 310, 298, 309, 312)
constexpr int PP_COST = 4;

template <class CT, int D> struct PpTraits {
    static constexpr bool Q4 = sizeof(CT) == 1, BF = std::is_same<CT, __nv_bfloat16>::value;
    static constexpr int THREADS = Q4 ? 512 : 384;                // two softmax warpgroups, one of MMA / TMA / clearing, one of unpacking
    static constexpr int TILE = PP_KEYS * D * 2;                  // K or V of a unit in 16 bits; also one tile of Q
    static constexpr int SLOTS = Q4 ? 3 : D == 64 ? 6 : 4;        // K and V in turn
    static_assert(Q4 || SLOTS % 2 == 0, "V always in the same slots");
    static constexpr int HALF = (16 * (D / 2 + D / 16) + 127) / 128 * 128;
    static constexpr int RAW = Q4 ? 8 * HALF : 0, RAW_SLOTS = Q4 ? 4 : 0;
    static constexpr size_t SMEM = 1024 + 2 * TILE + (size_t)SLOTS * TILE + (size_t)RAW_SLOTS * RAW;
    // (a prompt of 8192 tokens: SLACK 0 561 us, 2 530, 4 505, 8 495)
    static constexpr int SLACK = 8;
    static constexpr float LIFT = BF ? 0.f : 7.f;                 // exponent: fp16 weights up to 2^15, so that one of 2^-31 of its row's largest is the last one there
    // registers a thread of the softmax warpgroups, of the MMA / TMA / clearing warpgroup and of the unpacking one: at most the launch's, 384 x 168 or 512 x 128
    static constexpr int REGS_SOFT = Q4 ? 184 : 208, REGS_MMA = Q4 ? 64 : 80, REGS_UNPACK = 80;
    static_assert(128 * (2 * REGS_SOFT + REGS_MMA + (Q4 ? REGS_UNPACK : 0)) <= THREADS * (Q4 ? 128 : 168), "more than the launch has");
};

__device__ __forceinline__ void pp_bar() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ bool pp_any(bool x) {
    uint32_t y;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 2, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(y) : "r"((uint32_t)x) : "memory");
    return y != 0;
}
// B operand that lies [k][64 n] (n contiguous, 128-byte swizzle): 64-wide pieces of n `lead` bytes apart, groups of eight k 1024
__device__ __forceinline__ uint64_t pp_desc_n(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// 32 columns into registers; the caller waits for all of its loads at once
__device__ __forceinline__ void pp_ld32(uint32_t taddr, float *r) {
    uint32_t *u = reinterpret_cast<uint32_t *>(r);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]),
          "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]),
          "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
        : "r"(taddr));
}
// ... after which they may be used (and not before: the empty statements keep the compiler from moving a use up)
template <int N> __device__ __forceinline__ void pp_wait_ld(float *r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(r[i]));
}
__device__ __forceinline__ void pp_st32(uint32_t taddr, const uint32_t *u) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
        ::"r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]),
          "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]),
          "r"(u[27]), "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ uint32_t pp_below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; }      // bits 0 .. n - 1
// 32 bytes of a row, in one store where rows begin at multiples of 32
__device__ __forceinline__ void pp_store32(__nv_bfloat16 *to, const uint32_t *y, bool wide) {
    if (wide)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                     ::"l"(to), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]), "r"(y[4]), "r"(y[5]), "r"(y[6]), "r"(y[7])
                     : "memory");
    else {
        reinterpret_cast<uint4 *>(to)[0] = make_uint4(y[0], y[1], y[2], y[3]);
        reinterpret_cast<uint4 *>(to)[1] = make_uint4(y[4], y[5], y[6], y[7]);
    }
}
__device__ __forceinline__ float pp_max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// 2^x of two values, on the special-function units.  (16 a clock and SM take as long as the products do, but neither is busy for more than half of the time: one in
// eight by a cubic in the fraction instead 534 -> 536 us for a prompt of 8192 tokens, three in eight 623.)
__device__ __forceinline__ uint64_t pp_ex2_pair(uint64_t x) {
    float a, b;
    skn_unpack2(x, a, b);
    return skn_pack2(pa_ex2(a), pa_ex2(b));
}

// The kernel's waits: two seconds are enough for anything but a segment that is computed again (3.3 us a key), for which the other warps wait.  A minute is 18 million keys.
constexpr uint64_t PP_WAIT_NS = 60000000000ull;
__device__ __forceinline__ bool pp_wait(uint64_t *bar, uint32_t parity, int lane) { return tc_wait_warp<PP_WAIT_NS>(bar, parity, lane); }

// A CTA's share of the line, segment by segment: one warp walks it ahead of the others and leaves the segments in shared memory
struct PpWalk {
    long long u, u_end, total, a;               // a: where the present block and head begin
    int n_cta, seq, rb, head;
    PagedSeq sq;
};
__device__ __forceinline__ int pp_blocks(const PagedAttn &p, const PagedSeq &q) { return (q.n * p.group + PP_ROWS - 1) / PP_ROWS; }     // (fewer than 2^30 rows)
__device__ __forceinline__ PagedSpan pp_span(const PagedAttn &p, const PagedSeq &q, int rb) {
    const int r0 = rb * PP_ROWS, r1 = min(r0 + PP_ROWS, q.n * p.group) - 1;
    return paged_span(p, q.len - q.n + r0 / p.group, q.len - q.n + r1 / p.group, PP_KEYS);
}
__device__ __forceinline__ bool pp_next(const PagedAttn &p, PpWalk &w, PagedSegment &g) {
    for (;;) {                                   // the next block of which this share has units
        if (w.u >= w.u_end || w.seq >= p.st.n_seqs) return false;
        if (w.rb < pp_blocks(p, w.sq)) {
            g.span = pp_span(p, w.sq, w.rb);
            const int length = g.span.units + PP_COST, skip = (int)min((long long)(p.st.heads - w.head), paged_div(w.u - w.a, length));
            w.a += (long long)skip * length;
            w.head += skip;
            if (w.head < p.st.heads) {
                g.u0 = (int)max(0LL, w.u - w.a - PP_COST);
                g.u1 = (int)min((long long)g.span.units, w.u_end - w.a - PP_COST);
                w.u = min(w.u_end, w.a + length);
                if (g.u1 > g.u0) break;
            } else {
                w.head = 0;
                ++w.rb;
            }
            continue;
        }
        w.rb = w.head = 0;                       // the next sequence with rows for this launch: a lane each
        for (int s0 = w.seq + 1;; s0 += 32) {
            const int s = s0 + (int)(threadIdx.x & 31);
            PagedSeq sq = {0, 0, 0};
            if (s < p.st.n_seqs) sq = paged_mine(p, s);
            const unsigned have = __ballot_sync(0xffffffffu, sq.n > 0);
            if (have || s0 + 32 >= p.st.n_seqs) {
                const int at = have ? __ffs(have) - 1 : 0;
                w.seq = have ? s0 + at : p.st.n_seqs;
                w.sq.first = __shfl_sync(0xffffffffu, sq.first, at);
                w.sq.n = __shfl_sync(0xffffffffu, sq.n, at);
                w.sq.len = __shfl_sync(0xffffffffu, sq.len, at);
                break;
            }
        }
    }
    g.seq = w.seq; g.head = w.head; g.first = w.sq.first; g.n = w.sq.n; g.len = w.sq.len;
    g.row0 = w.rb * PP_ROWS;
    g.rows = min(PP_ROWS, w.sq.n * p.group - g.row0);
    if (g.u0 == 0 && g.u1 == g.span.units) {     // (the divisions are not free)
        g.c0 = (int)blockIdx.x;
        g.n_parts = 1;
        return true;
    }
    const long long a = w.a + PP_COST;
    g.c0 = (int)paged_div((a + 1) * w.n_cta - 1, w.total);
    g.n_parts = (int)paged_div((a + g.span.units) * w.n_cta - 1, w.total) - g.c0 + 1;
    g.slot = paged_slot(g, (int)blockIdx.x);
    return true;
}

// Whether some key of the segment's unit j is seen by nobody (or may be: the first tokens' last unit and the window's first one count as such)
__device__ __forceinline__ bool pp_hides(const PagedAttn &p, const PagedSegment &g, int j) {
    const int i = g.u0 + j, k0 = (i < g.span.a ? i : i + g.span.gap) * PP_KEYS;
    const int pmin = g.len - g.n + g.row0 / p.group, pmax = g.len - g.n + (g.row0 + g.rows - 1) / p.group;
    const int from = p.window ? max(0, max(0, pmin) - p.window + 1) : 0;
    return k0 + PP_KEYS - 1 > pmax || (k0 < from && k0 + PP_KEYS > p.sinks);
}

template <class CT, int D>
__global__ void __launch_bounds__(PpTraits<CT, D>::THREADS, 1)
skn_paged_prompt_kernel(const __grid_constant__ PagedAttn p, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                        const __grid_constant__ CUtensorMap mks, const __grid_constant__ CUtensorMap mvs) {
    using T = PpTraits<CT, D>;
    using IO = __nv_bfloat16;
    constexpr int THREADS = T::THREADS, SLOTS = T::SLOTS, TILE = T::TILE, NBLK = D / 32;
    extern __shared__ uint8_t raw_smem[];
    uint8_t *const base = reinterpret_cast<uint8_t *>(((uintptr_t)raw_smem + 1023) & ~(uintptr_t)1023);
    uint8_t *const q_tile = base, *const ring = base + 2 * TILE, *const raw_ring = ring + SLOTS * TILE;
    __shared__ uint64_t full[SLOTS], empty[SLOTS], raw_full[4], raw_empty[4];
    __shared__ alignas(16) PagedSegment seg_ring[4];      // no rows: the last one
    __shared__ uint64_t seg_full[4], seg_empty[4];
    __shared__ uint64_t s_full[2], p_full[4], pv_done[2], q_full[2], o_free[2], clean[SLOTS];
    __shared__ long long warp_sum[THREADS / 32];
    __shared__ long long found_at;
    __shared__ int found[2];
    __shared__ uint32_t tmem_slot;
    __shared__ unsigned ticket;
    __shared__ int starts[THREADS + 1];
    __shared__ PagedScratch<D, 256> scratch;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const PagedStep &st = p.st;

    if (tid == 0) {
        for (int i = 0; i < SLOTS; ++i) {
            skn_mbar_init(&full[i], T::Q4 ? 4 : 1);
            skn_mbar_init(&empty[i], 1);
            skn_mbar_init(&clean[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            skn_mbar_init(&raw_full[i], 1);
            skn_mbar_init(&raw_empty[i], 4);
            skn_mbar_init(&seg_full[i], 1);
            skn_mbar_init(&seg_empty[i], T::Q4 ? 14 : 11);        // 8 warps of softmax, MMA, TMA, clearing or 4 of unpacking
        }
        for (int i = 0; i < 2; ++i) {
            skn_mbar_init(&s_full[i], 1);
            skn_mbar_init(&p_full[2 * i], 4);
            skn_mbar_init(&p_full[2 * i + 1], 4);
            skn_mbar_init(&pv_done[i], 1);
            skn_mbar_init(&q_full[i], 4);
            skn_mbar_init(&o_free[i], 4);
        }
        skn_fence_mbar_init();
        found[0] = -1;
    }

    if (p.split) skn_pdl_launch_dependents();        // the launch for short sequences may take the SMs that this one leaves

    // ---- the line: items are the blocks of all sequences, each of them units x heads long ----------------------------------
    PpWalk w;
    {
        // The total first, then the block in which this CTA's share begins (which is known at once where there are no more blocks than threads).
        // Sequences THREADS at a time: where their blocks start, then a block per thread
        long long share = -1, at = 0, x = 0;
        int seq = 0, rb = 0, rounds = 0;             // this thread's block
        for (int pass = 0; pass < 2; ++pass) {
            if (pass && rounds == 1) {
                if (at <= share && share < at + x) {
                    found[0] = seq;
                    found[1] = rb;
                    found_at = at;
                }
                break;
            }
            long long run = 0;
            for (int s0 = 0; s0 < st.n_seqs; s0 += THREADS) {
                const int mine = s0 + tid < st.n_seqs ? pp_blocks(p, paged_mine(p, s0 + tid)) : 0;
                int upto = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += y;
                }
                if (lane == 31) warp_sum[warp] = upto;
                __syncthreads();
                int n_blocks = 0;
                for (int i = 0; i < THREADS / 32; ++i) {
                    if (i < warp) upto += (int)warp_sum[i];
                    n_blocks += (int)warp_sum[i];
                }
                starts[tid] = upto - mine;
                __syncthreads();
                for (int b0 = 0; b0 < n_blocks; b0 += THREADS) {
                    const int b = b0 + tid;
                    x = 0;
                    if (b < n_blocks) {              // the last sequence that starts at or before b (those without blocks start where the next one does)
                        int lo = 0, hi = THREADS - 1;
                        while (lo < hi) {
                            const int mid = (lo + hi + 1) >> 1;
                            if (starts[mid] <= b) lo = mid; else hi = mid - 1;
                        }
                        seq = s0 + lo;
                        rb = b - starts[lo];
                        x = (long long)(pp_span(p, paged_mine(p, seq), rb).units + PP_COST) * st.heads;
                    }
                    long long inc = x;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const long long y = __shfl_up_sync(0xffffffffu, inc, o);
                        if (lane >= o) inc += y;
                    }
                    if (lane == 31) warp_sum[warp] = inc;
                    __syncthreads();
                    at = run + inc - x;
                    for (int i = 0; i < THREADS / 32; ++i) {
                        if (i < warp) at += warp_sum[i];
                        run += warp_sum[i];
                    }
                    if (pass && at <= share && share < at + x) {
                        found[0] = seq;
                        found[1] = rb;
                        found_at = at;
                    }
                    if (pass == 0) ++rounds;
                    __syncthreads();
                }
            }
            if (pass == 0) {
                w.total = run;
                if (run == 0) return;
                const long long want = paged_div(run + PP_COST, PP_COST + 1);        // a CTA for each block of a unit
                w.n_cta = want < (long long)gridDim.x ? (int)want : (int)gridDim.x;
                if ((int)blockIdx.x >= w.n_cta) return;
                share = w.u = paged_div(run * blockIdx.x, w.n_cta);
                w.u_end = paged_div(run * (blockIdx.x + 1), w.n_cta);
            }
        }
        __syncthreads();
        w.seq = found[0];
        w.rb = found[1];
        w.head = 0;
        w.a = found_at;
        w.sq = paged_mine(p, w.seq);
    }
    if (warp == 8) tc_alloc(&tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    PagedSegment g = {};
    uint32_t n_taken = 0;
    bool got = true;                                 // no wait for a segment has run out
    auto take = [&] {                                // the next segment, by a whole warp
        const uint32_t i = n_taken & 3;
        got = got && pp_wait(&seg_full[i], n_taken >> 2 & 1, lane);
        if (!got) return false;
        g = seg_ring[i];
        __syncwarp();
        if (lane == 0) skn_mbar_arrive(&seg_empty[i]);
        ++n_taken;
        return g.rows > 0;
    };

    // ---- softmax: warps 0 .. 3 rows 0 .. 127 of a block, warps 4 .. 7 the others ---------------------------------------------
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(T::REGS_SOFT));
        const int tile = warp >> 2, r = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        const uint32_t ts = tmem + tile * 128 + lanes, to = tmem + 256 + tile * D + lanes;
        uint32_t n_units = 0;                        // of this tile so far
        const bool wide = ((reinterpret_cast<uintptr_t>(p.out) | (uintptr_t)(2 * p.out_stride)) & 31) == 0;
        bool ok = true;                              // once a wait has run out the share is only walked: the barriers below want every warp
        // A segment's queries, this thread's row: for fp16 products times a power of two that brings the row's largest to 2^14 .. 2^15; returns the
        // factor of its scores
        auto load_queries = [&] {
            const int R = tile * 128 + r, t = (g.row0 + R) / p.group;
            const bool real = R < g.rows;
            const uint4 *q = reinterpret_cast<const uint4 *>(static_cast<const IO *>(p.q) + (int64_t)(g.first + t) * p.q_stride + (g.head * p.group + (g.row0 + R) % p.group) * D);
            uint8_t *const qt = q_tile + tile * TILE + r * 128;
            uint4 x[D / 8];
#pragma unroll
            for (int c = 0; c < D / 8; ++c) x[c] = real ? q[c] : make_uint4(0, 0, 0, 0);
            float f = 1.f;
            if constexpr (T::BF) {
                const uint32_t keep = p.scale == 0.f ? 0u : 0xFFFFFFFFu, flip = p.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
                for (int c = 0; c < D / 8; ++c) x[c] = make_uint4((x[c].x ^ flip) & keep, (x[c].y ^ flip) & keep, (x[c].z ^ flip) & keep, (x[c].w ^ flip) & keep);
            } else {
                uint32_t top = 0;                    // largest size, as the bits of a bf16
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    const uint32_t a = __vmaxu2(x[c].x & 0x7FFF7FFFu, x[c].y & 0x7FFF7FFFu), b = __vmaxu2(x[c].z & 0x7FFF7FFFu, x[c].w & 0x7FFF7FFFu);
                    top = __vmaxu2(top, __vmaxu2(a, b));
                }
                top = max(top & 0xFFFFu, top >> 16);
                int e = 14 - ((int)(top >> 7) - 127);
                e = top > 0 && top < 0x7F80u ? max(-120, min(120, e)) : 0;
                const float up = p.scale == 0.f ? 0.f : __uint_as_float((uint32_t)(127 + e) << 23) * (p.scale < 0.f ? -1.f : 1.f);
                f = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    uint32_t y[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] = pack_f16(__uint_as_float(y[i] << 16) * up, __uint_as_float(y[i] & 0xFFFF0000u) * up);
                    x[c] = make_uint4(y[0], y[1], y[2], y[3]);
                }
            }
#pragma unroll
            for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint4 *>(qt + (c >> 3) * 16384 + (((c & 7) ^ (r & 7)) << 4)) = x[c];
            skn_fence_proxy_async();
            __syncwarp();
            if (lane == 0) skn_mbar_arrive(&q_full[tile]);
            // (a scale of zero moves into the queries: hidden scores of minus infinity stay what they are)
            return (p.scale == 0.f ? 1.f : fabsf(p.scale)) * f;
        };
        bool more = take();
        more = !pp_any(!got) && more;                // (the barriers below want every warp)
        float cs_next = 0.f;
        if (more && tile * 128 < g.rows) cs_next = load_queries();
        while (more) {
            const PagedSegment now = g;              // g: the next one, whose queries are handed over before this one's outputs are written
            const int R = tile * 128 + r;
            const bool real = R < now.rows, used = tile * 128 < now.rows;
            const int t = (now.row0 + R) / p.group, pos = real ? now.len - now.n + t : -1;
            const float cs = cs_next;
            float m = PA_NONE, l = cs < INFINITY ? 0.f : cs - cs;        // (a factor beyond fp32 makes scores of minus infinity, as of hidden keys: computed again)
            if (used && ok) {
                const int ta = (now.row0 + tile * 128) / p.group, tb = (now.row0 + min(tile * 128 + 127, now.rows - 1)) / p.group;
                const int pmin = now.len - now.n + ta, pmax = now.len - now.n + tb;

                for (int j = 0; j < now.u1 - now.u0; ++j, ++n_units) {
                    const int i = now.u0 + j, k0 = (i < now.span.a ? i : i + now.span.gap) * PP_KEYS;
                    if (!pp_wait(&s_full[tile], n_units & 1, lane)) { ok = false; break; }
                    tc_fence_after();
                    float v[PP_KEYS];
#pragma unroll
                    for (int c = 0; c < 4; ++c) pp_ld32(ts + 32 * c, v + 32 * c);
                    pp_wait_ld<PP_KEYS>(v);
                    const bool whole = k0 + PP_KEYS - 1 <= pmin && (!p.window || k0 > pmax - p.window || k0 + PP_KEYS <= p.sinks);
                    if (!whole) {
                        const int hi = pos - k0, lo = p.window ? pos - p.window + 1 - k0 : -1, sk = p.sinks - k0;
#pragma unroll
                        for (int b = 0; b < PP_KEYS; b += 32) {
                            const uint32_t seen = pp_below(hi + 1 - b) & (~pp_below(lo - b) | pp_below(sk - b));
#pragma unroll
                            for (int c = 0; c < 32; ++c) v[b + c] = seen >> c & 1 ? v[b + c] : -INFINITY;
                        }
                    }
                    float top = pp_max3(v[0], v[1], v[2]), top2 = pp_max3(v[3], v[4], v[5]);     // (a NaN stays one)
#pragma unroll
                    for (int c = 6; c < 126; c += 4) {
                        top = pp_max3(top, v[c], v[c + 1]);
                        top2 = pp_max3(top2, v[c + 2], v[c + 3]);
                    }
                    top = pp_max3(top, v[126], v[127]);
                    top = pp_max3(top, top2, top2);
                    if (top != top) l = top;
                    top *= cs;
                    if (__any_sync(0xffffffffu, top > m + (float)T::SLACK)) {
                        const float fresh = fmaxf(m, top), fix = pa_ex2(m - fresh);
                        m = fresh;
                        l *= fix;
                        if (j > 0) {
                            if (!pp_wait(&pv_done[tile], (n_units - 1) & 1, lane)) { ok = false; break; }
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < D; c += 32) {
                                float o[32];
                                pp_ld32(to + c, o);
                                pp_wait_ld<32>(o);
#pragma unroll
                                for (int k = 0; k < 32; ++k) o[k] *= fix;
                                pp_st32(to + c, reinterpret_cast<uint32_t *>(o));
                            }
                            tc_wait_st();
                        }
                    }
                    const uint64_t cs2 = skn_pack2(cs, cs), off2 = skn_pack2(T::LIFT - m, T::LIFT - m);
                    uint64_t sum = 0, sum2 = 0;      // (two chains of 32 additions; one of 64: 533 -> 547 us for a prompt of 8192 tokens)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t pk[32];
#pragma unroll
                        for (int c = 0; c < 32; ++c) {
                            const uint64_t x = skn_fma2(skn_pack2(v[64 * h + 2 * c], v[64 * h + 2 * c + 1]), cs2, off2);
                            const uint64_t y = pp_ex2_pair(x);
                            (c & 1 ? sum : sum2) = skn_add2(c & 1 ? sum : sum2, y);
                            float a, b;
                            skn_unpack2(y, a, b);
                            pk[c] = T::BF ? pack_bf16(a, b) : pack_f16(a, b);
                        }
                        pp_st32(ts + 32 * h, pk);
                        tc_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) skn_mbar_arrive(&p_full[2 * tile + h]);
                    }
                    float a, b;
                    skn_unpack2(skn_add2(sum, sum2), a, b);
                    l += a + b;
                }
            }
            // the next segment's queries: these are done with since the last scores
            more = take();
            if (more && tile * 128 < g.rows) cs_next = load_queries();
            // ---- out, or to the other CTAs of the block -------------------------------------------------------------------------
            const bool shared = now.n_parts > 1;
            float *part = p.parts + (int64_t)now.slot * PP_ROWS * (D + 4);          // [D / 4][256] float4, then [256] maximum, [256] sum
            IO *const out = static_cast<IO *>(p.out) + (int64_t)(now.first + t) * p.out_stride + (now.head * p.group + (now.row0 + R) % p.group) * D;
            bool odd = false;
            if (used) {
                if (ok) ok = pp_wait(&pv_done[tile], (n_units - 1) & 1, lane);
                if (!(ok && got) && lane == 0) *st.status = SKN_ERR_TIMEOUT;
                tc_fence_after();
                const float inv = 1.f / l;
                const uint32_t none = now.len - now.n + t < 0 ? 0u : 0x7FFF7FFFu;      // without a weight: zero where nothing is seen, NaN where all scores were minus infinity
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    float o[32];
                    pp_ld32(to + c, o);
                    pp_wait_ld<32>(o);
                    if (c + 32 == D) {               // the accumulators may be written again
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) skn_mbar_arrive(&o_free[tile]);
                    }
                    float s = 0.f;
#pragma unroll
                    for (int k = 0; k < 32; ++k) s += o[k];
                    odd |= !(fabsf(s) < INFINITY);
                    if (shared) {
#pragma unroll
                        for (int k = 0; k < 32; k += 4) reinterpret_cast<float4 *>(part)[((c + k) / 4) * PP_ROWS + R] = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                    } else {
                        uint32_t y[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) y[k] = l == 0.f ? none : pack_bf16(o[2 * k] * inv, o[2 * k + 1] * inv);
                        if (real) {
#pragma unroll
                            for (int k = 0; k < 16; k += 8) pp_store32(out + c + 2 * k, y + k, wide);
                        }
                    }
                }
                odd = real && (odd || !(fabsf(l) < INFINITY));
                if (shared) {
                    part[D * PP_ROWS + R] = m;
                    part[(D + 1) * PP_ROWS + R] = l;
                }
            }
            if (pp_any(!got)) more = false;
            if (pp_any(odd)) {
                const PagedSegment again = now;      // (a copy: the address of the one that the loops use is not taken)
                paged_redo<CT, D, 256, IO>(p, again, PP_KEYS, scratch, [] { pp_bar(); }, [=, &p](int row, float rm, float rl, float acc) {
                    const int tr = (now.row0 + row) / p.group;
                    if (shared) {
                        if (tid < D) part[((tid / 4) * PP_ROWS + row) * 4 + (tid & 3)] = acc;
                        if (tid == 0) {
                            part[D * PP_ROWS + row] = rm + T::LIFT;      // (its weights are not lifted)
                            part[(D + 1) * PP_ROWS + row] = rl;
                        }
                    } else if (tid < D)
                        static_cast<IO *>(p.out)[(int64_t)(now.first + tr) * p.out_stride + (now.head * p.group + (now.row0 + row) % p.group) * D + tid] =
                            __float2bfloat16_rn(rl != 0.f ? acc / rl : now.len - now.n + tr < 0 ? 0.f : NAN);
                });
            }
            if (shared) {
                __threadfence();
                pp_bar();
                if (tid == 0) ticket = atomicInc(&p.tickets[paged_slot(now, now.c0)], (unsigned)now.n_parts - 1);
                pp_bar();
                if (ticket == (unsigned)now.n_parts - 1 && real) {
                    __threadfence();
                    auto part_of = [&](int k) { return p.parts + (int64_t)paged_slot(now, now.c0 + min(k, now.n_parts - 1)) * PP_ROWS * (D + 4); };
                    float top = PA_NONE, sum = 0.f;
                    for (int k = 0; k < now.n_parts; ++k) top = fmaxf(top, __ldcg(part_of(k) + D * PP_ROWS + R));
                    for (int k = 0; k < now.n_parts; ++k) sum = fmaf(__ldcg(part_of(k) + (D + 1) * PP_ROWS + R), exp2f(__ldcg(part_of(k) + D * PP_ROWS + R) - top), sum);
                    const float inv = 1.f / sum;
                    const uint32_t none = now.len - now.n + t < 0 ? 0u : 0x7FFF7FFFu;
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) {
                        float4 o[4] = {};
                        for (int k = 0; k < now.n_parts; k += 4) {       // four parts' loads on their way at once
                            float4 y[4][4];
                            float f[4];
#pragma unroll
                            for (int b = 0; b < 4; ++b) {
                                f[b] = k + b < now.n_parts ? exp2f(__ldcg(part_of(k + b) + D * PP_ROWS + R) - top) : 0.f;
#pragma unroll
                                for (int e = 0; e < 4; ++e) y[b][e] = __ldcg(reinterpret_cast<const float4 *>(part_of(k + b)) + (c / 4 + e) * PP_ROWS + R);
                            }
#pragma unroll
                            for (int b = 0; b < 4; ++b)
                                if (f[b] != 0.f)
#pragma unroll
                                    for (int e = 0; e < 4; ++e) {
                                        o[e].x = fmaf(y[b][e].x, f[b], o[e].x); o[e].y = fmaf(y[b][e].y, f[b], o[e].y);
                                        o[e].z = fmaf(y[b][e].z, f[b], o[e].z); o[e].w = fmaf(y[b][e].w, f[b], o[e].w);
                                    }
                        }
                        uint32_t y[8];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            y[2 * e] = sum == 0.f ? none : pack_bf16(o[e].x * inv, o[e].y * inv);
                            y[2 * e + 1] = sum == 0.f ? none : pack_bf16(o[e].z * inv, o[e].w * inv);
                        }
                        pp_store32(out + c, y, wide);
                    }
                }
                pp_bar();                            // (the ticket is read)
            }
        }
    }
    // ---- MMAs: warp 8 --------------------------------------------------------------------------------------------------------
    else if (warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T::REGS_MMA));
    if (warp == 8) {
        constexpr uint32_t FMT = T::BF ? 1u << 7 | 1u << 10 : 0u;
        constexpr uint32_t ID_S = 1u << 4 | FMT | (PP_KEYS >> 3) << 17 | 8u << 24, ID_O = 1u << 4 | FMT | 1u << 16 | (D >> 3) << 17 | 8u << 24;
        int slot = 0, parity = 0;                    // of the next K or V
        uint32_t units[2] = {0, 0}, segs[2] = {0, 0};
        bool ok = true;
        auto step = [&] {
            if (++slot == SLOTS) {
                slot = 0;
                parity ^= 1;
            }
        };
        auto scores = [&](int tile, int at) {        // S of a tile from the keys in slot `at`
            const uint32_t qa = skn_smem_u32(q_tile + tile * TILE), ka = skn_smem_u32(ring + at * TILE);
            if (tc_elect()) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t off = (k >> 2) * 16384 + (k & 3) * 32;
                    tc_mma_bf16(tmem + tile * 128, tc_smem_desc(qa + off), tc_smem_desc(ka + off), ID_S, k > 0);
                }
                tc_commit(&s_full[tile]);
            }
            __syncwarp();
        };
        while (ok && take()) {
            const int n = g.u1 - g.u0, tiles = g.rows > 128 ? 2 : 1;
            int k_slot = slot;
            for (int x = 0; x < tiles && ok; ++x) ok = pp_wait(&q_full[x], segs[x] & 1, lane);
            ok = ok && pp_wait(&full[slot], parity, lane);
            if (!ok) break;
            tc_fence_after();
            for (int x = 0; x < tiles; ++x) scores(x, slot);
            if (tc_elect()) tc_commit(&empty[k_slot]);
            __syncwarp();
            step();
            for (int j = 0; j < n && ok; ++j) {
                const int v_slot = slot;
                ok = pp_wait(T::Q4 ? &full[slot] : &clean[slot], parity, lane);
                step();
                const bool more = j + 1 < n;
                k_slot = slot;
                const uint32_t va = skn_smem_u32(ring + v_slot * TILE);
                for (int x = 0; x < tiles && ok; ++x) {
                    for (int h = 0; h < 2 && ok; ++h) {          // the weights come in halves
                        ok = pp_wait(&p_full[2 * x + h], units[x] & 1, lane);
                        if (ok && j == 0 && h == 0 && segs[x] > 0) ok = pp_wait(&o_free[x], (segs[x] - 1) & 1, lane);
                        if (!ok) break;
                        tc_fence_after();
                        if (tc_elect()) {
#pragma unroll
                            for (int k = 4 * h; k < 4 * h + 4; ++k)
                                tc_mma_ts(tmem + 256 + x * D, tmem + x * 128 + 8 * k, pp_desc_n(va + k * 2048, PP_KEYS * 128), ID_O, j > 0 || k > 0);
                            if (h) {
                                tc_commit(&pv_done[x]);
                                if (x == tiles - 1) tc_commit(&empty[v_slot]);
                            }
                        }
                        __syncwarp();
                    }
                    if (!ok) break;
                    ++units[x];
                    if (more) {
                        if (x == 0) ok = pp_wait(&full[k_slot], parity, lane);
                        if (!ok) break;
                        tc_fence_after();
                        scores(x, k_slot);
                        if (x == tiles - 1) {
                            if (tc_elect()) tc_commit(&empty[k_slot]);
                            __syncwarp();
                        }
                    }
                }
                if (more) step();
            }
            for (int x = 0; x < tiles; ++x) ++segs[x];
        }
        if (!(ok && got) && lane == 0) *st.status = SKN_ERR_TIMEOUT;
    }
    // ---- loads: warp 9 -----------------------------------------------------------------------------------------------------------
    else if (warp == 9) {
        int slot = 0, parity = 0;
        bool ok = true;
        uint32_t loads = 0;
        while (ok && take()) {
            const int n = g.u1 - g.u0;
            const int pmin = g.len - g.n + g.row0 / p.group, pmax = g.len - g.n + (g.row0 + g.rows - 1) / p.group;
            const int seen_from = p.window ? max(0, max(0, pmin) - p.window + 1) : 0;
            // a box is a page's rows, up to 128 (Q4_0: 32); a lane per box of K (16-bit types: and half of the dims)
            const int box_shift = T::Q4 ? min(st.page_shift, 5) : min(st.page_shift, 7), boxes = PP_KEYS >> box_shift;
            for (int j = 0; j < n && ok; ++j) {
                const int i = g.u0 + j, k0 = (i < g.span.a ? i : i + g.span.gap) * PP_KEYS;
                int page = -1;
                const int b = lane & (boxes - 1), kb = k0 + (b << box_shift);
                if (lane < boxes * (T::Q4 ? 1 : D / 64)) {
                    bool need = false;               // some row sees some of the box
                    for (int k = kb; k < kb + (1 << box_shift); k += 16) need |= k <= pmax && (k + 15 >= seen_from || k < p.sinks);
                    if (need) page = paged_page(st, g.seq, kb);
                }
                const int count = __popc(__ballot_sync(0xffffffffu, page >= 0));
                const int row = kb & ((1 << st.page_shift) - 1);
                for (int kv = 0; kv < 2 && ok; ++kv) {
                    const CUtensorMap *map = kv ? &mv : &mk;
                    if constexpr (!T::Q4) {
                        if (loads >= (uint32_t)SLOTS) ok = pp_wait(&empty[slot], parity ^ 1, lane);
                        if (!ok) break;
                        uint8_t *dst = ring + slot * TILE;
                        if (lane == 0) {
                            if (count) skn_mbar_expect_tx(&full[slot], (uint32_t)count << box_shift << 7);
                            else skn_mbar_arrive(&full[slot]);
                        }
                        __syncwarp();
                        if (page >= 0) {
                            const int h = lane / boxes;
                            tma_3d(dst + h * 16384 + (b << box_shift) * 128, map, 0, ((page * st.heads + g.head) << st.page_shift) + row, h, &full[slot]);
                        }
                        ++loads;
                        if (++slot == SLOTS) {
                            slot = 0;
                            parity ^= 1;
                        }
                    } else {
                        if (loads >= 4) ok = pp_wait(&raw_empty[slot], parity ^ 1, lane);
                        if (!ok) break;
                        uint8_t *dst = raw_ring + slot * T::RAW + ((b << box_shift) >> 4) * T::HALF;
                        if (lane == 0) {
                            if (count) skn_mbar_expect_tx(&raw_full[slot], ((uint32_t)count << box_shift) * (D / 2 + D / 16));
                            else skn_mbar_arrive(&raw_full[slot]);
                        }
                        __syncwarp();
                        if (page >= 0) {
                            tma_3d(dst, map, row * 4, 0, page * st.heads + g.head, &raw_full[slot]);
                            tc_tma_load_2d(dst + (D / 2 << box_shift), kv ? &mvs : &mks, row * (D / 64), page * st.heads + g.head, &raw_full[slot]);
                        }
                        ++loads;
                        if (++slot == 4) {
                            slot = 0;
                            parity ^= 1;
                        }
                    }
                }
            }
        }
        if (!(ok && got) && lane == 0) *st.status = SKN_ERR_TIMEOUT;
        // nothing is on its way when the CTA ends: every load is waited for by who reads it, unless a wait ran out
        if (!(ok && got))
            for (int i = 0; i < (T::Q4 ? 4 : SLOTS); ++i) {
                uint64_t *bar = T::Q4 ? &raw_full[i] : &full[i];
                tc_wait_warp(bar, i < slot ? parity : parity ^ 1, lane);
            }
    }
    // ---- 16-bit types: rows of V that nobody sees are cleared, warp 10 -------------------------------------------------------------
    else if (!T::Q4 && warp == 10) {
        int slot = 0, parity = 0;
        bool ok = true;
        auto step = [&] {
            if (++slot == SLOTS) {
                slot = 0;
                parity ^= 1;
            }
        };
        while (ok && take()) {
            const int pmin = g.len - g.n + g.row0 / p.group, pmax = g.len - g.n + (g.row0 + g.rows - 1) / p.group;
            const int seen_from = p.window ? max(0, max(0, pmin) - p.window + 1) : 0;
            for (int j = 0; j < g.u1 - g.u0 && ok; ++j) {
                step();                              // K
                ok = pp_wait(&full[slot], parity, lane);
                if (!ok) break;
                if (pp_hides(p, g, j)) {
                    const int i = g.u0 + j, k0 = (i < g.span.a ? i : i + g.span.gap) * PP_KEYS;
                    uint8_t *v = ring + slot * TILE;
                    for (int x = lane; x < PP_KEYS * (D / 8); x += 32) {
                        const int row = x / (D / 8), c = x % (D / 8), key = k0 + row;
                        if (!(key <= pmax && (key >= seen_from || key < p.sinks))) *reinterpret_cast<uint4 *>(v + (c >> 3) * 16384 + row * 128 + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
                    }
                    skn_fence_proxy_async();
                    __syncwarp();
                }
                if (lane == 0) skn_mbar_arrive(&clean[slot]);      // V lies in every second slot: once a round
                step();
            }
        }
        if (!(ok && got) && lane == 0) *st.status = SKN_ERR_TIMEOUT;
    }
    // ---- the walk: warp 11 ------------------------------------------------------------------------------------------------------------
    else if (warp == 11) {
        bool ok = true;
        uint32_t k = 0;
        for (bool more = true; more; ++k) {
            more = pp_next(p, w, g);
            if (!more) g.rows = 0;
            if (k >= 4 && !pp_wait(&seg_empty[k & 3], (k >> 2 & 1) ^ 1, lane)) {
                ok = false;
                break;
            }
            if (lane == 0) {
                seg_ring[k & 3] = g;
                skn_mbar_arrive(&seg_full[k & 3]);
            }
            __syncwarp();
        }
        if (!ok && lane == 0) *st.status = SKN_ERR_TIMEOUT;
    }
    }
    // ---- Q4_0: quants to fp16, warps 12 .. 15, a key per thread -----------------------------------------------------------------------
    else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T::REGS_UNPACK));
        int slot = 0, parity = 0, raw = 0, raw_parity = 0;
        uint32_t tiles = 0;
        bool ok = true;
        const int row = tid & 127;
        while (ok && take()) {
            const int pmin = g.len - g.n + g.row0 / p.group, pmax = g.len - g.n + (g.row0 + g.rows - 1) / p.group;
            const int seen_from = p.window ? max(0, max(0, pmin) - p.window + 1) : 0;
            for (int j = 0; j < g.u1 - g.u0 && ok; ++j) {
                const int i = g.u0 + j, key = (i < g.span.a ? i : i + g.span.gap) * PP_KEYS + row;
                const bool need = key <= pmax && (key >= seen_from || key < p.sinks);
                for (int kv = 0; kv < 2; ++kv) {
                    ok = pp_wait(&raw_full[raw], raw_parity, lane);
                    if (ok && tiles >= (uint32_t)SLOTS) ok = pp_wait(&empty[slot], parity ^ 1, lane);
                    if (!ok) break;
                    const int box_shift = min(st.page_shift, 5), in = row & ((1 << box_shift) - 1);
                    const uint8_t *src = raw_ring + raw * T::RAW + ((row - in) >> 4) * T::HALF;
                    uint8_t *dst = ring + slot * TILE + row * 128;
#pragma unroll
                    for (int b = 0; b < NBLK; ++b) {
                        uint4 u = need ? *reinterpret_cast<const uint4 *>(src + (((b << box_shift) + in) << 4)) : make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
                        __half_raw dr = {need ? *reinterpret_cast<const unsigned short *>(src + (D / 2 << box_shift) + (in * NBLK + b) * 2) : (unsigned short)0};
                        if ((dr.x & 0x7000) == 0x7000) dr.x = 0x7FFF;        // from 2^13 on: see the head of this file
                        const __half d = dr;
                        const __half2 d2 = __half2half2(d), off = __float2half2_rn(-1032.f);
                        const uint32_t ws[4] = {u.x, u.y, u.z, u.w};
                        uint32_t h[16];
#pragma unroll
                        for (int x = 0; x < 4; ++x)
#pragma unroll
                            for (int hi = 0; hi < 2; ++hi) {
                                const uint32_t n = (hi ? ws[x] >> 4 : ws[x]) & 0x0F0F0F0Fu;
#pragma unroll
                                for (int y = 0; y < 2; ++y) {
                                    const uint32_t z = __byte_perm(n, 0x64646464u, y ? 0x4342 : 0x4140);
                                    const __half2 v = __hmul2(__hadd2(*reinterpret_cast<const __half2 *>(&z), off), d2);
                                    h[8 * hi + 2 * x + y] = *reinterpret_cast<const uint32_t *>(&v);
                                }
                            }
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const int c = 4 * b + x;
                            *reinterpret_cast<uint4 *>(dst + (c >> 3) * 16384 + (((c & 7) ^ (row & 7)) << 4)) = make_uint4(h[4 * x], h[4 * x + 1], h[4 * x + 2], h[4 * x + 3]);
                        }
                    }
                    skn_fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) {
                        skn_mbar_arrive(&raw_empty[raw]);
                        skn_mbar_arrive(&full[slot]);
                    }
                    ++tiles;
                    if (++raw == 4) {
                        raw = 0;
                        raw_parity ^= 1;
                    }
                    if (++slot == SLOTS) {
                        slot = 0;
                        parity ^= 1;
                    }
                }
            }
        }
        if (!(ok && got) && lane == 0) *st.status = SKN_ERR_TIMEOUT;
    }
    __syncthreads();
    tc_fence_after();
    if (warp == 8) tc_dealloc(tmem, 512);
}

template <class CT, int D> static cudaError_t prompt_launch(const skn_paged *pc, const PagedAttn &p) {
    using T = PpTraits<CT, D>;
    auto *kern = skn_paged_prompt_kernel<CT, D>;
    static uint64_t done = 0;
    const cudaError_t e = paged_attributes(kern, T::SMEM, pc->ctx->device, &done);
    if (e != cudaSuccess) return e;
    kern<<<pc->ctx->sm_count, T::THREADS, T::SMEM, pc->ctx->stream>>>(p, pc->wide[0], pc->wide[1], pc->wide[2], pc->wide[3]);
    return cudaGetLastError();
}
