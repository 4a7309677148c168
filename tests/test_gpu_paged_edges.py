"""Paged KV cache on the GPU: values, steps and calls at the edges of what it takes, against the oracle in 64 bits (tolerances as in
test_gpu_paged.py)."""
import ctypes
import threading

import numpy as np
import pytest
import torch

import skainet_b200 as skn
from oracle import paged as oracle
from skainet_b200.parallel import Exchange
from test_gpu_paged import IO, Step, bf16, check, filled, run_attend, tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,news", [([300], [40]), ([300, 70], [1, 1]), ([2100, 40], [33, 20]), ([260], [260])])
def test_keys_beyond_fp16_in_4_bits(ctx, io, dim, lens, news):
    """A 4-bit block holds values up to 8 x 65504.  One dimension of every key is 1e5, of which queries of either sign (and of none) make scores of +-1e4; then
    keys whose value beyond fp16 meets another one that brings the score back.  Every row's block is computed in fp32: no term for rows in fp16.  (No bound
    on the norm: a score of 1e4 in fp32 is a multiple of 2^-10, by which a weight is off.)"""
    kv, group, page = 2, 4, 32
    for kind in range(2):
        step = Step(5, lens, news, page)
        cache = skn.PagedKVCache(ctx, step.n_pages, page, kv, dim, "q4_0")
        ref = oracle.Pages(step.n_pages, page, kv, dim, "q4_0")
        g = np.random.default_rng(dim + kind)
        total = int(step.lens.sum())
        k, v = (g.standard_normal((total, kv, dim)).astype(np.float32) for _ in range(2))
        q = bf16(g.standard_normal((step.n, kv * group, dim)))
        if kind == 0:
            k[:, :, 5] = 1e5
            q[:, :, 5] = np.array([-1, 1, -0.5, 0])[np.arange(kv * group) % 4]
        else:                                              # -7e4 + 6e4 or -1e4
            k[:, :, 5], k[:, :, 40] = 0, -1e4
            k[::2, :, 5], k[::2, :, 40] = 7e4, 6e4
            q[:, :, 5], q[:, :, 40] = -1, 1
        cache.append(k, v, step.table, step.full, step.lens)
        ref.append(k, v, step.table, step.full, step.lens)
        want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, 0.125)
        assert np.isfinite(want).all() and np.abs(want).max() > 0.1
        err = np.abs(run_attend(cache, step, q, io, scale=0.125) - want)
        tol = tolerance(want, mass, reach, 0.0 if io == "f32" else 2.0 ** -11, 0.0, io)
        assert np.all(err <= tol), f"largest excess {np.max(err / tol):.3g} at {np.unravel_index(np.argmax(err / tol), err.shape)}"
        cache.close()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,news,some", [([40], [40], 10), ([70, 20], [1, 1], 70), ([3000], [60], 3000), ([3000, 5], [60, 1], 2970), ([9, 300], [12, 40], 6)])
def test_scores_of_minus_infinity(ctx, io, dtype, lens, news, some):
    """The first `some` keys hold minus infinity in one dimension: with a positive query their weights are zero, and 0 / 0 where all visible ones are such.
    Rows at negative positions see nothing and are zero; with a query of the other sign (or of none) everything is NaN."""
    kv, group, dim, page = 1, 4, 64, 16
    step = Step(5, lens, news, page)
    cache, ref = filled(ctx, step, kv, dim, dtype, 3)
    g = np.random.default_rng(7)
    n = int(np.maximum(step.lens, 0).sum())
    k, v = (g.standard_normal((n, kv, dim)).astype(np.float32) for _ in range(2))
    at = np.concatenate([np.arange(int(x)) for x in step.lens])
    k[at < some, 0, 3] = -np.inf
    q = bf16(g.standard_normal((step.n, kv * group, dim)))
    q[:, :, 3] = np.array([1, 2, -1, 0.25])
    cache.append(k, v, step.table, step.full, step.lens)
    ref.append(k, v, step.table, step.full, step.lens)
    with np.errstate(invalid="ignore"):
        want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, 0.125)
    out = run_attend(cache, step, q, io, scale=0.125)
    odd = np.isnan(want)
    assert odd[:, 2].any() and np.array_equal(np.isnan(out), odd)
    reach[..., 0] = np.where(np.isfinite(reach[..., 0]), reach[..., 0], 0.125 * 6 * dim)      # |k| and |q| below 6, a product a dimension: no more for keys with a weight
    rows = ~odd.any(axis=2)
    check(out[rows], want[rows], mass[rows], reach[rows], io, dtype, max(news) > 1)
    cache.close()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("dtype,key,query", [("bf16", 2.0 ** 40, 2.0 ** 75), ("f16", 2.0 ** 10, 2.0 ** 105), ("q4_0", 2.0 ** 10, 2.0 ** 105)])
@pytest.mark.parametrize("lens,news", [([60], [1]), ([60, 30], [40, 1]), ([5000], [50]), ([5000, 9], [1, 1])])
def test_scores_far_below_zero(ctx, io, dtype, key, query, lens, news):
    """scores of about -1e33 and less, distances as large: every row is the value of the key that is least far below, which is drawn anew every 50 tokens"""
    kv, group, dim, page = 2, 4, 64, 16
    step = Step(5, lens, news, page)
    cache = skn.PagedKVCache(ctx, step.n_pages, page, kv, dim, dtype)
    ref = oracle.Pages(step.n_pages, page, kv, dim, dtype)
    g = np.random.default_rng(3)
    total = int(step.lens.sum())
    k = np.zeros((total, kv, dim), dtype=np.float32)
    at = np.concatenate([np.arange(int(x)) for x in step.lens])
    k[:, :, 0] = key * (1 + ((at * 29 + 11) % 50)[:, None] / 64)                     # exact in every type
    k[at >= 50, :, 0] = key * 2                                                       # ... and twice as far from the 50th on
    v = g.standard_normal((total, kv, dim)).astype(np.float32)
    q = np.zeros((step.n, kv * group, dim), dtype=np.float32)
    q[:, :, 0] = -query
    cache.append(k, v, step.table, step.full, step.lens)
    ref.append(k, v, step.table, step.full, step.lens)
    want, _, _ = ref.attend(q, step.table, step.starts, step.lens, 0.125)
    assert np.abs(want).max() > 1
    out = run_attend(cache, step, q, io, scale=0.125)
    # one weight of one: an output is the value itself, rounded (bf16 rows) or summed and divided in fp32
    assert np.all(np.abs(out - want) <= (2.0 ** -8 if io == "bf16" else 2.0 ** -20) * np.abs(want))
    cache.close()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("lens,news", [([60], [1]), ([60, 30], [40, 1]), ([3000, 9], [1, 1])])
def test_queries_near_the_largest_number(ctx, io, lens, news):
    """queries of -2^122 and 4-bit keys of 2^-17: scores of -2^102, though the factor between the quants' products and the scores is more than fp32 holds"""
    kv, group, dim, page = 2, 4, 64, 16
    step = Step(5, lens, news, page)
    cache = skn.PagedKVCache(ctx, step.n_pages, page, kv, dim, "q4_0")
    ref = oracle.Pages(step.n_pages, page, kv, dim, "q4_0")
    g = np.random.default_rng(3)
    total = int(step.lens.sum())
    k = np.zeros((total, kv, dim), dtype=np.float32)
    at = np.concatenate([np.arange(int(x)) for x in step.lens])
    k[:, :, 0] = 2.0 ** -21 * (16 + (at * 29 + 11) % 50 + 50 * (at >= 50))[:, None]      # 8 times a multiple of 2^-24
    v = g.standard_normal((total, kv, dim)).astype(np.float32)
    q = np.zeros((step.n, kv * group, dim), dtype=np.float32)
    q[:, :, 0] = -2.0 ** 122
    cache.append(k, v, step.table, step.full, step.lens)
    ref.append(k, v, step.table, step.full, step.lens)
    want, _, _ = ref.attend(q, step.table, step.starts, step.lens, 0.125)
    assert np.abs(want).max() > 1
    out = run_attend(cache, step, q, io, scale=0.125)
    # fp32: distances between scores of 2^98 and more leave one weight of one; equal keys none twice among the nearest
    assert np.all(np.abs(out - want) <= (2.0 ** -8 if io == "bf16" else 2.0 ** -20) * np.abs(want))
    cache.close()


def test_scales_beyond_fp32_are_refused(ctx):
    """scores are formed in base 2: the scale times log2(e) is a number too"""
    step = Step(3, [40], [2], 16)
    cache, _ = filled(ctx, step, 2, 64, "bf16", 3)
    q = torch.zeros(2, 4, 64, device="cuda", dtype=torch.bfloat16)
    for scale in (3e38, -3e38, float("inf")):
        with pytest.raises(skn.SknError, match="scale"):
            cache.attend(np.zeros((2, 4, 64), dtype=np.float32), step.table, step.starts, step.lens, scale=scale)
        with pytest.raises(skn.SknError, match="scale"):
            cache.attend_dev(step.batch(), q, torch.zeros_like(q), scale=scale)
    cache.close()


@pytest.mark.parametrize("dim", [64, 128])
def test_small_queries_beside_a_large_one(ctx, dim):
    """Single tokens over 4 bits: queries of bf16 rows are multiples of 2^-34 of the row's largest there (2^-38 over other caches).  The largest meets zeros, the
    others, around 2^-33 of it, keys of 1e4."""
    for dtype, step_of in (("q4_0", -34), ("f16", -38)):
        step = Step(5, [200, 17], [1, 1], 32)
        kv, group = 2, 4
        cache = skn.PagedKVCache(ctx, step.n_pages, 32, kv, dim, dtype)
        ref = oracle.Pages(step.n_pages, 32, kv, dim, dtype)
        g = np.random.default_rng(dim)
        total = int(step.lens.sum())
        k, v = (g.standard_normal((total, kv, dim)).astype(np.float32) for _ in range(2))
        k[:, :, :32] = 0
        k *= 1e4
        q = g.integers(-6, 7, (step.n, kv * group, dim)) * np.exp2(20.0 + step_of)
        q[:, :, 0] = 2.0 ** 20
        q = bf16(q)
        cache.append(k, v, step.table, step.full, step.lens)
        ref.append(k, v, step.table, step.full, step.lens)
        want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, 0.125)
        check(run_attend(cache, step, q, "bf16", scale=0.125), want, mass, reach, "bf16", dtype, False)
        cache.close()


@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_values_of_unequal_blocks(ctx, io):
    """4 bits, single tokens: values of the first 32 dimensions are 2^20 times the others'.  A key's part may miss 2^-32 (2^-37) of the largest weight times the largest
    value beside what the weights' own rounding takes."""
    kv, group, dim, page = 2, 4, 128, 32
    step = Step(5, [300, 21], [1, 1], page)
    cache = skn.PagedKVCache(ctx, step.n_pages, page, kv, dim, "q4_0")
    ref = oracle.Pages(step.n_pages, page, kv, dim, "q4_0")
    g = np.random.default_rng(2)
    total = int(step.lens.sum())
    k, v = (g.standard_normal((total, kv, dim)).astype(np.float32) for _ in range(2))
    v[:, :, :32] *= 2.0 ** 10
    v[:, :, 32:] *= 2.0 ** -10
    q = bf16(g.standard_normal((step.n, kv * group, dim)))
    cache.append(k, v, step.table, step.full, step.lens)
    ref.append(k, v, step.table, step.full, step.lens)
    want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, 0.125)
    out = run_attend(cache, step, q, io, scale=0.125)
    most = np.empty((step.n, kv * group, 1))               # each row's largest weight of a sum of one
    for s in range(step.n):
        for h in range(kv * group):
            z = ref.rows("k", s, int(step.lens[s]), step.table)[h // group] @ q[s, h].astype(np.float64) * 0.125
            most[s, h] = 1 / np.exp(z - z.max()).sum()
    miss = step.lens[:, None, None] * most * np.abs(ref.v).max() * 2.0 ** (-37 if io == "f32" else -32)
    tol = tolerance(want, mass, reach, 0.0 if io == "f32" else 2.0 ** -11, 0.0, io) + miss
    assert np.all(np.abs(out - want) <= tol)
    cache.close()


def _counters(cache):
    """device address and bytes of a cache's join counters: among the pointers of its structure, the only allocation of 64 bytes an SM"""
    cuda = ctypes.CDLL("libcuda.so.1")
    words = (ctypes.c_uint64 * 152).from_address(cache.handle.value)
    size = 64 * torch.cuda.get_device_properties(0).multi_processor_count
    for w in words:
        base, n = ctypes.c_uint64(), ctypes.c_size_t()
        if w and cuda.cuMemGetAddressRange_v2(ctypes.byref(base), ctypes.byref(n), ctypes.c_uint64(w)) == 0 and base.value == w and n.value == size:
            return cuda, w, size
    raise AssertionError("no counters")


@pytest.mark.parametrize("dtype", ["f16", "q4_0"])
def test_a_cache_is_whole_after_a_wait_that_ran_out(dtype):
    """A kernel that gives up leaves counters of its joins as they are (here: written by the host).  The report of a wait that ran out, of any kernel of the
    context, sets them back, so that the next step is right."""
    c0, c1 = skn.Context(0), skn.Context(0)
    c0.set_wait_limit_ms(50)
    ex = Exchange.connect_local([c0, c1], 4096)
    caches = []
    for lens, news, io in (([5000, 40], [50, 1], "bf16"), ([5000, 3], [1, 1], "f32")):
        step = Step(5, lens, news, 32)
        cache, _ = filled(c0, step, 2, 128, dtype, 5)
        q = bf16(np.random.default_rng(1).standard_normal((step.n, 8, 128)))
        caches.append((cache, step, q, io, run_attend(cache, step, q, io)))
    for cache, *_ in caches:
        cuda, at, size = _counters(cache)
        back = (ctypes.c_uint32 * (size // 4))()
        torch.cuda.synchronize()
        assert cuda.cuMemcpyDtoH_v2(back, ctypes.c_uint64(at), ctypes.c_size_t(size)) == 0 and not any(back)
        assert cuda.cuMemsetD32_v2(ctypes.c_uint64(at), ctypes.c_uint32(2 ** 31), ctypes.c_size_t(size // 4)) == 0
    part, out = torch.ones(1024, device="cuda"), torch.zeros(1024, device="cuda")
    torch.cuda.synchronize()
    ex[0].all_reduce(part, None, out, 1024)                 # of two ranks the other one never joins
    with pytest.raises(skn.SknError, match="bounded wait"):
        c0.sync()
    for cache, step, q, io, want in caches:
        for _ in range(3):
            assert np.array_equal(run_attend(cache, step, q, io), want)
        cache.close()
    for e in ex:
        e.close()
    c0.close()
    c1.close()


def test_segments_that_take_seconds_to_compute_again(ctx):
    """An infinity that every row sees, in front of two million keys: the blocks' second computation takes seconds, longer than the other warps of their CTAs
    wait.  Rows against the formula in 64 bits by torch; exponentials and weights as for fp32 rows of long sums, outputs rounded to bf16."""
    kv, group, dim, page, n, new = 8, 64, 64, 128, 2_000_000, 76
    pages = -(-n // page)
    pools = [torch.randn(pages, kv, page, dim, device="cuda").to(torch.float16) for _ in range(2)]
    pools[1][0, :, 0, 3] = float("inf")
    cache = skn.PagedKVCache(ctx, pages, page, kv, dim, "f16", pools=pools)
    b = skn.PagedBatch(torch.arange(pages, dtype=torch.int32, device="cuda")[None], torch.tensor([0, new], dtype=torch.int32, device="cuda"),
                       torch.tensor([n], dtype=torch.int32, device="cuda"), new, new)
    q = (8 * torch.randn(new, kv * group, dim, device="cuda")).bfloat16()
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    cache.attend_dev(b, q, out, scale=0.125)
    ctx.sync()
    assert (out[..., 3] == float("inf")).all()
    for row, head in ((0, 0), (40, 200), (75, 511)):
        k, v = (p[:, head // group].reshape(-1, dim)[:n - new + row + 1].double() for p in pools)
        z = k @ q[row, head].double() * 0.125
        w = torch.softmax(z, 0)
        keep = torch.arange(dim) != 3
        want, mass = (w @ v)[keep], (w @ v.abs())[keep]
        reach = 0.125 * (k.abs() @ q[row, head].double().abs()).max()
        # sums of two million weights, 256 at a time: 7813 roundings of 2^-24 at worst
        tol = mass * (torch.expm1(2 * 2.0 ** -19 * reach) + 2.0 ** -18 + 7813 * 2.0 ** -24) + 2.0 ** -8 * want.abs()
        assert ((out[row, head].double()[keep] - want).abs() <= tol).all()
    cache.close()


def test_rows_written_over_others_are_refused(ctx):
    """queries that are turned into a place of which other rows are still read, rows that are gathered over one another; beside one another is right"""
    kv, H, dim = 2, 4, 64
    step = Step(3, [40, 30], [2, 3], 16)
    cache, _ = filled(ctx, step, kv, dim, "bf16", 3, rot=64)
    b, n = step.batch(), step.n
    wide = torch.randn(n + 1, 2 * H + 2 * kv, dim, device="cuda").bfloat16()
    flat = wide.view(-1)
    q, k, v = wide[:n, :H], wide[:n, H:H + kv], wide[:n, H + kv:H + 2 * kv]
    over_q = [wide[1:, :H], wide[:n, 1:H + 1][:, :H], flat[:n * H * dim].view(n, H, dim)]
    for out in over_q:
        with pytest.raises(skn.SknError, match="over q"):
            cache.append_dev(b, k.clone(), v.clone(), q, out)
    for out in (wide[:n, H:2 * H], wide[:n, H + kv:2 * H + kv], wide[:n, H + 1:2 * H + 1], flat[n * dim:n * dim + n * H * dim].view(n, H, dim)):
        with pytest.raises(skn.SknError, match="over k or v"):
            cache.append_dev(b, k, v, q.clone(), out)
    dense = torch.zeros(2 * n * kv * dim, device="cuda")
    at = [dense[i * dim:i * dim + n * kv * dim].view(n, kv, dim) for i in (0, 1, n * kv - 1, n * kv)]
    for i, j in ((0, 0), (0, 1), (0, 2), (2, 0), (1, 3)):
        with pytest.raises(skn.SknError, match="over v_out"):
            cache.gather_dev(b, at[i], at[j])
    torch.cuda.synchronize()
    own = torch.zeros(n, H, dim, device="cuda").bfloat16()
    beside = wide[:n, H + 2 * kv:]
    was = wide.clone()
    torch.cuda.synchronize()
    cache.append_dev(b, k, v, q, own)
    cache.append_dev(b, k, v, q, beside)
    cache.gather_dev(b, at[0], at[3])
    cache.append_dev(b, k, v, q, q)
    ctx.sync()
    assert torch.equal(own, beside) and torch.equal(own, q) and torch.equal(wide[:n, H:H + 2 * kv], was[:n, H:H + 2 * kv]) and torch.equal(wide[n], was[n])
    assert torch.equal(at[3], v.float())
    one = Step(3, [40], [1], 16)                           # one row: no other one that its stride could meet
    b1 = one.batch()
    q1 = wide[:1, :H].clone()
    torch.cuda.synchronize()
    cache.append_dev(b1, k[:1], v[:1], wide[:1, :H], wide[:1, :H])
    cache.append_dev(b1, k[:1], v[:1], q1, q1.view(-1).as_strided((1, H, dim), (2 * H * dim, dim, 1)))
    ctx.sync()
    cache.close()


@pytest.mark.parametrize("dtype,io", [("f16", "f32"), ("bf16", "bf16"), ("q4_0", "bf16")])
@pytest.mark.parametrize("news", [[1, 1, 0], [20, 1, 3]])
def test_a_bound_of_new_tokens_that_says_nothing(ctx, dtype, io, news):
    """max_new is an upper bound: the largest number is taken as the step's rows, by the choice of the kernel and by its grid"""
    kv, group, dim = 2, 8, 64
    step = Step(3, [400, 90, 30], news, 16, padding=2)
    cache, ref = filled(ctx, step, kv, dim, dtype, 3)
    g = np.random.default_rng(3)
    k, v = (g.standard_normal((step.n, kv, dim)).astype(np.float32) for _ in range(2))
    q = bf16(g.standard_normal((step.n, kv * group, dim)))
    t = [torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda() for a in (step.table, step.starts, step.lens)]
    kd, vd, qd = (torch.from_numpy(a).cuda().to(IO[io]) for a in (k, v, q))
    out = torch.zeros_like(qd)
    b = skn.PagedBatch(*t, step.n, 2 ** 31 - 1)
    kr, vr = kd.float().cpu().numpy(), vd.float().cpu().numpy()
    ref.append(kr, vr, step.table, step.starts, step.lens)
    want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, 0.125)
    torch.cuda.synchronize()
    cache.append_dev(b, kd, vd)
    cache.attend_dev(b, qd, out)
    ctx.sync()
    n = int(step.starts[-1])
    check(out.float().cpu().numpy()[:n], want[:n], mass[:n], reach[:n], io, dtype, True)
    assert not out[n:].any()
    cache.close()


@pytest.mark.parametrize("dtype", ["q4_0", "bf16"])
@pytest.mark.parametrize("heads", [63, 64, 256])
def test_many_kv_heads(ctx, dtype, heads):
    dim, page = 128, 16
    step = Step(3, [33, 5, 20], [3, 5, 1], page)
    cache, ref = filled(ctx, step, heads, dim, dtype, 3, rot=64, pairs="halves")
    g = np.random.default_rng(heads)
    k, v = (g.standard_normal((step.n, heads, dim)).astype(np.float32) for _ in range(2))
    q = g.standard_normal((step.n, heads, dim)).astype(np.float32)
    cache.append(k, v, step.table, step.starts, step.lens)
    ref.append(k, v, step.table, step.starts, step.lens)
    kk, vv = cache.gather(step.table, step.full, step.lens)
    for s in range(3):
        a, b = step.full[s], step.full[s + 1]
        assert np.array_equal(kk[a:b].transpose(1, 0, 2), ref.rows("k", s, b - a, step.table))
        assert np.array_equal(vv[a:b].transpose(1, 0, 2), ref.rows("v", s, b - a, step.table))
    want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, 0.1)
    check(run_attend(cache, step, q, "f32", scale=0.1), want, mass, reach, "f32", dtype, False)
    cache.close()


def test_caches_of_many_and_of_few_heads_at_once():
    """two threads, each with a context of its own, append to 4-bit caches of 256 and of 64 heads: neither takes shared memory away from the other's launches"""
    def work(heads, out):
        try:
            with skn.Context(0) as c:
                cache = skn.PagedKVCache(c, 2, 16, heads, 128, "q4_0")
                k = np.random.default_rng(heads).standard_normal((1, heads, 128)).astype(np.float32)
                for _ in range(2000):
                    cache.append(k, k, [[0]], [0, 1], [1])
                cache.close()
        except Exception as e:                              # told by the main thread
            out.append(e)

    failed = []
    threads = [threading.Thread(target=work, args=(h, failed)) for h in (256, 64)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_sequences_out_of_order_are_reported(ctx):
    """row ranges that go back are reported by every call of the step, whether or not one of its rows is looked for among them"""
    step = Step(3, [40, 9, 20, 20, 30], [5, 0, 0, 0, 3], 16)
    cache, _ = filled(ctx, step, 2, 64, "f16", 3)
    b = step.batch(starts=np.array([0, 5, 3, 3, 3, 8], dtype=np.int32), n=8)          # the second sequence: rows 5 to 3
    k, q = torch.zeros(8, 2, 64, device="cuda"), torch.zeros(8, 4, 64, device="cuda")
    out, kk, vv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(k)
    torch.cuda.synchronize()
    for call in (lambda: cache.append_dev(b, k, k), lambda: cache.gather_dev(b, kk, vv), lambda: cache.attend_dev(b, q, out)):
        call()
        with pytest.raises(skn.SknError, match="out of range"):
            ctx.sync()
        ctx.sync()
    cache.close()


def test_pools_over_one_another_are_refused(ctx):
    n = skn.PagedKVCache.pool_bytes(4, 16, 2, 64, "f16")
    memory = torch.zeros(2 * n, dtype=torch.uint8, device="cuda")
    for a, b in ((0, 0), (0, n - 16), (n, 16)):
        with pytest.raises(skn.SknError, match="over the other"):
            skn.PagedKVCache(ctx, 4, 16, 2, 64, "f16", pools=(memory[a:a + n], memory[b:b + n]))
    for a, b in ((0, n), (n, 0)):
        skn.PagedKVCache(ctx, 4, 16, 2, 64, "f16", pools=(memory[a:a + n], memory[b:b + n])).close()


@pytest.mark.parametrize("dim,group", [(64, 1), (128, 8), (64, 16), (128, 32)])
def test_weights_of_single_tokens_over_bf16(ctx, dim, group):
    """values that nearly cancel: an output's own rounding is small beside that of weights in bf16.  Two terms leave 2^-8 of 2^-8 of a weight."""
    kv = 2
    step = Step(5, [2, 5, 33, 300], [1, 1, 1, 1], 16)
    cache = skn.PagedKVCache(ctx, step.n_pages, 16, kv, dim, "bf16")
    ref = oracle.Pages(step.n_pages, 16, kv, dim, "bf16")
    g = np.random.default_rng(dim)
    total = int(step.lens.sum())
    k, v = (g.standard_normal((total, kv, dim)).astype(np.float32) for _ in range(2))
    at = np.concatenate([np.arange(int(x)) for x in step.lens])
    v = (np.where(at % 2, -8, 8)[:, None, None] + v).astype(np.float32)
    q = bf16(0.2 * g.standard_normal((step.n, kv * group, dim)))
    cache.append(k, v, step.table, step.full, step.lens)
    ref.append(k, v, step.table, step.full, step.lens)
    want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, 0.125)
    err = np.abs(run_attend(cache, step, q, "bf16", scale=0.125) - want)
    assert np.all(err <= tolerance(want, mass, reach, 2.0 ** -16, 0.0, "bf16"))
    cache.close()


def test_a_timeout_behind_another_report_sets_a_cache_back(ctx):
    """the status word holds the last of several reports: here rows out of range, after counters were left above zero"""
    step = Step(5, [5000, 40], [50, 1], 32)
    cache, _ = filled(ctx, step, 2, 128, "bf16", 5)
    q = bf16(np.random.default_rng(1).standard_normal((step.n, 8, 128)))
    want = run_attend(cache, step, q, "bf16")
    cuda, at, size = _counters(cache)
    torch.cuda.synchronize()
    assert cuda.cuMemsetD32_v2(ctypes.c_uint64(at), ctypes.c_uint32(2 ** 31), ctypes.c_size_t(size // 4)) == 0
    k = torch.zeros(step.n, 2, 128, device="cuda")
    torch.cuda.synchronize()
    cache.gather_dev(step.batch(lens=[9000, 40]), k, torch.zeros_like(k))
    with pytest.raises(skn.SknError, match="out of range"):
        ctx.sync()
    for _ in range(2):
        assert np.array_equal(run_attend(cache, step, q, "bf16"), want)
    cache.close()


@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
def test_queries_are_turned_in_64_bits(ctx, pairs):
    """one rounding to fp32, near and far positions; the angle of a position has 2^-50 of it"""
    dim, kv, H = 128, 1, 5
    step = Step(3, [5, 200, 70001], [5, 9, 20], 128)
    cache = skn.PagedKVCache(ctx, step.n_pages, 128, kv, dim, "bf16", rot_dims=96, rot_pairs=pairs)
    g = np.random.default_rng(5)
    q = (g.standard_normal((step.n, H, dim)) * np.exp2(g.integers(-9, 9, (step.n, H, dim)))).astype(np.float32)
    k = g.standard_normal((step.n, kv, dim)).astype(np.float32)
    got = cache.append(k, k, step.table, step.starts, step.lens, q)
    want = oracle.rotate(q, [p for _, p in oracle.positions(step.starts, step.lens)], 96, 10000.0, pairs)
    assert np.all(np.abs(got - want) <= 2.0 ** -24 * np.abs(want) + 70001 * 2.0 ** -50 * np.abs(q).max(axis=2, keepdims=True))
    cache.close()
