"""Paged KV cache on the GPU against the oracle in 64 bits.

Cached rows are compared bit for bit: keys are rotated in 64 bits and rounded as the type says.  Rotated queries: cosine and sine rounded to
fp32 and two rounded operations, 3 x 2^-24 (|x| + |y|), bf16 rows a rounding of 2^-8 more.  Attention, with mass = sum p |v| and
reach = scale max sum |q k|: fp32 accumulation of at most 16 products of two or three terms is off by 16 x 2^-23 reach at worst, which
moves a weight by twice that; exponentials, weights in 22 bits or more and sums take 2^-18 mass.  A weight far below its row's largest has no
relative accuracy: two fp16 terms (fp32 rows) of weights lifted by 2^14 end at 2^-24, 2^-38 of the largest, one term (bf16 rows) lifted by
2^7 or more at 2^-31, so an output may miss 2^-38 or 2^-30 of each value (a dimension whose heavy keys hold exact zeros shows it).  bf16 rows: weights rounded by 2^-8 (bf16
caches) or 2^-11, outputs by 2^-8; caches of 4 bits enter products of many rows rounded to fp16, 2^-11 of reach and mass each."""
import numpy as np
import pytest
import torch

import skainet_b200 as skn
from conftest import FP32_TOL
from oracle import paged as oracle

pytestmark = pytest.mark.gpu
IO = {"f32": torch.float32, "bf16": torch.bfloat16}


def bf16(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).bfloat16().float().numpy()


class Step:
    """Sequences of the given lengths and new tokens over scattered pages"""

    def __init__(self, seed, lens, news, page, spare=2, padding=0, first=0):
        g = np.random.default_rng(seed)
        self.lens, self.page = np.asarray(lens, dtype=np.int32), page
        per = [-(-int(n) // page) for n in lens]
        self.n_pages = sum(per) + spare
        order = g.permutation(self.n_pages)
        self.table = np.full((len(lens), max(per + [1])), -1, dtype=np.int32)
        at = 0
        for s, n in enumerate(per):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.starts = np.concatenate([[first], first + np.cumsum(news)]).astype(np.int32)
        self.n = int(self.starts[-1]) + padding
        self.full = np.concatenate([[0], np.cumsum(self.lens)]).astype(np.int32)       # every token of every sequence

    def batch(self, starts=None, lens=None, n=None, table=None):
        starts = self.starts if starts is None else starts
        lens = self.lens if lens is None else lens
        table = self.table if table is None else table
        return skn.PagedBatch(*(torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda() for a in (table, starts, lens)),
                              self.n if n is None else n, max(1, int(np.diff(starts).max(initial=1))))


def filled(ctx, step, heads, dim, dtype, seed, rot=0, pairs="adjacent"):
    """(cache, oracle pages) holding every sequence's tokens but for the step's own"""
    g = np.random.default_rng(seed)
    new = np.diff(step.starts)
    lens = np.maximum(step.lens - new, 0)
    starts = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    k, v = (g.standard_normal((int(starts[-1]), heads, dim)).astype(np.float32) for _ in range(2))
    cache = skn.PagedKVCache(ctx, step.n_pages, step.page, heads, dim, dtype, rot_dims=rot, rot_pairs=pairs)
    ref = oracle.Pages(step.n_pages, step.page, heads, dim, dtype, rot, 10000.0, pairs)
    cache.append(k, v, step.table, starts, lens)
    ref.append(k, v, step.table, starts, lens)
    return cache, ref


def check(out, ref, mass, reach, io, dtype, many):
    w = 0.0 if io == "f32" else 2.0 ** -8 if dtype == "bf16" else 2.0 ** -11
    k4 = 2.0 ** -11 if many and io == "bf16" and dtype == "q4_0" else 0.0
    tol = tolerance(ref, mass, reach, w, k4, io)
    err = np.abs(np.asarray(out, dtype=np.float64) - ref)
    assert np.all(err <= tol), f"largest excess {np.max(err / tol):.3g} at {np.unravel_index(np.argmax(err / tol), err.shape)}"
    if io == "f32" and np.linalg.norm(ref) > 0:
        assert np.linalg.norm(err) <= FP32_TOL * np.linalg.norm(ref)


def tolerance(ref, mass, reach, w, k4, io):
    reach, total = reach[..., :1], reach[..., 1:]
    return (mass * (np.expm1(2 * (2.0 ** -19 + k4) * reach) + w + k4 + 2.0 ** -18) * 1.01 + total * (2.0 ** -38 if io == "f32" else 2.0 ** -30)
            + (2.0 ** -8 * np.abs(ref) if io == "bf16" else 0) + 1e-30)


def run_attend(cache, step, q, io, given=None, **kw):
    """through the host form (fp32) or on the device"""
    if io == "f32" and given is None:
        return cache.attend(q, step.table, step.starts, step.lens, **kw)
    qd = torch.from_numpy(q).cuda().to(IO[io])
    out = torch.zeros_like(qd) if given is None else torch.from_numpy(given).cuda().to(IO[io])
    torch.cuda.synchronize()
    cache.attend_dev(step.batch(), qd, out, **kw)
    cache.ctx.sync()
    return out.float().cpu().numpy()


SHAPES = [([1], [1]), ([17], [17]), ([5, 64, 33], [1, 1, 1]), ([130, 1, 47], [3, 1, 20])]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "q4_0"])
@pytest.mark.parametrize("dim,page,heads,rot,pairs", [(64, 16, 1, 64, "adjacent"), (128, 16, 2, 128, "halves"), (128, 64, 3, 48, "halves"), (64, 32, 2, 0, "adjacent"),
                                                      (128, 128, 8, 64, "adjacent"), (64, 16, 5, 16, "halves")])
@pytest.mark.parametrize("lens,news", SHAPES)
def test_append_and_gather(ctx, dtype, dim, page, heads, rot, pairs, lens, news):
    step = Step(7, lens, news, page)
    g = np.random.default_rng(sum(lens) + dim + heads)
    k, v, q = (g.standard_normal((step.n, h, dim)).astype(np.float32) * 3 for h in (heads, heads, 2 * heads))
    cache, ref = filled(ctx, step, heads, dim, dtype, 11, rot, pairs)
    got_q = cache.append(k, v, step.table, step.starts, step.lens, q)
    want_q = ref.append(k, v, step.table, step.starts, step.lens, q)
    tol = 3 * 2.0 ** -24 * (2 * np.abs(q).max(axis=2, keepdims=True)) + np.zeros_like(want_q)
    tol[:, :, rot:] = 0
    assert np.all(np.abs(got_q - want_q) <= tol)
    kk, vv = cache.gather(step.table, step.full, step.lens)
    cache.close()
    for s in range(len(lens)):
        a, b = step.full[s], step.full[s + 1]
        assert np.array_equal(kk[a:b].transpose(1, 0, 2), ref.rows("k", s, b - a, step.table))
        assert np.array_equal(vv[a:b].transpose(1, 0, 2), ref.rows("v", s, b - a, step.table))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "q4_0"])
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
def test_append_of_joint_bf16_rows(ctx, dtype, pairs):
    """q, k and v are parts of one projection's rows, padded rows before and behind the sequences; q is rotated in place; far positions"""
    lens, news, D, kv, H, page = [70000, 40], [3, 9], 128, 2, 6, 32
    step = Step(3, lens, news, page, padding=4, first=2)
    g = torch.Generator().manual_seed(5)
    joint = torch.randn(step.n, H + 2 * kv, D, generator=g).bfloat16()
    q, k, v = (joint[:, a:b].float().numpy() for a, b in ((0, H), (H, H + kv), (H + kv, H + 2 * kv)))
    ref = oracle.Pages(step.n_pages, page, kv, D, dtype, 64, 10000.0, pairs)
    want = ref.append(k, v, step.table, step.starts, step.lens, q)
    dev = joint.cuda()
    cache = skn.PagedKVCache(ctx, step.n_pages, page, kv, D, dtype, rot_dims=64, rot_pairs=pairs)
    torch.cuda.synchronize()
    qd = dev[:, :H]
    b = step.batch()
    cache.append_dev(b, dev[:, H:H + kv], dev[:, H + kv:], qd, qd)
    kk, vv = (torch.full((step.n, kv, D), 7.0, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    cache.gather_dev(b, kk, vv)
    ctx.sync()
    got = dev[:, :H].float().cpu().numpy()
    assert np.all(np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 4 * 2.0 ** -24 * 2 * np.abs(q).max())
    assert np.array_equal(dev[:, H:].cpu().view(torch.int16), joint[:, H:].view(torch.int16))
    for r in (0, 1, step.n - 1, step.n - 4):
        assert np.array_equal(got[r], q[r]) and (kk[r] == 7).all() and (vv[r] == 7).all()
    for i, (s, p) in enumerate(oracle.positions(step.starts, step.lens)):
        i += 2
        assert np.array_equal(kk[i].cpu().numpy(), ref.k[step.table[s, p // page], :, p % page])
        assert np.array_equal(vv[i].cpu().numpy(), ref.v[step.table[s, p // page], :, p % page])
    cache.close()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "q4_0"])
def test_append_writes_its_rows_only(ctx, dtype):
    step, kv, D = Step(2, [21, 50, 3], [2, 1, 5], 16, spare=3), 3, 64     # the last sequence has two padded rows
    n = skn.PagedKVCache.pool_bytes(step.n_pages, 16, kv, D, dtype)
    pools = [torch.randint(0, 255, (n,), dtype=torch.uint8, device="cuda") for _ in range(2)]
    before = [p.clone() for p in pools]
    cache = skn.PagedKVCache(ctx, step.n_pages, 16, kv, D, dtype, pools=pools)
    k = np.random.default_rng(1).standard_normal((step.n, kv, D)).astype(np.float32)
    cache.append(k, -k, step.table, step.starts, step.lens)
    row = {"q4_0": D // 2 + D // 16}.get(dtype, 2 * D)
    touched = torch.zeros(step.n_pages, kv, 16, dtype=torch.bool)
    for s, p in oracle.positions(step.starts, step.lens):
        if p >= 0:
            touched[step.table[s, p // 16], :, p % 16] = True
    for a, b in zip(pools, before):
        differ = (a != b).cpu().reshape(step.n_pages, kv, 16 * row)
        if dtype == "q4_0":
            quants = differ[..., :16 * D // 2].unflatten(-1, (D // 32, 16, 16)).any(-1).any(2)
            rows = quants | differ[..., 16 * D // 2:].unflatten(-1, (16, -1)).any(-1)
        else:
            rows = differ.unflatten(-1, (16, row)).any(-1)
        assert not (rows & ~touched).any()
        assert (rows | ~touched).all()
    cache.close()


ATTEND = [  # lens, news, kv heads, group, dim, page
    ([1], [1], 1, 1, 64, 16), ([2, 1, 16, 17], [1, 1, 1, 1], 2, 4, 128, 16), ([300, 31, 32, 33, 1025], [1, 1, 1, 1, 1], 2, 1, 64, 32),
    ([900, 77], [1, 1], 3, 5, 128, 64), ([515], [4], 2, 3, 128, 128), ([64, 200], [2, 5], 1, 8, 64, 16), ([40, 97], [40, 30], 2, 4, 128, 16),
    ([260, 3, 150], [129, 3, 1], 1, 7, 64, 32), ([600], [300], 1, 2, 128, 64), ([128, 129], [128, 129], 1, 16, 64, 128), ([70], [1], 1, 64, 128, 16),
    ([100, 0, 50, 9], [1, 0, 0, 1], 2, 2, 64, 16), ([33, 5], [12, 9], 2, 2, 128, 16)]


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "q4_0"])
@pytest.mark.parametrize("lens,news,kv,group,dim,page", ATTEND)
def test_attend(ctx, io, dtype, lens, news, kv, group, dim, page):
    step = Step(len(lens) + dim, lens, news, page)
    cache, ref = filled(ctx, step, kv, dim, dtype, 5)
    g = np.random.default_rng(dim + page)
    k, v = (g.standard_normal((step.n, kv, dim)).astype(np.float32) for _ in range(2))
    q = bf16(1.5 * g.standard_normal((step.n, kv * group, dim))) if io == "bf16" else (1.5 * g.standard_normal((step.n, kv * group, dim))).astype(np.float32)
    cache.append(k, v, step.table, step.starts, step.lens)
    ref.append(k, v, step.table, step.starts, step.lens)
    want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, dim ** -0.5)
    check(run_attend(cache, step, q, io), want, mass, reach, io, dtype, max(news) > 1)
    cache.close()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "q4_0"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (17, 33), (64, 16), (100, 5), (31, 1000), (5000, 3)])
@pytest.mark.parametrize("lens,news,page", [([400, 20, 1], [1, 1, 1], 16), ([333, 150], [150, 131], 32), ([300], [7], 64)])
def test_window_and_first_tokens(ctx, io, dtype, window, sinks, lens, news, page):
    """pages that no query sees are given back (their entries say -1)"""
    kv, group, dim = 2, 4, 64
    step = Step(window + sinks, lens, news, page)
    cache, ref = filled(ctx, step, kv, dim, dtype, 3)
    g = np.random.default_rng(window)
    k, v = (g.standard_normal((step.n, kv, dim)).astype(np.float32) for _ in range(2))
    q = bf16(2 * g.standard_normal((step.n, kv * group, dim)))
    cache.append(k, v, step.table, step.starts, step.lens)
    ref.append(k, v, step.table, step.starts, step.lens)
    want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, 0.2, window, sinks)
    for s in range(len(lens)):
        lo = max(0, lens[s] - news[s] - window + 1) // page
        step.table[s, -(-sinks // page):lo] = -1
    check(run_attend(cache, step, q, io, scale=0.2, window=window, sinks=sinks), want, mass, reach, io, dtype, max(news) > 1)
    cache.close()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "q4_0"])
@pytest.mark.parametrize("lens,news,window,sinks", [([700, 40], [1, 1], 0, 0), ([700], [1], 100, 4), ([300, 260], [150, 9], 0, 0), ([500], [200], 64, 2), ([90], [3], 16, 0)])
def test_nothing_hidden_reaches_an_output(ctx, io, dtype, lens, news, window, sinks):
    """Rows behind the length, later tokens' rows, rows outside the window and pages of nobody hold NaN and infinities: outputs are as accurate as
    without them (not the same bits: a step may be summed in another order then).  A NaN that is seen reaches the rows that see it and no other."""
    kv, group, dim, page = 2, 4, 128, 32
    step = Step(1, lens, news, page)
    n = skn.PagedKVCache.pool_bytes(step.n_pages, page, kv, dim, dtype)
    pools = [torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2)]
    cache = skn.PagedKVCache(ctx, step.n_pages, page, kv, dim, dtype, pools=pools)
    g = np.random.default_rng(9)
    k, v = (g.standard_normal((int(step.lens.sum()), kv, dim)).astype(np.float32) for _ in range(2))
    q = bf16(g.standard_normal((step.n, kv * group, dim)))
    cache.append(k, v, step.table, step.full, step.lens)
    ref = oracle.Pages(step.n_pages, page, kv, dim, dtype)
    ref.append(k, v, step.table, step.full, step.lens)
    want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, dim ** -0.5, window, sinks)
    check(run_attend(cache, step, q, io, window=window, sinks=sinks), want, mass, reach, io, dtype, max(news) > 1)

    def rows(pool):                       # [pages, heads, page, bytes of a row that make it NaN or infinite]
        p = pool.reshape(step.n_pages, kv, -1)
        return p[..., page * dim // 2:].unflatten(-1, (page, -1)) if dtype == "q4_0" else p.unflatten(-1, (page, -1))

    seen = torch.zeros(step.n_pages, page, dtype=torch.bool)
    for s, p in oracle.positions(step.starts, step.lens):
        t = np.arange(p + 1)
        t = t[(t > p - window) | (t < sinks)] if window else t
        seen[step.table[s, t // page], t % page] = True
    where = (~seen).cuda()
    bad = torch.tensor({"f16": [0x00, 0x7C, 0xFF, 0xFF, 0x00, 0xFC], "bf16": [0x80, 0x7F, 0xFF, 0xFF, 0x80, 0xFF], "q4_0": [0xFF, 0xFF, 0x00, 0x7C, 0x00, 0xFC]}[dtype],
                       dtype=torch.uint8, device="cuda")
    for pool in pools:
        r = rows(pool).transpose(1, 2)
        fill = bad.repeat(r.shape[-1] // 6 + 1)[:r.shape[-1]]
        r[where] = fill
    torch.cuda.synchronize()
    check(run_attend(cache, step, q, io, window=window, sinks=sinks), want, mass, reach, io, dtype, max(news) > 1)
    # rows that later queries of the same sequence see, and earlier ones do not
    s = 0
    last = int(step.lens[s]) - 1
    for pool in pools:
        rows(pool)[int(step.table[s, last // page]), :, last % page] = bad[2] if dtype != "q4_0" else bad[0]
    torch.cuda.synchronize()
    out = run_attend(cache, step, q, io, window=window, sinks=sinks)
    sees = int(step.starts[s + 1]) - 1
    assert np.isnan(out[sees]).all()
    keep = np.arange(step.n) != sees
    check(out[keep], want[keep], mass[keep], reach[keep], io, dtype, max(news) > 1)
    cache.close()


def test_infinities_in_part_of_a_tile(ctx):
    """an infinite value among later tokens of the same tile, in one dimension only"""
    kv, group, dim, page = 1, 2, 64, 16
    for dtype in ("f16", "bf16"):
        step = Step(4, [64], [48], page)
        cache, ref = filled(ctx, step, kv, dim, dtype, 5)
        g = np.random.default_rng(9)
        k, v = (g.standard_normal((step.n, kv, dim)).astype(np.float32) for _ in range(2))
        q = bf16(g.standard_normal((step.n, kv * group, dim)))
        v[30, 0, 5] = np.inf
        cache.append(k, v, step.table, step.starts, step.lens)
        for io in ("f32", "bf16"):
            out = run_attend(cache, step, q, io)
            assert np.isfinite(out[:30]).all()
            assert (out[30:, :, 5] == np.inf).all()
            rest = np.delete(out, 5, axis=2)
            assert np.isfinite(rest).all()
        cache.close()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "q4_0"])
def test_large_and_small_values(ctx, io, dtype):
    """scores of hundreds, queries and values of very different sizes, a value scale that grows along the sequence"""
    kv, group, dim, page = 2, 4, 128, 16
    for lens, news in (([300, 21], [1, 1]), ([300], [140])):
        step = Step(8, lens, news, page)
        cache = skn.PagedKVCache(ctx, step.n_pages, page, kv, dim, dtype)
        ref = oracle.Pages(step.n_pages, page, kv, dim, dtype)
        g = np.random.default_rng(4)
        total = int(step.lens.sum())
        grow = np.exp2(np.linspace(-11, 9, total)).astype(np.float32)[:, None, None]
        k, v = g.standard_normal((total, kv, dim)).astype(np.float32) * 4, g.standard_normal((total, kv, dim)).astype(np.float32) * grow
        q = bf16(g.standard_normal((step.n, kv * group, dim)) * np.exp2(g.integers(-20, 6, (step.n, kv * group, 1))))
        cache.append(k, v, step.table, step.full, step.lens)
        ref.append(k, v, step.table, step.full, step.lens)
        want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, 0.5)
        out = run_attend(cache, step, q, io, scale=0.5)
        k4 = 2.0 ** -11 if max(news) > 1 and io == "bf16" and dtype == "q4_0" else 0.0
        w = 0.0 if io == "f32" else 2.0 ** -8 if dtype == "bf16" else 2.0 ** -11
        tol = tolerance(want, mass, reach, w, k4, io)
        excess = np.abs(out - want) / tol
        assert excess.max() <= 1, f"{excess.max():.3g} at {np.unravel_index(excess.argmax(), excess.shape)}"
        cache.close()


@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_rows_of_nobody_stay(ctx, io):
    step = Step(6, [40, 2, 130], [4, 5, 70], 16, padding=3, first=2)          # the second sequence has three padded rows
    cache, ref = filled(ctx, step, 2, 64, "bf16", 3)
    g = np.random.default_rng(3)
    k, v = (g.standard_normal((step.n, 2, 64)).astype(np.float32) for _ in range(2))
    q = bf16(g.standard_normal((step.n, 8, 64)))
    cache.append(k, v, step.table, step.starts, step.lens)
    ref.append(k, v, step.table, step.starts, step.lens)
    given = bf16(g.standard_normal(q.shape))
    want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, 0.125, given=given)
    out = run_attend(cache, step, q, io, given=given)
    for r in (0, 1, step.n - 3, step.n - 1):
        assert np.array_equal(out[r], given[r])
    assert np.array_equal(out[6:9], np.zeros_like(out[6:9]))
    check(out[2:-3], want[2:-3], mass[2:-3], reach[2:-3], io, "bf16", True)
    cache.close()


@pytest.mark.parametrize("dtype,io", [("f16", "f32"), ("bf16", "bf16"), ("q4_0", "bf16"), ("q4_0", "f32")])
def test_serving_steps(ctx, dtype, io):
    """Prompts, then tokens, of sequences that share a first page and come and go; the decode step is a captured graph, replayed with tables
    and lengths rewritten in place"""
    kv, group, dim, page, D2 = 2, 4, 64, 16, 64
    g = np.random.default_rng(12)
    n_pages, cols = 40, 8
    cache = skn.PagedKVCache(ctx, n_pages, page, kv, dim, dtype, rot_dims=D2, rot_pairs="halves")
    ref = oracle.Pages(n_pages, page, kv, dim, dtype, D2, 10000.0, "halves")
    table = -np.ones((3, cols), dtype=np.int32)
    free = list(g.permutation(n_pages))
    shared = free.pop()
    lens = np.zeros(3, dtype=np.int32)

    def rows(n):
        return tuple(bf16(g.standard_normal((n, h, dim))) for h in (kv, kv, kv * group))

    def grow(s, n):
        lens[s] += n
        for c in range(-(-int(lens[s]) // page)):
            if table[s, c] < 0:
                table[s, c] = free.pop()

    def host(starts):
        k, v, q = rows(int(starts[-1]))
        got_q = cache.append(k, v, table, starts, lens, q)
        ref_q = ref.append(k, v, table, starts, lens, q)
        assert np.all(np.abs(got_q - ref_q) <= 6 * 2.0 ** -24 * np.abs(q).max())
        got_q = bf16(got_q)
        want, mass, reach = ref.attend(got_q, table, starts, lens, dim ** -0.5, 40, 3)
        st = Step.__new__(Step)
        st.table, st.starts, st.lens, st.n = table, starts, lens, int(starts[-1])
        check(run_attend(cache, st, got_q, io, window=40, sinks=3), want, mass, reach, io, dtype, True)

    table[0, 0] = shared
    grow(0, 16)
    host(np.array([0, 16, 16, 16], dtype=np.int32))
    table[1, 0] = table[2, 0] = shared                    # a common prefix of one page
    lens[1:] = 16
    grow(0, 21), grow(1, 5), grow(2, 33)
    host(np.array([0, 21, 26, 59], dtype=np.int32))

    # the decode step, captured on torch's capture stream
    dt, starts = torch.from_numpy(table).cuda(), torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    dl = torch.from_numpy(lens).cuda()
    b = skn.PagedBatch(dt, starts, dl, 3, 1)
    k, v = (torch.zeros(3, kv, dim, device="cuda", dtype=IO[io]) for _ in range(2))
    q, out = (torch.zeros(3, kv * group, dim, device="cuda", dtype=IO[io]) for _ in range(2))
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        cache.append_dev(b, k, v, q, q)
        cache.attend_dev(b, q, out, window=40, sinks=3)
    ctx.set_stream(None)
    for i in range(45):
        for s in range(3):
            grow(s, 1)
        if i == 20:                                       # one sequence ends; its pages come back, but for the shared one
            free.extend(int(p) for p in table[1, 1:] if p >= 0)
            table[1], lens[1] = -1, 0
            grow(1, 1)
        kn, vn, qn = rows(3)
        qr = ref.append(kn, vn, table, np.arange(4), lens, qn)
        for d, h in ((dt, table), (dl, lens), (k, kn), (v, vn), (q, qn)):
            d.copy_(torch.from_numpy(h))
        graph.replay()
        torch.cuda.synchronize()
        ctx.sync()
        got_q = q.float().cpu().numpy()
        assert np.all(np.abs(got_q - qr) <= (2.0 ** -8 * np.abs(qr) if io == "bf16" else 0) + 6 * 2.0 ** -24 * np.abs(qn).max())
        want, mass, reach = ref.attend(got_q, table, np.arange(4), lens, dim ** -0.5, 40, 3)
        check(out.float().cpu().numpy(), want, mass, reach, io, dtype, False)
    del graph
    cache.close()


def test_long_context_is_shared_out_and_joined(ctx):
    """one sequence of many tiles over all SMs, beside short ones; the same bits every time"""
    kv, group, dim, page = 2, 4, 128, 16
    for dtype, io in (("f16", "f32"), ("bf16", "bf16"), ("q4_0", "f32"), ("q4_0", "bf16")):
        step = Step(5, [20011, 3, 900], [1, 1, 1], page)
        cache, ref = filled(ctx, step, kv, dim, dtype, 5)
        g = np.random.default_rng(2)
        k, v = (g.standard_normal((3, kv, dim)).astype(np.float32) for _ in range(2))
        q = bf16(3 * g.standard_normal((3, kv * group, dim)))
        cache.append(k, v, step.table, step.starts, step.lens)
        ref.append(k, v, step.table, step.starts, step.lens)
        want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, dim ** -0.5)
        first = run_attend(cache, step, q, io)
        check(first, want, mass, reach, io, dtype, False)
        for _ in range(5):
            assert np.array_equal(run_attend(cache, step, q, io), first)
        cache.close()


@pytest.mark.parametrize("dtype", ["f16", "q4_0"])
def test_offsets_beyond_32_bits(ctx, dtype):
    kv, dim, page = 8, 128, 128
    n_pages = 20000 if dtype == "f16" else 64000          # 5.2 and 4.7 GB a pool
    cache = skn.PagedKVCache(ctx, n_pages, page, kv, dim, dtype)
    g = np.random.default_rng(2)
    table = np.array([[n_pages - 1, 0, n_pages // 2]], dtype=np.int32)
    lens, starts = np.array([300], dtype=np.int32), np.array([0, 300], dtype=np.int32)
    k, v = (g.standard_normal((300, kv, dim)).astype(np.float32) for _ in range(2))
    cache.append(k, v, table, starts, lens)
    kk, vv = cache.gather(table, starts, lens)
    assert np.array_equal(kk, oracle.held(k, dtype)) and np.array_equal(vv, oracle.held(v, dtype))
    small = oracle.Pages(3, page, kv, dim, dtype)
    t3 = np.array([[2, 0, 1]])
    small.append(k, v, t3, starts, lens)
    for io, news in (("f32", 1), ("bf16", 1), ("bf16", 40)):
        step = Step.__new__(Step)
        step.table, step.starts, step.lens, step.n = table, np.array([0, news], dtype=np.int32), lens, news
        q = bf16(g.standard_normal((news, 2 * kv, dim)))
        want, mass, reach = small.attend(q, t3, step.starts, lens, dim ** -0.5)
        check(run_attend(cache, step, q, io), want, mass, reach, io, dtype, news > 1)
    cache.close()


def test_host_refusals(ctx):
    cache = skn.PagedKVCache(ctx, 4, 16, 2, 64, "bf16")
    k = np.ones((20, 2, 64), dtype=np.float32)
    q = np.ones((20, 4, 64), dtype=np.float32)
    starts, lens = [0, 20], [20]
    cache.append(k, k, [[0, 1]], starts, lens)
    kept = cache.gather([[0, 1]], starts, lens)
    bad = [([[0, 4]], starts, lens), ([[0, -1]], starts, lens), ([[0]], starts, lens), ([[0, 1]], [0, 21], lens), ([[0, 1]], [5, 2], lens),
           ([[0, 1]], [-1, 20], lens), ([[0, 1]], starts, [-3])]
    for table, st, ln in bad:
        with pytest.raises((skn.SknError, ValueError)):
            cache.append(k, k, table, st, ln)
        with pytest.raises((skn.SknError, ValueError)):
            cache.attend(q, table, st, ln)
        with pytest.raises((skn.SknError, ValueError)):
            cache.gather(table, st, ln, 20)
    with pytest.raises(skn.SknError, match="written twice"):
        cache.append(k, k, [[0, 0]], starts, lens)
    with pytest.raises(skn.SknError, match="written twice"):
        cache.append(k, k, [[0, 1], [1, 0]], [0, 10, 20], [20, 10])
    for kw in ({"window": -1}, {"sinks": -1}, {"scale": float("nan")}):
        with pytest.raises(skn.SknError):
            cache.attend(q, [[0, 1]], starts, lens, **kw)
    with pytest.raises(ValueError):
        cache.attend(np.ones((20, 3, 64), dtype=np.float32), [[0, 1]], starts, lens)
    with pytest.raises(ValueError):
        cache.attend(np.ones((20, 130, 64), dtype=np.float32), [[0, 1]], starts, lens)
    with pytest.raises(ValueError):
        cache.append(k[:, :1], k[:, :1], [[0, 1]], starts, lens)
    for a, b in zip(kept, cache.gather([[0, 1]], starts, lens)):
        assert np.array_equal(a, b)
    # nothing to do
    assert cache.attend(q, np.zeros((0, 0), dtype=np.int32), [0], []).shape == q.shape
    assert not cache.attend(q, [[0, 1]], [3, 3], lens).any()
    cache.close()


def test_device_tables_out_of_range(ctx):
    """what only the kernels can see: a page that is none, rows beyond the step, lengths beyond the table; the rest of the step is right"""
    kv, dim, page = 2, 64, 16
    for dtype, io in (("bf16", "bf16"), ("f16", "f32"), ("q4_0", "f32")):
        for new in (1, 24):
            step = Step(3, [40, 60], [new, new], page)
            cache, ref = filled(ctx, step, kv, dim, dtype, 3)
            g = np.random.default_rng(1)
            k, v = (bf16(g.standard_normal((step.n, kv, dim))) for _ in range(2))
            q = bf16(g.standard_normal((step.n, 8, dim)))
            cache.append(k, v, step.table, step.starts, step.lens)
            ref.append(k, v, step.table, step.starts, step.lens)
            want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, 0.125)
            kd, vd, qd = (torch.from_numpy(a).cuda().to(IO[io]) for a in (k, v, q))
            faults = []
            for entry in (-1, step.n_pages, 2 ** 31 - 1, -2 ** 31):
                t = step.table.copy()
                t[0, 2] = entry
                faults.append(step.batch(table=t))
            faults += [step.batch(lens=[4000, 60]), step.batch(lens=[-1, 60])]
            for b in faults:
                out = torch.zeros_like(qd)
                torch.cuda.synchronize()
                cache.append_dev(b, kd, vd)
                cache.attend_dev(b, qd, out)
                with pytest.raises(skn.SknError, match="out of range"):
                    ctx.sync()
                ctx.sync()
                check(out.float().cpu().numpy()[new:], want[new:], mass[new:], reach[new:], io, dtype, new > 1)
            for starts in ([0, step.n + 9, step.n + 9], [-2, new, step.n]):
                b = skn.PagedBatch(*(torch.tensor(a, dtype=torch.int32, device="cuda") for a in (step.table.tolist(), starts, step.lens.tolist())), step.n, step.n + 9)
                out = torch.zeros_like(qd)
                torch.cuda.synchronize()
                cache.append_dev(b, kd, vd)
                cache.attend_dev(b, qd, out)
                with pytest.raises(skn.SknError, match="out of range"):
                    ctx.sync()
            cache.close()


def test_device_refusals(ctx):
    step = Step(3, [40], [2], 16)
    cache, _ = filled(ctx, step, 2, 64, "bf16", 3)
    b = step.batch()
    k = torch.zeros(2, 2, 64, device="cuda", dtype=torch.bfloat16)
    q = torch.zeros(2, 4, 64, device="cuda", dtype=torch.bfloat16)
    for bad in (q.float(), q.half(), q[:, :, :32], torch.zeros(2, 4, 72, device="cuda", dtype=torch.bfloat16)[:, :, 3:67], q.cpu(), q[:1]):
        with pytest.raises((ValueError, skn.SknError)):
            cache.attend_dev(b, bad, q)
        with pytest.raises((ValueError, skn.SknError)):
            cache.append_dev(b, k, k, q, bad)
    wide = torch.zeros(2 * 260 + 8, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(skn.SknError):                     # rows that start between 16-byte boundaries
        cache.attend_dev(b, wide.as_strided((2, 4, 64), (260, 64, 1)), q)
    with pytest.raises(skn.SknError):
        cache.attend_dev(b, wide.as_strided((2, 4, 64), (256, 64, 1), 4), q)
    with pytest.raises(ValueError):                       # overlapping rows
        cache.attend_dev(b, wide.as_strided((2, 4, 64), (128, 64, 1)), q)
    with pytest.raises(ValueError):
        skn.PagedBatch(torch.zeros(1, 3, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), 1, 1)
    with pytest.raises(ValueError):
        skn.PagedKVCache(ctx, 4, 16, 2, 64, "bf16", pools=[torch.zeros(100, device="cuda", dtype=torch.uint8)] * 2)
    cache.close()


def test_another_stream(ctx):
    step = Step(3, [300, 40], [1, 1], 16)
    cache, ref = filled(ctx, step, 2, 128, "f16", 3)
    g = np.random.default_rng(1)
    q = bf16(g.standard_normal((2, 8, 128)))
    k = bf16(g.standard_normal((2, 2, 128)))
    qr = ref.append(k, k, step.table, step.starts, step.lens, q)
    want, mass, reach = ref.attend(qr, step.table, step.starts, step.lens, 128 ** -0.5)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        ctx.set_stream(side.cuda_stream)
        b = step.batch()
        kd, qd = torch.from_numpy(k).cuda(), torch.from_numpy(q).cuda()
        out = torch.empty_like(qd)
        cache.append_dev(b, kd, kd, qd, qd)
        cache.attend_dev(b, qd, out)
        ctx.sync()
        ctx.set_stream(None)
    check(out.cpu().numpy(), want, mass, reach, "f32", "f16", False)
    cache.close()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "q4_0"])
@pytest.mark.parametrize("dim,heads,rot,pairs", [(64, 1, 32, "adjacent"), (128, 3, 128, "halves")])
def test_long_steps(ctx, dtype, dim, heads, rot, pairs):
    """steps of thousands of rows, of an odd number, over many short sequences (some without a row), padded on both sides"""
    page = 16
    g = np.random.default_rng(dim)
    news = g.integers(0, 30, 150)
    lens = np.where(news > 0, news + g.integers(0, 40, 150), 3)
    lens[5], news[5] = 4, 9                                # five padded rows
    step = Step(9, lens, news, page, padding=6, first=3)
    step.n += 1 - step.n % 2
    assert step.n >= 2048 and step.n % 4
    k, v, q = (g.standard_normal((step.n, h, dim)).astype(np.float32) for h in (heads, heads, 2 * heads))
    cache, ref = filled(ctx, step, heads, dim, dtype, 11, rot, pairs)
    got_q = cache.append(k, v, step.table, step.starts, step.lens, q)
    want_q = ref.append(k, v, step.table, step.starts, step.lens, q)
    tol = 3 * 2.0 ** -24 * (2 * np.abs(q).max(axis=2, keepdims=True)) + np.zeros_like(want_q)
    tol[:, :, rot:] = 0
    assert np.all(np.abs(got_q - want_q) <= tol)
    b, given = step.batch(), torch.full((step.n, heads, dim), 7.0, device="cuda")
    kk, vv = given.clone(), given.clone()
    torch.cuda.synchronize()
    cache.gather_dev(b, kk, vv)
    ctx.sync()
    cache.close()
    want = [np.full((step.n, heads, dim), 7.0) for _ in range(2)]
    for i, (s, p) in enumerate(oracle.positions(step.starts, step.lens)):
        if p >= 0:
            for w, pool in zip(want, (ref.k, ref.v)):
                w[3 + i] = pool[step.table[s, p // page], :, p % page]
    assert np.array_equal(kk.cpu().numpy(), want[0]) and np.array_equal(vv.cpu().numpy(), want[1])


@pytest.mark.parametrize("dtype,io", [("f16", "bf16"), ("bf16", "f32"), ("q4_0", "bf16"), ("q4_0", "f32")])
@pytest.mark.parametrize("n_seqs,most,group", [(600, 1, 4), (600, 5, 8), (70, 1, 64)])
def test_many_sequences(ctx, dtype, io, n_seqs, most, group):
    g = np.random.default_rng(n_seqs + most)
    lens = g.integers(most, 60, n_seqs)
    news = g.integers(0, most + 1, n_seqs) if most > 1 else np.ones(n_seqs, dtype=np.int64)
    step = Step(2, lens, news, 16)
    kv, dim = 2, 64
    cache, ref = filled(ctx, step, kv, dim, dtype, 3)
    k, v = (g.standard_normal((step.n, kv, dim)).astype(np.float32) for _ in range(2))
    q = bf16(g.standard_normal((step.n, kv * group, dim)))
    cache.append(k, v, step.table, step.starts, step.lens)
    ref.append(k, v, step.table, step.starts, step.lens)
    want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, 0.125)
    check(run_attend(cache, step, q, io), want, mass, reach, io, dtype, most * group > 32)
    cache.close()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "q4_0"])
@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_scales(ctx, io, dtype, scale):
    """the mean of what is seen; the smallest products weigh most"""
    kv, group, dim = 2, 4, 128
    for lens, news, window in (([150, 3], [1, 1], 0), ([150, 140], [50, 33], 0), ([200], [60], 40)):
        step = Step(2, lens, news, 32)
        cache, ref = filled(ctx, step, kv, dim, dtype, 3)
        g = np.random.default_rng(1)
        k, v = (g.standard_normal((step.n, kv, dim)).astype(np.float32) for _ in range(2))
        q = bf16(g.standard_normal((step.n, kv * group, dim)))
        cache.append(k, v, step.table, step.starts, step.lens)
        ref.append(k, v, step.table, step.starts, step.lens)
        want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, scale, window, 2)
        check(run_attend(cache, step, q, io, scale=scale, window=window, sinks=2), want, mass, reach, io, dtype, max(news) > 1)
        cache.close()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "q4_0"])
@pytest.mark.parametrize("lens,news", [([333, 20], [1, 1]), ([333, 200], [150, 9])])
def test_rows_within_wider_ones(ctx, io, dtype, lens, news):
    """queries are parts of a joint projection's rows; outputs rows at multiples of 16 bytes that are none of 32, the rest of which stays"""
    kv, group, dim = 2, 3, 64
    step = Step(2, lens, news, 32)
    cache, ref = filled(ctx, step, kv, dim, dtype, 3)
    g = np.random.default_rng(1)
    k, v = (g.standard_normal((step.n, kv, dim)).astype(np.float32) for _ in range(2))
    q = bf16(g.standard_normal((step.n, kv * group, dim)))
    cache.append(k, v, step.table, step.starts, step.lens)
    ref.append(k, v, step.table, step.starts, step.lens)
    want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, 0.125)
    H = kv * group
    joint = torch.full((step.n, H + 2 * kv, dim), 3.0, device="cuda", dtype=IO[io])
    joint[:, :H] = torch.from_numpy(q).to(IO[io])
    width = H * dim + 8
    flat = torch.full((step.n * width + 8,), 5.0, device="cuda", dtype=IO[io])
    out = flat.as_strided((step.n, H, dim), (width, dim, 1), 8)
    torch.cuda.synchronize()
    cache.attend_dev(step.batch(), joint[:, :H], out)
    ctx.sync()
    check(out.float().cpu().numpy(), want, mass, reach, io, dtype, max(news) > 1)
    assert (flat[8:].view(step.n, width)[:, H * dim:] == 5).all() and (flat[:8] == 5).all()
    cache.close()


def test_outputs_beside_their_queries_only(ctx):
    """outputs in the same rows as the queries are right where they lie beside them, and refused where they lie over them"""
    kv, group, dim = 2, 4, 64
    step = Step(2, [90, 40], [20, 1], 16)
    cache, ref = filled(ctx, step, kv, dim, "bf16", 3)
    H = kv * group
    wide = torch.randn(step.n + 1, 2 * H + 1, dim, device="cuda").bfloat16()
    q = wide[:step.n, 1:H + 1]
    want, mass, reach = ref.attend(q.float().cpu().numpy(), step.table, step.starts, step.lens, 0.125)
    b = step.batch()
    for out in (q, wide[:step.n, :H], wide[:step.n, 2:H + 2], wide[:step.n, H:2 * H], wide[1:, 1:H + 1], wide.view(-1)[:step.n * H * dim].view(step.n, H, dim)):
        with pytest.raises(skn.SknError, match="over q"):
            cache.attend_dev(b, q, out)
    torch.cuda.synchronize()
    cache.attend_dev(b, q, wide[:step.n, H + 1:])
    ctx.sync()
    check(wide[:step.n, H + 1:].float().cpu().numpy(), want, mass, reach, "bf16", "bf16", True)
    cache.close()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_infinity_in_a_long_context(ctx, dtype):
    """seen by every row of blocks with tens of thousands of keys, in one dimension"""
    kv, group, dim, page = 1, 8, 64, 64
    step = Step(4, [40000], [40], page)
    cache, ref = filled(ctx, step, kv, dim, dtype, 5)
    g = np.random.default_rng(9)
    k, v = (g.standard_normal((step.n, kv, dim)).astype(np.float32) for _ in range(2))
    q = bf16(g.standard_normal((step.n, kv * group, dim)))
    cache.append(k, v, step.table, step.starts, step.lens)
    ref.append(k, v, step.table, step.starts, step.lens)
    want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, 0.125)
    row = step.table[:1, :1], [0, 1], [1]
    was = cache.gather(*row)
    was[1][0, 0, 3] = np.inf
    cache.append(was[0], was[1], *row)
    for io in ("bf16", "f32"):
        out = run_attend(cache, step, q, io)
        assert (out[..., 3] == np.inf).all()
        keep = np.arange(dim) != 3
        check(out[..., keep], want[..., keep], mass[..., keep], reach[..., np.concatenate([[True], keep])], io, dtype, True)
    cache.close()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "q4_0"])
def test_captured_prompts(ctx, dtype):
    """a captured step of up to 24 new tokens a sequence, replayed with other lengths, row counts, tables and windows' beginnings"""
    kv, group, dim, page, rows = 2, 4, 64, 16, 60
    g = np.random.default_rng(3)
    n_pages, cols = 64, 12
    cache = skn.PagedKVCache(ctx, n_pages, page, kv, dim, dtype)
    ref = oracle.Pages(n_pages, page, kv, dim, dtype)
    dt, starts = torch.zeros(3, cols, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    dl = torch.zeros(3, dtype=torch.int32, device="cuda")
    b = skn.PagedBatch(dt, starts, dl, rows, 24)
    k, v = (torch.zeros(rows, kv, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    q, out = (torch.zeros(rows, kv * group, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        cache.append_dev(b, k, v)
        cache.attend_dev(b, q, out, window=50, sinks=2)
    ctx.set_stream(None)
    lens = np.zeros(3, dtype=np.int32)
    for i in range(12):
        news = np.array([g.integers(0, 25), 0 if i % 3 else 24, g.integers(1, 9)], dtype=np.int32)
        if i == 6:
            lens[:] = 0
        lens = (lens + news).astype(np.int32)
        assert lens.max() <= cols * page
        table = g.permutation(n_pages)[:3 * cols].reshape(3, cols).astype(np.int32) if i in (0, 6) else table
        at = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        kn, vn, qn = (bf16(g.standard_normal((rows, h, dim))) for h in (kv, kv, kv * group))
        given = bf16(g.standard_normal(qn.shape))
        for d, h in ((dt, table), (starts, at), (dl, lens), (k, kn), (v, vn), (q, qn), (out, given)):
            d.copy_(torch.from_numpy(h))
        graph.replay()
        torch.cuda.synchronize()
        ctx.sync()
        ref.append(kn, vn, table, at, lens)
        want, mass, reach = ref.attend(qn, table, at, lens, dim ** -0.5, 50, 2, given=given)
        got, n = out.float().cpu().numpy(), int(at[-1])
        assert np.array_equal(got[n:], given[n:])
        check(got[:n], want[:n], mass[:n], reach[:n], "bf16", dtype, True)
    del graph
    cache.close()


def test_two_contexts_at_once(ctx):
    """caches of two contexts work on streams of their own: each has its workspace"""
    other = skn.Context(0)
    jobs = []
    for i, c in enumerate((ctx, other)):
        for news in ([1, 1, 1], [20, 3, 40]):
            step = Step(5 + i, [5000 + 900 * i, 300, 2000], news, 32)
            cache, _ = filled(c, step, 2, 128, "bf16", 5 + i)
            q = torch.randn(step.n, 8, 128, device="cuda").bfloat16()
            out = torch.zeros_like(q)
            torch.cuda.synchronize()
            b = step.batch()
            cache.attend_dev(b, q, out)
            c.sync()
            jobs.append((cache, b, q, out, out.clone(), c))
    torch.cuda.synchronize()
    for _ in range(30):
        for cache, b, q, out, first, c in jobs:
            cache.attend_dev(b, q, out)
    ctx.sync()
    other.sync()
    for cache, b, q, out, first, c in jobs:
        assert torch.equal(out, first)
        cache.close()
    other.close()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "q4_0"])
@pytest.mark.parametrize("group,window", [(3, 0), (8, 60), (12, 0), (40, 0)])
def test_steps_of_prompts_and_single_tokens(ctx, io, dtype, group, window):
    """in one step: prompts, portions of prompts, single tokens, sequences without a row, padded ones"""
    kv, dim = 2, 64
    step = Step(2, [50, 700, 3, 9, 260, 120, 2, 30], [50, 1, 3, 0, 1, 12, 4, 2], 16, padding=2)
    cache, ref = filled(ctx, step, kv, dim, dtype, 3)
    g = np.random.default_rng(group)
    k, v = (g.standard_normal((step.n, kv, dim)).astype(np.float32) for _ in range(2))
    q = bf16(g.standard_normal((step.n, kv * group, dim)))
    cache.append(k, v, step.table, step.starts, step.lens)
    ref.append(k, v, step.table, step.starts, step.lens)
    given = bf16(g.standard_normal(q.shape))
    want, mass, reach = ref.attend(q, step.table, step.starts, step.lens, 0.125, window, 2, given=given)
    out = run_attend(cache, step, q, io, given=given, window=window, sinks=2)
    n = int(step.starts[-1])
    assert np.array_equal(out[n:], given[n:])
    check(out[:n], want[:n], mass[:n], reach[:n], io, dtype, True)
    cache.close()


def test_calls_without_their_parts(ctx):
    step = Step(3, [40], [2], 16)
    cache, _ = filled(ctx, step, 2, 64, "bf16", 3)
    k = torch.zeros(2, 2, 64, device="cuda", dtype=torch.bfloat16)
    q = torch.zeros(2, 4, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="q_out"):
        cache.append_dev(step.batch(), k, k, q)
    wide = skn.PagedBatch(torch.zeros(1, 2 ** 23 + 1, dtype=torch.int32, device="cuda"), torch.tensor([0, 2], dtype=torch.int32, device="cuda"),
                          torch.tensor([2], dtype=torch.int32, device="cuda"), 2, 2)
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="pages"):
        cache.attend_dev(wide, q, torch.zeros_like(q))
    cache.close()
