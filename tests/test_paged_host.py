"""Paged KV cache without a GPU: the oracle against second formulations, and what the library refuses before it touches a device."""
import ctypes

import numpy as np
import pytest

import skainet_b200 as skn
from oracle import paged as oracle
from skainet_b200 import _ffi


def test_q4_0_of_the_oracle_is_ggufs():
    gguf = pytest.importorskip("gguf")
    g = np.random.default_rng(1)
    x = g.standard_normal((64, 128)).astype(np.float32) * np.exp2(g.integers(-12, 9, (64, 1))).astype(np.float32)
    x[3] = 0
    x[4, :32] = np.where(np.arange(32) % 2, 1.5, -1.5)       # equals: the first one decides the sign of d
    q, d = oracle.quantize_q4_0(x)
    raw = gguf.quants.quantize(x, gguf.GGMLQuantizationType.Q4_0).reshape(-1, 18)
    assert np.array_equal(raw[:, :2].copy().view(np.float16).reshape(d.shape), d)
    qs = raw[:, 2:]
    assert np.array_equal(np.concatenate([qs & 15, qs >> 4], axis=1).reshape(q.shape), q)


def test_attention_of_the_oracle_against_a_dense_mask():
    g = np.random.default_rng(2)
    p = oracle.Pages(6, 16, 2, 64, "bf16", 32, 10000.0, "halves")
    table, starts, lens = np.array([[4, 2], [5, 1]]), np.array([0, 20, 29]), np.array([20, 30])
    k, v, q = (g.standard_normal((29, n, 64)).astype(np.float32) for n in (2, 2, 4))
    early = g.standard_normal((21, 2, 64)).astype(np.float32)
    p.append(early, early, table[1:], np.array([0, 21]), np.array([21]))
    qr = p.append(k, v, table, starts, lens, q)
    out, _, _ = p.attend(qr, table, starts, lens, 0.1, 7, 3)
    for s, (a, b) in enumerate(((0, 20), (20, 29))):
        n = int(lens[s])
        pos, key = np.arange(n - (b - a), n)[:, None], np.arange(n)
        mask = (key <= pos) & ((key > pos - 7) | (key < 3))
        for h in range(4):
            z = np.where(mask, qr[a:b, h] @ p.rows("k", s, n, table)[h // 2].T * 0.1, -np.inf)
            w = np.exp(z - z.max(axis=1, keepdims=True))
            ref = w @ p.rows("v", s, n, table)[h // 2] / w.sum(axis=1, keepdims=True)
            np.testing.assert_allclose(out[a:b, h], ref, rtol=1e-12, atol=1e-12)


def test_rotation_turns_by_the_difference_of_positions():
    g = np.random.default_rng(3)
    for pairs in ("adjacent", "halves"):
        q, k = g.standard_normal((2, 1, 64)), g.standard_normal((2, 1, 64))
        q[1], k[1] = q[0], k[0]
        a, b = oracle.rotate(q, [5, 1005], 64, 10000.0, pairs), oracle.rotate(k, [2, 1002], 64, 10000.0, pairs)
        assert abs((a[0] * b[0]).sum() - (a[1] * b[1]).sum()) < 1e-9


@pytest.mark.parametrize("over,message", [
    ({"dtype": 0}, "not element type 0"), ({"dtype": 2}, "not element type 2"), ({"dim": 96}, "head_dim"), ({"page": 24}, "a page holds"),
    ({"page": 256}, "a page holds"), ({"rot": 8}, "multiple of 16"), ({"rot": 144}, "multiple of 16"), ({"rot": -16}, "multiple of 16"),
    ({"pairs": 2}, "pairing"), ({"base": 0.0}, "rot_base"), ({"base": float("nan")}, "rot_base"), ({"pages": 0}, "positive"), ({"heads": 0}, "positive"),
    ({"heads": 257}, "positive")])
def test_specifications_are_refused(over, message):
    s = {"heads": 2, "dim": 64, "page": 16, "dtype": 1, "pages": 4, "rot": 64, "pairs": 0, "base": 10000.0} | over
    spec = _ffi.PagedSpec(s["heads"], s["dim"], s["page"], s["dtype"], s["pages"], s["rot"], s["pairs"], 0, s["base"])
    n = ctypes.c_int64()
    assert _ffi.lib().skn_paged_pool_bytes(ctypes.byref(spec), ctypes.byref(n)) != 0
    assert message in _ffi.lib().skn_last_error(None).decode()


@pytest.mark.parametrize("dtype,dim,page,heads,pages,bytes_", [
    ("f16", 64, 16, 1, 1, 2048), ("bf16", 128, 32, 8, 3, 8 * 3 * 32 * 256), ("q4_0", 128, 16, 2, 5, 2 * 5 * 16 * 72),
    ("q4_0", 64, 128, 1, 1, 128 * 36), ("f16", 128, 128, 8, 100000, 100000 * 8 * 128 * 256)])
def test_pool_bytes(dtype, dim, page, heads, pages, bytes_):
    assert skn.PagedKVCache.pool_bytes(pages, page, heads, dim, dtype) == bytes_


def test_bad_handles_are_refused():
    L, out, b = _ffi.lib(), ctypes.c_void_p(), _ffi.PagedBatchSpec()
    spec = _ffi.PagedSpec(1, 64, 16, 1, 1, 0, 0, 0, 1.0)
    assert L.skn_paged_create(None, ctypes.byref(spec), None, None, ctypes.byref(out)) == 7
    assert L.skn_paged_destroy(None) == 7
    assert L.skn_paged_info(None, None, None, None) == 7
    assert L.skn_paged_append(None, ctypes.byref(b), None, None, None, 0, None) == 7
    assert L.skn_paged_append_dev(None, ctypes.byref(b), 0, None, 0, None, 0, None, 0, 0, None, 0) == 7
    assert L.skn_paged_gather(None, ctypes.byref(b), None, None) == 7
    assert L.skn_paged_gather_dev(None, ctypes.byref(b), 0, None, None) == 7
    assert L.skn_paged_attn(None, ctypes.byref(b), None, 1, 1.0, 0, 0, None) == 7
    assert L.skn_paged_attn_dev(None, ctypes.byref(b), 0, None, 0, 1, 1.0, 0, 0, None, 0) == 7
    assert L.skn_paged_pool_bytes(None, None) == 8


def test_names_are_refused():
    for kw in ({"dtype": "f32"}, {"rot_pairs": "thirds"}):
        with pytest.raises(ValueError):
            skn.PagedKVCache(None, 1, 16, 1, 64, **kw)
    with pytest.raises(ValueError):
        skn.PagedKVCache.pool_bytes(1, 16, 1, 64, "q8_0")
