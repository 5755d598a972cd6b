"""qk_norm_rope on the GPU against the formulas in 64 bits; the tolerance counts the roundings."""
import numpy as np
import pytest

import paged_util as U
from gpu_util import ctx, dev, host

pytestmark = pytest.mark.gpu
NP = {"f16": np.float16, "f32": np.float32}


def inputs(rng, t, hq, hkv, d, ty, rot, n_pos):
    x = rng.standard_normal((t, hq + 2 * hkv, d), dtype=np.float32).astype(NP[ty])
    ang = rng.uniform(0, 6.3, (n_pos, rot // 2)) if rot else None
    cs = np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32) if rot else None
    return x, cs, rng.integers(0, n_pos, t).astype(np.int32)


def run(x, cs, pos, hq, hkv, page, n_pages, slots, out, wq=None, wk=None, bias=0.0, pairs=False, seq_major=False, eps=1e-6, fused=True,
        in_place=False):
    """(q_out, K pool, V pool): pools and q_out start as sentinels."""
    import argus_hip as A
    import torch
    t, _, d = x.shape
    shape = (n_pages, page, hkv, d) if seq_major else (n_pages, hkv, page, d)
    kc, vc = (torch.full(shape, 3.0, dtype=torch.float16, device="cuda") for _ in range(2))
    xd = dev(x)
    q, k, v = xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:]
    if not fused:
        q, k, v = (z.contiguous() for z in (q, k, v))
    q_out = q if in_place else torch.full((t, hq, d), 3.0, dtype=getattr(torch, {"f16": "float16", "f32": "float32"}[out]), device="cuda")
    opt = lambda w: None if w is None else dev(w)  # noqa: E731
    ctx().qk_norm_rope(q, k, v, opt(pos), opt(cs), q_out, kc, vc, dev(slots), q_weight=opt(wq), k_weight=opt(wk), eps=eps, weight_bias=bias,
                       interleaved=pairs, layout=A.SEQ_MAJOR if seq_major else A.HEAD_MAJOR)
    pools = [host(c) if seq_major else host(c).transpose(0, 2, 1, 3) for c in (kc, vc)]
    return host(q_out), pools[0].reshape(-1, hkv, d), pools[1].reshape(-1, hkv, d)


def check(x, cs, pos, hq, hkv, slots, got, out, wq, wk, bias, pairs, eps=1e-6):
    q, kc, vc = got
    live = np.ones(len(x), bool) if pos is None else (pos >= 0) & ((cs is None) | (pos < (0 if cs is None else len(cs))))
    kept = live & (slots >= 0) & (slots < len(kc))
    safe = None if pos is None else np.where(live, pos, 0)
    ref, tol = U.norm_rope(x[:, :hq], wq, bias, eps, cs, safe, pairs, NP[out])
    U.within(q[live], ref[live], tol[live], "q")
    assert (q[~live] == 3.0).all(), "a padding row was written"
    ref, tol = U.norm_rope(x[:, hq:hq + hkv], wk, bias, eps, cs, safe, pairs, np.float16)
    U.within(kc[slots[kept]], ref[kept], tol[kept], "k")
    assert np.array_equal(vc[slots[kept]], x[:, hq + hkv:].astype(np.float16)[kept])
    rest = np.ones(len(kc), bool)
    rest[slots[kept]] = False
    assert (kc[rest] == 3.0).all() and (vc[rest] == 3.0).all(), "a row that is no token's slot was written"


@pytest.mark.parametrize("t,hq,hkv,d,rot,page,ty,out,norm,pairs,seq_major", [
    (1, 32, 8, 128, 128, 16, "f32", "f32", True, False, False),
    (5, 32, 8, 128, 128, 16, "f16", "f16", True, False, True),
    (33, 14, 2, 64, 64, 32, "f16", "f32", True, True, False),
    (70, 14, 2, 64, 32, 16, "f32", "f16", False, False, False),
    (17, 8, 4, 256, 256, 64, "f16", "f16", True, False, False),
    (129, 8, 4, 256, 128, 16, "f32", "f32", True, True, True),
    (9, 3, 1, 128, 8, 16, "f16", "f16", True, False, False),
    (9, 3, 1, 128, 120, 16, "f32", "f32", True, True, False),
    (9, 5, 5, 64, 56, 1024, "f32", "f16", False, True, False),
    (21, 32, 8, 128, 0, 16, "f16", "f16", True, False, False),
    (1000, 4, 2, 64, 64, 16, "f16", "f16", True, False, False),
])
def test_against_formulas(t, hq, hkv, d, rot, page, ty, out, norm, pairs, seq_major):
    rng = np.random.default_rng(t * d + rot)
    x, cs, pos = inputs(rng, t, hq, hkv, d, ty, rot, 300)
    n_pages = U.ceil_div(t, page) + 3
    slots = rng.permutation(n_pages * page)[:t].astype(np.int32)
    bias = 1.0 if pairs else 0.0
    wq, wk = ((1 - bias + 0.3 * rng.standard_normal(d)).astype(np.float32) if norm else None for _ in range(2))
    for fused in (True, False):
        got = run(x, cs, pos if rot else None, hq, hkv, page, n_pages, slots, out, wq, wk, bias, pairs, seq_major, fused=fused)
        check(x, cs, pos if rot else None, hq, hkv, slots, got, out, wq, wk, bias, pairs)


def test_padding_tokens_and_tokens_without_a_slot():
    rng = np.random.default_rng(2)
    x, cs, pos = inputs(rng, 40, 8, 2, 128, "f16", 128, 50)
    slots = rng.permutation(5 * 16)[:40].astype(np.int32)
    pos[[3, 11, 39]] = -1, 50, 2 ** 31 - 1
    slots[[4, 12]] = -1, 80
    w = np.ones(128, np.float32)
    got = run(x, cs, pos, 8, 2, 16, 5, slots, "f16", w, w)
    check(x, cs, pos, 8, 2, slots, got, "f16", w, w, 0.0, False)
    # no rotation: positions only mark padding
    got = run(x, None, pos, 8, 2, 16, 5, slots, "f16", w, w)
    check(x, None, pos, 8, 2, slots, got, "f16", w, w, 0.0, False)


def test_only_one_of_the_two_norms_and_a_zero_row():
    rng = np.random.default_rng(5)
    x, cs, pos = inputs(rng, 6, 4, 2, 64, "f32", 64, 50)
    x[2] = 0.0  # mean of squares 0: eps alone
    slots = np.arange(6, dtype=np.int32)
    w = (1 + 0.2 * rng.standard_normal(64)).astype(np.float32)
    for wq, wk in ((w, None), (None, w)):
        check(x, cs, pos, 4, 2, slots, run(x, cs, pos, 4, 2, 16, 2, slots, "f32", wq, wk, eps=1e-5), "f32", wq, wk, 0.0, False, eps=1e-5)


def test_in_place_queries():
    rng = np.random.default_rng(6)
    x, cs, pos = inputs(rng, 50, 8, 2, 128, "f16", 64, 90)
    slots = np.arange(50, dtype=np.int32)
    w = np.ones(128, np.float32)
    a = run(x, cs, pos, 8, 2, 16, 4, slots, "f16", w, w)
    b = run(x, cs, pos, 8, 2, 16, 4, slots, "f16", w, w, in_place=True)
    for u, v in zip(a, b):
        assert np.array_equal(u, v)


def test_infinite_and_nan_inputs_stay_in_their_head():
    rng = np.random.default_rng(7)
    x, cs, pos = inputs(rng, 4, 4, 2, 64, "f16", 64, 50)
    y = x.copy()
    y[1, 2, 5], y[2, 4, 0] = np.inf, np.nan  # a query head, a key head
    slots = np.arange(4, dtype=np.int32)
    w = np.ones(64, np.float32)
    a, b = (run(z, cs, pos, 4, 2, 16, 1, slots, "f16", w, w) for z in (x, y))
    same_q, same_k = np.ones((4, 4), bool), np.ones((16, 2), bool)
    same_q[1, 2], same_k[2, 0] = False, False
    assert np.array_equal(a[0][same_q], b[0][same_q]) and np.array_equal(a[1][same_k], b[1][same_k]) and np.array_equal(a[2], b[2])
    assert np.isnan(b[0][1, 2]).any() and np.isnan(b[1][2, 0]).any()


def test_a_pool_beyond_32_bit_offsets():
    # 2^20 + 2 pages of 16 tokens x 2 heads x 128 channels: 8.6 GB per pool, the last page behind 2^32 elements
    import torch
    rng = np.random.default_rng(8)
    n, hkv, d = (1 << 20) + 2, 2, 128
    x, cs, pos = inputs(rng, 3, 4, hkv, d, "f16", 128, 50)
    kc, vc = (torch.empty((n, hkv, 16, d), dtype=torch.float16, device="cuda") for _ in range(2))
    kc[-1], vc[-1] = 3.0, 3.0
    slots = np.array([(n - 1) * 16 + 15, (n - 1) * 16, 7], np.int32)
    xd = dev(x)
    q_out = torch.empty((3, 4, d), dtype=torch.float16, device="cuda")
    ctx().qk_norm_rope(xd[:, :4], xd[:, 4:6], xd[:, 6:], dev(pos), dev(cs), q_out, kc, vc, dev(slots))
    ref, tol = U.norm_rope(x[:, 4:6], None, 0.0, 0.0, cs, pos, False, np.float16)
    last = host(kc[-1])
    U.within(last[:, 15], ref[0], tol[0], "last row")
    U.within(last[:, 0], ref[1], tol[1], "first row of the last page")
    U.within(host(kc[0])[:, 7], ref[2], tol[2], "page 0")
    assert np.array_equal(host(vc[-1])[:, 15], x[0, 6:]) and (last[:, 1:15] == 3.0).all()


def test_refusals():
    import argus_hip as A
    import torch
    c = ctx()
    f = lambda *s, ty=torch.float16: torch.zeros(s, dtype=ty, device="cuda")  # noqa: E731
    i = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731

    def call(q=None, k=None, v=None, pos=None, cs=None, out=None, kc=None, vc=None, slots=None, **kw):
        q = f(2, 4, 64) if q is None else q
        kc = f(3, 2, 16, 64) if kc is None else kc
        return c.qk_norm_rope(q, f(2, 2, 64) if k is None else k, f(2, 2, 64) if v is None else v, i(2) if pos is None else pos,
                              f(5, 64, ty=torch.float32) if cs is None else cs, f(2, 4, 64) if out is None else out, kc,
                              kc.clone() if vc is None else vc, i(2) if slots is None else slots, check=False, **kw)

    assert call() == A.OK
    assert call(cs=f(5, 60, ty=torch.float32)) == A.ERR_INVALID and call(cs=f(5, 72, ty=torch.float32)) == A.ERR_INVALID
    assert call(kc=f(3, 2, 24, 64)) == A.ERR_UNSUPPORTED
    assert call(q=f(2, 4, 96), k=f(2, 2, 96), v=f(2, 2, 96), out=f(2, 4, 96), kc=f(3, 2, 16, 96)) == A.ERR_UNSUPPORTED
    odd = f(2 * 4 * 64 + 1)[1:].view(2, 4, 64)
    assert call(q=odd) == A.ERR_INVALID and call(out=odd) == A.ERR_INVALID
    assert call(q=f(2, 4 * 64 + 2)[:, :256].view(2, 4, 64)) == A.ERR_INVALID
    for bad in (dict(k=f(2, 3, 64)), dict(out=f(3, 4, 64)), dict(slots=i(3)), dict(vc=f(4, 2, 16, 64)), dict(q_weight=f(63, ty=torch.float32))):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(k=f(2, 2, 64, ty=torch.float32)), dict(kc=f(3, 2, 16, 64, ty=torch.float32)), dict(q_weight=f(64)),
                dict(q=f(2, 4, 64, ty=torch.bfloat16), k=f(2, 2, 64, ty=torch.bfloat16), v=f(2, 2, 64, ty=torch.bfloat16))):
        with pytest.raises(TypeError):
            call(**bad)
    # nothing to do
    assert call(q=f(0, 4, 64), k=f(0, 2, 64), v=f(0, 2, 64), out=f(0, 4, 64), pos=i(0), slots=i(0)) == A.OK
