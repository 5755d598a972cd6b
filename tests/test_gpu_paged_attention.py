"""paged_attention on the GPU against plain softmax attention in 64 bits, request by request."""
import numpy as np
import pytest

import paged_util as U
from gpu_util import ctx, dev, host

pytestmark = pytest.mark.gpu
NP = {"f16": np.float16, "f32": np.float32}


def setup(seed, past, new, hq, hkv, d, page, ty, seq_major=False, poison=True, gain=1.5, pad_rows=3):
    """Device tensors of one call; rows of q behind the last request hold NaN."""
    rng = np.random.default_rng(seed)
    kc, vc, table, n_pages, rows = U.make_cache(rng, past, new, page, hkv, d, seq_major, poison=poison)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = (gain * rng.standard_normal((cu[-1] + pad_rows, hq, d), dtype=np.float32)).astype(NP[ty])
    q[cu[-1]:] = np.nan
    kv = np.array([x + y for x, y in zip(past, new)], np.int32)
    return dict(q=q, kc=kc, vc=vc, table=table, cu=cu, kv=kv, rows=rows, new=list(new), seq_major=seq_major)


def call(st, softcap=0.0, window=0, scale=0.0, hints=True, out=None, workspace=None, context=None, **kw):
    import argus_hip as A
    import torch
    d = {k: dev(st[k]) for k in ("q", "kc", "vc", "table", "cu", "kv")}
    if out is None:
        out = torch.full(st["q"].shape, -9.0, dtype=d["q"].dtype, device="cuda")
    if hints:
        kw = dict(dict(max_new=max(st["new"] + [0]), max_kv=int(max(list(st["kv"]) + [0]))), **kw)
    rc = (context or ctx()).paged_attention(d["q"], d["kc"], d["vc"], d["table"], d["cu"], d["kv"], out, softcap=softcap, window=window,
                                            scale=scale, layout=A.SEQ_MAJOR if st["seq_major"] else A.HEAD_MAJOR, workspace=workspace, **kw)
    assert rc == 0
    return host(out)


def check(st, got, softcap=0.0, window=0, scale=None, only=None):
    cu, kv = st["cu"], st["kv"]
    for s, r in enumerate(st["rows"]):
        if only is not None and s not in only:
            continue
        new = int(cu[s + 1] - cu[s])
        if not new:
            continue
        ref, tol = U.attention(st["q"][cu[s]:cu[s + 1]], r, int(kv[s]), new, softcap, window, scale, st["q"].dtype.type)
        U.within(got[cu[s]:cu[s + 1]], ref, tol, "request %d (%d new of %d)" % (s, new, kv[s]))
    assert (got[cu[-1]:] == -9.0).all(), "rows behind the last request were written"


HEADS = {"llama": (8, 2, 128), "qwen": (14, 2, 64), "gemma": (4, 2, 256), "mha": (3, 3, 64), "wide": (24, 1, 128), "one": (1, 1, 256), "huge": (200, 1, 64)}


@pytest.mark.parametrize("ty", ["f16", "f32"])
@pytest.mark.parametrize("heads", ["llama", "qwen", "gemma", "mha", "wide", "one", "huge"])
@pytest.mark.parametrize("past,new", [
    ([0], [1]), ([1], [1]), ([15], [1]), ([16], [1]), ([700], [1]),
    ([300, 0, 33, 64, 999], [1, 1, 1, 1, 1]),              # single tokens
    ([120, 17, 500], [2, 4, 3]),                           # drafts
    ([0], [37]), ([0, 5], [130, 64]), ([400, 31], [33, 129]),  # chunks
    ([600, 12, 0, 77, 250], [1, 40, 1, 0, 5]),             # mixed, one idle
])
def test_lengths_and_heads(past, new, heads, ty):
    hq, hkv, d = HEADS[heads]
    page = 16 if len(past) % 2 else 64
    st = setup(len(past) * 1000 + sum(past) + hq, past, new, hq, hkv, d, page, ty, seq_major=heads in ("qwen", "one"))
    check(st, call(st))


@pytest.mark.parametrize("ty", ["f16", "f32"])
@pytest.mark.parametrize("page", [16, 32, 128, 1024])
@pytest.mark.parametrize("softcap,window", [(50.0, 0), (0.0, 1), (0.0, 37), (5.0, 128), (0.0, 100000)])
def test_soft_cap_window_and_page_sizes(softcap, window, page, ty):
    for hq, hkv, d in ((8, 4, 256), (8, 2, 64)):
        st = setup(page + window, [500, 90, 0, 1040], [1, 70, 33, 6], hq, hkv, d, page, ty, seq_major=page == 32)
        check(st, call(st, softcap, window), softcap, window)


@pytest.mark.parametrize("ty", ["f16", "f32"])
def test_long_requests_beside_short_ones(ty):
    # requests cut along their length beside requests that are not
    st = setup(3, [6000, 3, 2500, 0, 40], [1, 1, 9, 3, 1], 8, 2, 128, 16, ty)
    check(st, call(st))
    st = setup(4, [5000, 11], [40, 2], 4, 1, 64, 32, ty)
    check(st, call(st))
    check(st, call(st, window=700), window=700)


def test_many_requests():
    rng = np.random.default_rng(0)
    past = rng.integers(0, 60, 700)
    new = rng.integers(0, 3, 700)
    st = setup(5, [int(x) for x in past], [int(x) for x in new], 2, 1, 64, 16, "f16")
    check(st, call(st))
    check(st, call(st, hints=False))


def test_thousands_of_requests_and_a_few_long_ones_among_them():
    """More requests than workgroups, in blocks of 64 with long, empty and idle ones at their borders."""
    rng = np.random.default_rng(1)
    past, new = rng.integers(0, 20, 3001), rng.integers(0, 2, 3001)
    for at, p, n in ((0, 900, 1), (63, 500, 2), (64, 700, 30), (1500, 0, 40), (2944, 300, 1), (3000, 1500, 3)):
        past[at], new[at] = p, n
    st = setup(15, [int(x) for x in past], [int(x) for x in new], 2, 1, 64, 16, "f16")
    check(st, call(st))
    st["q"] = st["q"].astype(np.float32)
    check(st, call(st, hints=False))
    one = setup(16, [int(x) for x in past], [1] * 3001, 2, 1, 64, 16, "f16")
    check(one, call(one))


@pytest.mark.parametrize("size,ty", [(1e-4, "f32"), (300.0, "f32"), (60000.0, "f32"), (1e-30, "f32"), (1e30, "f32"), (1e-4, "f16"), (60000.0, "f16")])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_queries_of_any_size(size, ty, d):
    st = setup(17, [50, 9], [1, 40], 8, 2, d, 16, "f32", gain=1.0)
    st["q"] = (st["q"] * np.float32(size / 4.5)).astype(NP[ty])
    check(st, call(st, scale=0.08 / size), scale=0.08 / size)
    check(st, call(st, softcap=3.0, scale=0.08 / size), softcap=3.0, scale=0.08 / size)


def test_hints_do_not_change_what_is_computed():
    # unknown or loose bounds: the same rows, within the tolerance of the same reference
    st = setup(6, [900, 20, 0], [1, 50, 8], 8, 2, 128, 16, "f16")
    for kw in (dict(hints=False), dict(max_new=1000), dict(max_kv=100000), dict(min_new=1), dict(max_kv=10, max_new=50)):
        check(st, call(st, **kw))
    st = setup(7, [900, 20], [60, 50], 8, 2, 128, 16, "f16")
    for kw in (dict(min_new=50), dict(min_new=60), dict(min_new=10, max_new=2000)):
        check(st, call(st, **kw))


def test_one_long_row_per_head_dim_and_a_scale():
    for hq, hkv, d in ((14, 2, 64), (16, 2, 128), (2, 1, 256)):
        st = setup(d, [9000], [1], hq, hkv, d, 16, "f32")
        check(st, call(st, scale=0.05), scale=0.05)
        check(st, call(st, scale=-0.02), scale=-0.02)


@pytest.mark.parametrize("ty", ["f16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_unseen_keys_hold_has_no_influence(bad, d, ty):
    """The last tokens of a chunk carry NaN or infinities in K and V: rows before them must not see it."""
    for past, new, window, at in ((40, 90, 0, 100), (200, 4, 0, 202), (0, 1500, 0, 1400), (300, 3, 64, 20), (700, 80, 64, 640)):
        st = setup(past + new + d, [past], [new], 4, 2, d, 16, ty, poison=True)
        clean = call(st, window=window)
        check(st, clean, window=window)
        dirty = dict(st, kc=st["kc"].copy(), vc=st["vc"].copy())
        pg, off = st["table"][0, at // 16], at % 16
        dirty["kc"][pg, :, off], dirty["vc"][pg, :, off] = bad, bad
        dirty["vc"][pg, 0, off, 3] = 1.0
        got = call(dirty, window=window)
        pos = past + np.arange(new)
        blind = (pos < at) | ((window > 0) & (pos - window >= at))
        assert blind.any()
        assert np.array_equal(got[:new][blind], clean[:new][blind]), (past, new, at)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_visible_value_that_is_not_finite_reaches_the_rows_that_see_it(bad):
    for ty in ("f16", "f32"):
        for past, new, at in ((40, 90, 100), (200, 4, 202), (300, 1, 17), (20, 60, 3)):
            st = setup(past + at, [past], [new], 4, 2, 128, 16, ty)
            clean = call(st)
            st["vc"][st["table"][0, at // 16], 1, at % 16, 7] = bad
            got = call(st)
            pos = past + np.arange(new)
            seen = pos >= at
            hit = got[:new][seen][:, 2:, 7]  # heads of the second KV head
            assert np.isnan(hit).all() if np.isnan(bad) else ((hit == bad) | np.isnan(hit)).all() and (hit == bad).any()
            assert np.array_equal(got[:new][~seen], clean[:new][~seen])
            assert np.isfinite(got[:new, :2]).all()


def test_rows_that_see_nothing_and_requests_without_tokens():
    # more new tokens than the cache holds: the first rows stand before position 0
    for ty in ("f16", "f32"):
        for hq, hkv, d in ((8, 2, 128), (4, 2, 256), (14, 2, 64)):
            st = setup(1, [0, 10, 0], [50, 3, 2], hq, hkv, d, 16, ty)
            st["kv"] = np.array([20, 1, 0], np.int32)
            st["rows"] = [(k[:n], v[:n]) for (k, v), n in zip(st["rows"], (20, 1, 0))]
            got = call(st)
            check(st, got)
            assert (got[:30] == 0).all() and (got[50:52] == 0).all() and (got[53:55] == 0).all()


def test_logits_of_minus_infinity_and_large_logits():
    for ty in ("f16", "f32"):
        st = setup(2, [100, 30], [1, 40], 8, 2, 128, 16, ty, gain=60.0)  # logits of hundreds: one key takes all
        check(st, call(st))
        st["q"][:] = np.where(np.isnan(st["q"]), np.nan, 100.0)
        kc = st["kc"]
        kc[np.isfinite(kc)] = -np.inf  # every visible logit is -inf
        got = call(st)
        assert (got[:41] == 0).all()


def test_bad_page_numbers_stay_inside_the_pool():
    st = setup(8, [200, 300, 50], [1, 40, 1], 8, 2, 128, 16, "f16", poison=False)
    st["table"][0, 3], st["table"][0, 5], st["table"][1, 2], st["table"][1, 7] = -1, 1 << 30, st["kc"].shape[0], -(1 << 31)
    got = call(st)
    assert np.isfinite(got[:42]).all()
    check(st, got, only=[2])
    # more tokens than the table has room for
    st = setup(9, [60, 30], [1, 1], 8, 2, 128, 16, "f16", poison=False)
    st["kv"] = np.array([100000, 31], np.int32)
    got = call(st, hints=False)
    assert np.isfinite(got[:2]).all()
    check(st, got, only=[1])


def test_lengths_that_do_not_fit_the_rows():
    # device lengths that point outside q: nothing outside it is touched, the other requests are right
    st = setup(10, [60, 30, 20], [2, 3, 4], 8, 2, 128, 16, "f16", poison=False)
    st["cu"] = np.array([0, 2, 5, 1000], np.int32)
    st["kv"] = np.array([62, 33, 1015], np.int32)
    import torch
    out = torch.full((st["q"].shape[0] + 64,) + st["q"].shape[1:], -9.0, dtype=torch.float16, device="cuda")
    got = call(st, hints=False, out=out[:st["q"].shape[0]])
    assert (host(out[st["q"].shape[0]:]) == -9.0).all()
    for s in (0, 1):
        ref, tol = U.attention(st["q"][(0, 2)[s]:(2, 5)[s]], st["rows"][s], (62, 33)[s], (2, 3)[s])
        U.within(got[(0, 2)[s]:(2, 5)[s]], ref, tol)
    st["cu"] = np.array([5, 2, -7, 3], np.int32)  # not even ascending
    call(st, hints=False)


def test_strided_queries_and_outputs():
    import argus_hip as A
    import torch
    st = setup(11, [100, 7], [1, 50], 8, 2, 64, 16, "f16", pad_rows=0)
    t, hq, d = st["q"].shape
    wide = torch.zeros((t, 20, d), dtype=torch.float16, device="cuda")
    wide[:, 4:12] = dev(st["q"])
    res = torch.full((t, 2 * hq, d), -9.0, dtype=torch.float16, device="cuda")
    a = [dev(st[k]) for k in ("kc", "vc", "table", "cu", "kv")]
    assert ctx().paged_attention(wide[:, 4:12], *a, res[:, hq:], layout=A.HEAD_MAJOR) == 0
    got = host(res)
    assert (got[:, :hq] == -9.0).all()
    check(st, got[:, hq:])


def test_another_stream_and_another_context():
    import argus_hip as A
    import torch
    st = setup(12, [3000, 7], [1, 50], 8, 2, 64, 16, "f32")
    base = call(st)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = call(st)
    assert np.array_equal(got, base)
    assert np.array_equal(call(st, context=A.Context(0)), base)


def test_a_pool_beyond_32_bit_offsets():
    import torch
    rng = np.random.default_rng(13)
    n, hkv, d, page = (1 << 20) + 40, 2, 128, 16
    kc, vc = (torch.empty((n, hkv, page, d), dtype=torch.float16, device="cuda") for _ in range(2))
    past, new = [500, 3], [40, 1]
    table = np.full((2, 40), -1, np.int32)
    table[0, :34] = n - 1 - rng.permutation(36)[:34]  # all behind element 2^32
    table[1, 0] = 5
    rows = []
    for s in range(2):
        r = [rng.standard_normal((past[s] + new[s], hkv, d), dtype=np.float32).astype(np.float16) for _ in range(2)]
        for pool, x in zip((kc, vc), r):
            for i in range(U.ceil_div(len(x), page)):
                part = dev(x[i * page:(i + 1) * page]).transpose(0, 1)
                pool[int(table[s, i]), :, :part.shape[1]] = part
        rows.append(r)
    cu = np.array([0, 40, 41], np.int32)
    for ty in ("f16", "f32"):
        q = rng.standard_normal((41, 8, d), dtype=np.float32).astype(NP[ty])
        out = torch.empty((41, 8, d), dtype=getattr(torch, {"f16": "float16", "f32": "float32"}[ty]), device="cuda")
        ctx().paged_attention(dev(q), kc, vc, dev(table), dev(cu), dev(np.array([540, 4], np.int32)), out)
        got = host(out)
        for s in range(2):
            ref, tol = U.attention(q[cu[s]:cu[s + 1]], rows[s], past[s] + new[s], new[s], dtype=NP[ty])
            U.within(got[cu[s]:cu[s + 1]], ref, tol, ty)
    # the first of a chunk, alone: the single-token kernel on the far pages
        one = np.array([0, 1, 2], np.int32)
        ctx().paged_attention(dev(q), kc, vc, dev(table), dev(one), dev(np.array([540, 4], np.int32)), out, max_new=1)
        got = host(out)
        for s in range(2):
            ref, tol = U.attention(q[s:s + 1], rows[s], past[s] + new[s], 1, dtype=NP[ty])
            U.within(got[s:s + 1], ref, tol, ty)


def test_the_same_call_gives_the_same_bits():
    for ty in ("f16", "f32"):
        st = setup(14, [4000, 900, 0], [1, 30, 200], 8, 2, 128, 16, ty)
        a = call(st)
        for _ in range(3):
            assert np.array_equal(call(st), a)


def test_refusals():
    import argus_hip as A
    import torch
    f = lambda *s, ty=torch.float16: torch.zeros(s, dtype=ty, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731

    def go(q=None, kc=None, vc=None, table=None, cu=None, kv=None, out=None, **kw):
        q = f(4, 4, 64) if q is None else q
        kc = f(3, 2, 16, 64) if kc is None else kc
        return ctx().paged_attention(q, kc, f(*kc.shape) if vc is None else vc, i(2, 3) if table is None else table,
                                     i(3) if cu is None else cu, i(2) if kv is None else kv, torch.zeros_like(q) if out is None else out,
                                     check=False, **kw)

    assert go() == A.OK
    assert go(kc=f(3, 2, 24, 64)) == A.ERR_UNSUPPORTED and go(kc=f(3, 2, 2048, 64)) == A.ERR_UNSUPPORTED
    assert go(q=f(4, 4, 96), kc=f(3, 2, 16, 96)) == A.ERR_UNSUPPORTED
    assert go(kc=f(3, 3, 16, 64)) == A.ERR_INVALID  # 4 heads over 3
    assert go(window=-1) == A.ERR_INVALID and go(softcap=-1.0) == A.ERR_INVALID and go(softcap=float("nan")) == A.ERR_INVALID and go(softcap=1e-40) == A.ERR_INVALID
    assert go(scale=float("inf")) == A.ERR_INVALID and go(max_new=-1) == A.ERR_INVALID
    odd = f(4 * 4 * 64 + 4)[4:].view(4, 4, 64)
    assert go(q=odd, out=f(4, 4, 64)) == A.ERR_INVALID and go(out=odd) == A.ERR_INVALID
    assert go(q=f(0, 4, 64)) == A.OK and go(table=i(0, 3), cu=i(1), kv=i(0)) == A.OK
    for bad in (dict(cu=i(4)), dict(table=i(3, 3)), dict(out=f(5, 4, 64)), dict(q=f(4, 64, 4).transpose(1, 2)), dict(vc=f(4, 2, 16, 64))):
        with pytest.raises(ValueError):
            go(**bad)
    for bad in (dict(kc=f(3, 2, 16, 64, ty=torch.float32)), dict(q=f(4, 4, 64, ty=torch.bfloat16)), dict(out=f(4, 4, 64, ty=torch.float32)),
                dict(kv=i(2).long())):
        with pytest.raises(TypeError):
            go(**bad)
    with pytest.raises(ValueError):
        go(table=torch.zeros((2, 3), dtype=torch.int32))  # host memory
