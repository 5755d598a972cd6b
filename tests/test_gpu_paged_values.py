"""paged_attention on values that move a softmax's reference, leave F16's range or are not finite, over
requests long enough for every part of the kernels; against plain softmax attention in 64 bits."""
import numpy as np
import pytest

import paged_util as U
from test_gpu_paged_attention import NP, call, setup

pytestmark = pytest.mark.gpu
SHAPES = {64: (14, 2), 128: (8, 2), 256: (4, 2)}


def reference(q, k, v, kv_len, softcap=0.0, window=0, scale=None):
    """(out, tolerance) of one request, q [new, Hq, d]; keys whose logit is -inf have no weight without a cap.

    Errors, u = 2^-24: a logit is d products summed in F32, scaled by rounded factors, F32 queries held as two
    F16 halves (2^-22 of the terms' size), the cap's own evaluation ~8 roundings of the cap; a weight is off by
    twice that (weight and sum).  Sums run over steps of 16 keys.  F16: weights rounded to F16 (2^-11 each, and
    in the sum), then the output.  F32: weights are two halves, 2^-22 each.  Where a half is below F16's smallest
    normal number it is off by half of its smallest step instead, 2^-25; F32 rows are weighed with 2^10 at least
    in the place of 1, which makes that 2^-35 of the largest weight."""
    f16 = q.dtype == np.float16
    n, hq, d = q.shape
    g = hq // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    u = 2.0 ** -24
    pos = kv_len - n + np.arange(n)
    key = np.arange(kv_len)
    sees = key <= pos[:, None]
    if window:
        sees &= key > pos[:, None] - window
    out, tol = np.zeros((n, hq, d)), np.zeros((n, hq, d))
    for h in range(hq):
        qq, kk, vv = q[:, h].astype(np.float64), k[:, h // g].astype(np.float64), v[:, h // g].astype(np.float64)
        with np.errstate(invalid="ignore"):
            s = qq @ kk.T * scale
        assert not np.isnan(s).any() and not (s == np.inf).any()
        see = sees & ((s != -np.inf) | (softcap > 0))  # a cap makes them finite
        size = np.where(see, np.abs(qq) @ np.where(np.isfinite(kk), np.abs(kk), 0).T, 0).max(1) * abs(scale)
        if softcap:
            s = softcap * np.tanh(s / softcap)
        s = np.where(see, s, -np.inf)
        top = s.max(1, keepdims=True)
        p = np.exp(s - np.where(np.isfinite(top), top, 0))
        total = p.sum(1, keepdims=True)
        p = np.divide(p, total, out=np.zeros_like(p), where=total > 0)
        o = p @ vv
        a = p @ np.abs(vv)
        logit = (d + 8) * u * size + (0.0 if f16 else 2.0 ** -22 * size) + 8 * u * softcap
        w = 2 * logit + 16 * u + 2 * (see.sum(1) / 16 + 64) * u
        half = 2.0 ** -11 if f16 else 2.0 ** -21
        floor = (2.0 ** -25 if f16 else 2.0 ** -35) * (see @ np.abs(vv)) * p.max(1, keepdims=True)
        out[:, h] = o
        tol[:, h] = a * (w + 2 * half)[:, None] + 2 * floor + (2.0 ** -11 if f16 else u) * np.abs(o) * (1 + 1e-3) + (2.0 ** -25 if f16 else 1e-37)
    return out, tol


def check(st, got, what="", **kw):
    cu, kv = st["cu"], st["kv"]
    for s, (k, v) in enumerate(st["rows"]):
        ref, tol = reference(st["q"][cu[s]:cu[s + 1]], k, v, int(kv[s]), **kw)
        U.within(got[cu[s]:cu[s + 1]], ref, tol, "%s request %d" % (what, s))
    assert (got[cu[-1]:] == -9.0).all()


def put(st, s, keys, k=None, v=None, ch=slice(None)):
    """Sets channels `ch` of K and / or V of request s's tokens, in the pools and in the contiguous rows."""
    page = st["kc"].shape[2]
    for t in keys:
        for pool, row, x in ((st["kc"], st["rows"][s][0], k), (st["vc"], st["rows"][s][1], v)):
            if x is not None:
                row[t, :, ch] = x
                pool[st["table"][s, t // page], :, t % page, ch] = x


def levels(seed, past, new, d, ty, page=16):
    """A call whose channel 0 only adds to the logits: queries hold 8 there, keys 0 (see put)."""
    hq, hkv = SHAPES[d]
    st = setup(seed, past, new, hq, hkv, d, page, ty, gain=1.0)
    st["q"][:st["cu"][-1], :, 0] = 8.0
    for s in range(len(past)):
        put(st, s, range(past[s] + new[s]), k=0.0, ch=0)
    return st


@pytest.mark.parametrize("ty", ["f16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("softcap", [0.0, 80.0])
def test_keys_far_above_the_first_ones(softcap, d, ty):
    """Keys 12, 20, 30 and 60 nats above those in front of them, where tiles are taken without a maximum:
    tiles of even and odd number, keys in both halves of a tile, rows that see several of them, and a level
    that rises again."""
    nat = np.sqrt(d) / 8
    for past, new in (([1100], [48]), ([1800], [3]), ([0], [900]), ([2600, 700], [70, 130])):
        for jump in (12.0, 20.0, 30.0, 60.0):
            st = levels(d + past[0], past, new, d, ty)
            for s in range(len(past)):
                n = past[s] + new[s]
                for i, at in enumerate((n // 5, n // 5 + 17, n // 3, n // 2, n // 2 + 33, n // 2 + 65, n * 3 // 4)):
                    put(st, s, [at], k=nat * (jump + (i > 4)), ch=0)
            check(st, call(st, softcap), "jump %g past %r" % (jump, past), softcap=softcap)
        st = levels(d + past[0] + 1, past, new, d, ty)  # a level that climbs by 4 nats every 80 keys
        for s in range(len(past)):
            for t in range(past[s] + new[s]):
                put(st, s, [t], k=nat * min(4.0 * (t // 80), 70.0), ch=0)
        check(st, call(st, softcap), "climbing past %r" % (past,), softcap=softcap)


def infinite(st, s, keys):
    """The logits of these keys are -inf in every row: K holds -inf where all queries hold 1."""
    st["q"][:st["cu"][-1], :, 1] = 1.0
    put(st, s, keys, k=-np.inf, ch=1)


@pytest.mark.parametrize("ty", ["f16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_an_infinite_key_in_the_tile_behind_the_unmasked_steps(d, ty):
    """408 tokens in tiles of 32 keys (64 at d 64), none cut: the steps without a maximum end with tile 9 (3).
    The tile behind them holds the key; the one two further on, which takes its place, does not."""
    for past, new in (([360], [48]), ([360, 40], [48, 60])):
        for at in ((256, 259, 318) if d == 64 else (320, 325, 350)):
            st = setup(d + at, past, new, *SHAPES[d], d, 16, ty, gain=1.0)
            infinite(st, 0, [at])
            check(st, call(st), "key %d" % at)


@pytest.mark.parametrize("ty", ["f16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_whose_first_tiles_are_all_minus_infinity(d, ty):
    """The first keys have no weight in any row; the ones behind them are ordinary, or far below zero (they
    vanish against a reference of 0), with a long and a short end behind them."""
    for past, new in (([1100], [48]), ([0], [700]), ([2900, 350], [40, 60])):
        for level in (0.0, -200.0):
            st = levels(d + past[0] + 2, past, new, d, ty)
            for s in range(len(past)):
                put(st, s, range(past[s] + new[s]), k=np.sqrt(d) / 8 * level, ch=0)
                infinite(st, s, range(80))
            check(st, call(st), "level %g past %r" % (level, past))


@pytest.mark.parametrize("ty", ["f16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_infinite_keys_anywhere(d, ty):
    """Keys of -inf logits in tiles that are taken without masks: they have no weight, and a row that sees no
    other key is zeros."""
    for past, new in (([1100], [48]), ([0], [900]), ([2900, 350], [40, 60]), ([1500, 700], [1, 1]), ([400], [2])):
        st = levels(d + past[0] + 3, past, new, d, ty)
        for s in range(len(past)):
            n = past[s] + new[s]
            infinite(st, s, [n // 7, n // 3, n // 3 + 1, n // 2, n - 3] + list(range(n // 5, n // 5 + 150)))
        check(st, call(st), "past %r" % (past,))
        check(st, call(st, window=600), "window past %r" % (past,), window=600)
        check(st, call(st, softcap=4.0), "capped past %r" % (past,), softcap=4.0)
        for s in range(len(past)):
            infinite(st, s, range(past[s] + new[s]))
        assert (call(st)[:st["cu"][-1]] == 0).all()


@pytest.mark.parametrize("ty", ["f16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_key_that_is_not_a_number_reaches_the_rows_that_see_it(d, ty):
    for past, new, at in ((1100, 48, 200), (0, 900, 500), (2900, 40, 2920)):
        st = setup(d + at, [past], [new], *SHAPES[d], d, 16, ty, gain=1.0)
        clean = call(st)
        put(st, 0, [at], k=np.nan, ch=5)
        got = call(st)[:new]
        sees = past + np.arange(new) >= at
        assert np.isnan(got[sees]).all() and np.array_equal(got[~sees], clean[:new][~sees])


@pytest.mark.parametrize("ty", ["f16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_an_infinite_value_that_all_rows_see(d, ty):
    """A channel of V that holds an infinity is that infinity in the rows that see the key, NaN where they see
    both; other channels and other heads keep their bits."""
    hq, hkv = SHAPES[d]
    g = hq // hkv
    for past, new, window in ((1100, 48, 0), (0, 900, 0), (2900, 40, 0), (1500, 1, 0), (1500, 1, 300), (400, 2, 0), (9000, 1, 0)):
        st = setup(d + past, [past], [new], hq, hkv, d, 16, ty, gain=0.3)
        clean = call(st, window=window)
        first, second = past + new - 250, past + new - 200
        pool = st["vc"].transpose(0, 2, 1, 3)  # [page, token, head, channel]
        spot = lambda t, h, c, x: pool[st["table"][0, t // 16]].__setitem__((t % 16, h, c), x)  # noqa: E731
        spot(first, 1, 7, np.inf)
        spot(first, 1, 9, -np.inf)
        spot(first, 1, 11, np.inf)
        spot(second, 1, 11, -np.inf)
        got = call(st, window=window)
        pos = past + np.arange(new)[:, None]
        sees = lambda t: (pos >= t) & ((window == 0) | (pos - window < t))  # noqa: E731
        want = clean[:new].copy()
        mine = want[:, g:2 * g]
        mine[..., 7] = np.where(sees(first), np.inf, mine[..., 7])
        mine[..., 9] = np.where(sees(first), -np.inf, mine[..., 9])
        mine[..., 11] = np.where(sees(first), np.inf, mine[..., 11])
        mine[..., 11] = np.where(sees(second), np.where(sees(first), np.nan, -np.inf), mine[..., 11])
        special = ~np.isfinite(want)
        assert np.array_equal(got[:new][special], want[special], equal_nan=True), (past, new)
        rest = got[:new][~special]
        if ty == "f16" or new < 3:
            assert np.array_equal(rest, want[~special]), (past, new)
        else:  # a row that was formed again may differ in its last bits
            whole = ~special.any(-1)
            assert np.array_equal(got[:new][whole], want[whole]), (past, new)
            assert (np.abs(rest - want[~special]) <= 1e-4).all(), (past, new)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("softcap", [0.0, 90.0])
def test_a_long_tail_far_below_one_key_counts_in_f32(softcap, d):
    """One key takes nearly all the weight and holds 0 in V; what is left of the result is the thousands of keys
    17 to 22 nats below it."""
    for past, new in ((8191, 1), (8000, 48), (0, 1000), (20000, 2)):
        for at in (10, (past + new) // 2, past):
            for nats in (17.5, 20.0, 22.0):
                st = levels(d + past + 4, [past], [new], d, "f32")
                put(st, 0, [at], k=np.sqrt(d) / 8 * nats, ch=0)
                st["vc"][:] = np.abs(st["vc"])
                st["rows"][0][1][:] = np.abs(st["rows"][0][1])
                put(st, 0, [at], v=0.0)
                check(st, call(st, softcap), "%g nats at %d of %d" % (nats, at, past + new), softcap=softcap)


def test_a_step_whose_bounds_leave_no_request_a_token():
    # rows of a batch of fixed size, every request idle: whoever brings tokens would bring more than there are
    st = setup(1, [20, 5], [0, 0], 4, 2, 64, 16, "f16", pad_rows=4)
    assert (call(st, hints=False, min_new=8) == -9.0).all()
    assert (call(st, hints=False, min_new=8, max_new=8) == -9.0).all()


@pytest.mark.parametrize("ty", ["f16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_infinite_queries(d, ty):
    """A row whose query holds an infinity where all its keys have one sign: all logits -inf, the row is zeros;
    all +inf, NaN.  The size of its other channels does not matter; other rows are right (their bits may differ:
    rows of a workgroup share the choice of steps)."""
    for past, new in ((1100, 48), (700, 1), (900, 2), (0, 300)):
        st = setup(d + past + 5, [past], [new], *SHAPES[d], d, 16, ty, gain=100.0)
        put(st, 0, range(past + new), k=0.5, ch=2)
        st["q"][:new, :, 2] = 0.0
        ordinary = st["q"].copy()
        st["q"][0, 0, 2], st["q"][new - 1, 1, 2] = -np.inf, np.inf
        got = call(st)
        assert (got[0, 0] == 0).all() and np.isnan(got[new - 1, 1]).all(), (past, new)
        st["q"] = ordinary
        base = call(st)
        got[0, 0], got[new - 1, 1] = base[0, 0], base[new - 1, 1]
        check(st, got, "beside infinite queries, past %d" % past)


@pytest.mark.parametrize("ty", ["f16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("size,scale,softcap", [(1.0, 3.3e38, 0.0), (1.0, 10.0, 1.2e-38), (1e38, 1e5, 0.0), (1e38, 1.0, 1e-3), (1e38, -1e5, 0.0)])
def test_keys_of_zero_under_the_largest_factors(size, scale, softcap, d, ty):
    """Logits of zero stay zero whatever they are multiplied by: the rows are means."""
    if ty == "f16" and size > 60000:
        size = 60000.0
    for past, new in (([300], [60]), ([90], [1])):
        st = setup(d + past[0] + 6, past, new, *SHAPES[d], d, 16, ty, gain=0.2)
        st["q"] = (st["q"] * np.float32(size)).astype(NP[ty])
        put(st, 0, range(past[0] + new[0]), k=0.0)
        got = call(st, softcap, scale=scale)
        st["q"][:new[0]] = 0.0
        check(st, got, "scale %g cap %g" % (scale, softcap))
