"""References of the paged-cache operators in 64 bits (plain loops over requests and heads), with the
error an implementation may have, derived from the roundings it makes."""
import numpy as np

H = {np.dtype(np.float16): 2.0 ** -11, np.dtype(np.float32): 2.0 ** -24}  # half a step, relative


def ceil_div(a, b):
    return -(-a // b)


def plan(past, new, free, table, page, n_pages, capacity):
    """Loop form of page_plan; table is not modified."""
    table = np.array(table)
    width = table.shape[1]
    cu, kv, pos, slots, taken, short = [0], [], [], [], 0, 0
    for s, (x, y) in enumerate(zip(past, new)):
        x, y = max(int(x), 0), max(int(y), 0)
        had = min(ceil_div(x, page), width)
        need = max(0, min(ceil_div(x + y, page), width) - had) if y else 0
        for i in range(need):
            f = int(free[taken + i]) if taken + i < len(free) else -1
            table[s, had + i] = f if 0 <= f < n_pages else -1
        short += bool(y and (x + y > width * page or (need and table[s, had + need - 1] < 0)))
        taken += need
        kv.append(x + y)
        for i in range(y):
            p = x + i
            f = int(table[s, p // page]) if p // page < width else -1
            pos.append(p)
            slots.append(f * page + p % page if 0 <= f < n_pages else -1)
        cu.append(cu[-1] + y)
    counts = [cu[-1], taken, short]
    pad = max(0, capacity - len(pos))
    i32 = lambda v: np.array(v, np.int32)  # noqa: E731
    return dict(table=table.astype(np.int32), cu=i32(cu), kv=i32(kv), pos=i32((pos + [-1] * pad)[:capacity]),
                slots=i32((slots + [-1] * pad)[:capacity]), counts=i32(counts))


def norm_rope(x, w, bias, eps, cs, pos, interleaved, out_dtype):
    """(y, tolerance) of [tokens, heads, d]; cs [n_positions, rot] or None."""
    d = x.shape[-1]
    u = 2.0 ** -24
    y = x.astype(np.float64)
    rel = 0.0
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * (w.astype(np.float64) + bias)
        # sum of d squares (d / 8 lanes of 8, then a tree: at most 8 + 6 roundings deep, halved by the root),
        # mean, + eps, root, reciprocal, weight + bias, two products
        rel = (16 / 2 + 8) * u
    mag = np.abs(y)
    if cs is not None:
        rot = cs.shape[1]
        half = rot // 2
        c, s = cs[pos, :half].astype(np.float64)[:, None], cs[pos, half:].astype(np.float64)[:, None]
        i = np.arange(0, rot, 2) if interleaved else np.arange(half)
        j = i + 1 if interleaved else i + half
        a, b = y[..., i].copy(), y[..., j].copy()
        y[..., i], y[..., j] = a * c - b * s, b * c + a * s
        m = np.abs(a) + np.abs(b)
        mag[..., i] = mag[..., j] = m
        rel = rel + 3 * u  # product, product, sum
    tol = rel * mag + H[np.dtype(out_dtype)] * np.abs(y) * (1 + 1e-3) + (2.0 ** -25 if out_dtype == np.float16 else 1e-37)
    return y, tol


def attention(q, rows, kv_len, new, softcap=0.0, window=0, scale=None, dtype=np.float16):
    """(out, tolerance) of one request: q [new, Hq, d], rows = (k, v) [kv_len, Hkv, d] as stored."""
    k, v = rows
    n, hq, d = q.shape
    hkv = k.shape[1]
    g = hq // hkv
    scale = d ** -0.5 if scale is None else scale
    u = 2.0 ** -24
    out, tol = np.zeros((n, hq, d)), np.zeros((n, hq, d))
    for i in range(n):
        pos = kv_len - new + i
        lo, hi = max(0, pos - window + 1) if window else 0, min(pos, kv_len - 1) + 1
        if hi <= lo:
            continue
        for h in range(hq):
            kk, vv = k[lo:hi, h // g].astype(np.float64), v[lo:hi, h // g].astype(np.float64)
            qq = q[i, h].astype(np.float64)
            s = kk @ qq * scale
            size = float((np.abs(kk) @ np.abs(qq)).max() * abs(scale))  # of the terms a logit is summed from
            if softcap:
                s = softcap * np.tanh(s / softcap)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ vv
            a = p @ np.abs(vv)
            # logits: d products summed in F32 (and, for F32 queries, q held as two halves: 2^-22), scaled by
            # rounded factors; a soft cap moves nothing further apart but its own evaluation, ~8 roundings of
            # the cap.  A relative error of the weights is twice the logits' absolute one (weight and sum).
            logit = (d + 8) * u * size + (2.0 ** -22 * size if dtype == np.float32 else 0.0) + 8 * u * softcap
            w = 2 * logit + 16 * u + 2 * ((hi - lo) / 16 + 64) * u  # exp2, accumulation in steps of 16 keys
            # probabilities rounded to F16, or held as two halves (2^-22 each, down to 2^-25 of the largest
            # weight, which is 2^8 times smaller where the reference maximum trails); the same in the sum
            half = 2.0 ** -11 if dtype == np.float16 else 2.0 ** -21
            floor = (2.0 ** -25 if dtype == np.float16 else 2.0 ** -25) * np.abs(vv).sum(0) * p.max()
            tol[i, h] = a * (w + 2 * half) + 2 * floor + H[np.dtype(dtype)] * np.abs(out[i, h]) * (1 + 1e-3)
            tol[i, h] += 2.0 ** -25 if dtype == np.float16 else 1e-37
    return out, tol


def within(got, ref, tol, what=""):
    got = np.asarray(got, np.float64)
    assert np.isfinite(got).all(), what + ": not finite"
    over = np.abs(got - ref) - tol
    assert (over <= 0).all(), "%s: worst error %g over a tolerance of %g at %s" % (
        what, np.abs(got - ref).reshape(-1)[over.argmax()], tol.reshape(-1)[over.argmax()], np.unravel_index(over.argmax(), over.shape))


def make_cache(rng, past, new, page, hkv, d, seq_major=False, spare=3, poison=True):
    """Random pools holding every request's tokens in randomly ordered pages: (k_pool, v_pool, table,
    n_pages, [(k, v) of every request]).  Rows that belong to nobody hold NaN when `poison`."""
    want = [ceil_div(x + y, page) for x, y in zip(past, new)]
    n = sum(want) + spare
    order = rng.permutation(n)
    width = max(want + [1]) + 2
    table = np.full((len(past), width), -1, np.int32)
    pools = [np.full((n, page, hkv, d), np.nan if poison else 0.0, np.float16) for _ in range(2)]
    rows, at = [], 0
    for s, (x, y) in enumerate(zip(past, new)):
        mine = order[at:at + want[s]]
        at += want[s]
        table[s, :want[s]] = mine
        both = [rng.standard_normal((x + y, hkv, d), dtype=np.float32).astype(np.float16) for _ in range(2)]
        for pool, r in zip(pools, both):
            for i, pg in enumerate(mine):
                part = r[i * page:(i + 1) * page]
                pool[pg, :len(part)] = part
        rows.append(both)
    if not seq_major:
        pools = [np.ascontiguousarray(p.transpose(0, 2, 1, 3)) for p in pools]
    return pools[0], pools[1], table, n, rows
