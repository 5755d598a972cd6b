"""Workloads of the paged-cache operators: page_plan, qk_norm_rope and paged_attention.

Each operator in its plain form (elementary torch operations, 32-bit arithmetic) and as the calls a
server makes of the library: one plan per step, then per layer the norm + rotation + cache write and
the attention over the pages.  A case is a dict of plain values; the lengths of its requests follow
from the case alone, every value and page number from the seed.
"""
import os
import sys

import torch

own = False

_ctx = None


def _context():
    """The library context a program keeps for its lifetime."""
    global _ctx
    if _ctx is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "argus-engine_amd"))
        import argus_hip
        _ctx = argus_hip.Context(0)
    return _ctx


# ---- cases -------------------------------------------------------------------------------------------
# Every case: `decodes` requests of one new token and `chunks` requests of up to `chunk` new tokens, over
# up to `past` tokens already cached (`even`: all at the maximum), in pages of `page` tokens.

def _plan(name, decodes, chunks, chunk, past, page, even=False):
    return dict(name=name, op="page_plan", decodes=decodes, chunks=chunks, chunk=chunk, past=past, page=page, even=even)


def _rope(name, tokens, hq, hkv, d, rot, page, dtype, out, norm=True, pairs=False, bias=0.0):
    return dict(name=name, op="qk_norm_rope", tokens=tokens, hq=hq, hkv=hkv, d=d, rot=rot, page=page, dtype=dtype, out=out,
                norm=norm, pairs=pairs, bias=bias)


def _attn(name, decodes, chunks, chunk, past, hq, hkv, d, page, dtype, softcap=0.0, window=0, seq_major=False, even=False):
    return dict(name=name, op="paged_attention", decodes=decodes, chunks=chunks, chunk=chunk, past=past, hq=hq, hkv=hkv, d=d,
                page=page, dtype=dtype, softcap=softcap, window=window, seq_major=seq_major, even=even)


def listed():
    return [
        # one decode step of a server with 64 running requests
        _plan("plan_step", 64, 0, 0, 4096, 16),
        # a large mixed step: 2016 running requests and 32 prompts being read in chunks
        _plan("plan_mixed", 2016, 32, 2048, 16384, 32),
        # a decode step's projections, F32 activations as the engine keeps them
        _rope("rope_decode", 16, 32, 8, 128, 128, 16, "f32", "f32"),
        # a chunk of prompt tokens, F16 activations
        _rope("rope_chunk", 8192, 32, 8, 128, 128, 64, "f16", "f16"),
        # 256-channel heads, half of the channels rotated pairwise, norm weights stored as w - 1; odd token count
        _rope("rope_odd", 1237, 8, 4, 256, 128, 16, "f32", "f16", True, True, 1.0),
        # one short request, one new token: latency
        _attn("attn_decode_one", 1, 0, 0, 1023, 14, 2, 64, 16, "f32"),
        # sixteen long requests of uneven lengths, one new token each
        _attn("attn_decode_long", 16, 0, 0, 32768, 32, 8, 128, 16, "f32"),
        # soft-capped, windowed layer with 256-channel heads, many requests
        _attn("attn_decode_window", 64, 0, 0, 8191, 8, 4, 256, 32, "f16", 50.0, 2048),
        # four drafted tokens of each of 32 requests checked at once
        _attn("attn_draft", 0, 32, 4, 8188, 32, 8, 128, 64, "f16", even=True),
        # two prompts being read in chunks of 512 behind up to 8192 cached tokens
        _attn("attn_chunk", 0, 2, 512, 8192, 32, 8, 128, 16, "f16"),
        # decode requests and two odd chunks in one call, F32 activations, token-major pages
        _attn("attn_mixed", 46, 2, 777, 6000, 14, 2, 64, 32, "f32", seq_major=True),
        # a whole prompt with nothing cached
        _attn("attn_prompt", 0, 1, 8192, 0, 32, 8, 128, 64, "f16", even=True),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["page_plan", "qk_norm_rope", "paged_attention", "paged_attention", "paged_attention"])
    page = rng.choice([16, 32, 64, 128])
    if op == "page_plan":
        c = _plan("", _log(rng, 1, 2000), rng.choice([0, _log(rng, 1, 32)]), _log(rng, 2, 2048), _log(rng, 1, 16384), page)
    elif op == "qk_norm_rope":
        hq, hkv, d = rng.choice([(32, 8, 128), (14, 2, 64), (32, 8, 64), (8, 4, 256)])
        c = _rope("", _log(rng, 1, 8192 if d < 256 else 6000), hq, hkv, d, rng.choice([d, d, d // 2]), page,
                  rng.choice(["f16", "f32"]), rng.choice(["f16", "f32"]), rng.random() < 0.75, rng.random() < 0.4,
                  rng.choice([0.0, 1.0]))
    else:
        hq, hkv, d = rng.choice([(32, 8, 128), (14, 2, 64), (32, 8, 64), (8, 4, 256)])
        kind = rng.choice(["decode", "decode", "draft", "chunk", "chunk", "mixed"])
        if kind == "decode":
            past = _log(rng, 1, 32768)
            how = (_log(rng, 1, max(2, min(128, 400000 // past))), 0, 0, past)
        elif kind == "draft":
            past = _log(rng, 16, 16384)
            how = (0, _log(rng, 1, max(2, min(64, 200000 // past))), rng.randint(2, 8), past)
        elif kind == "chunk":
            how = (0, rng.randint(1, 4), _log(rng, 16, 1500), rng.choice([0, _log(rng, 16, 6000)]))
        else:
            how = (_log(rng, 2, 24), rng.randint(1, 2), _log(rng, 16, 700), _log(rng, 64, 5000))
        c = _attn("", *how[:3], how[3], hq, hkv, d, page, rng.choice(["f16", "f16", "f32"]), rng.choice([0.0, 0.0, 50.0]),
                  rng.choice([0, 0, _log(rng, 64, 4096)]), rng.random() < 0.3)
    del c["name"]
    return c


def _lengths(case):
    """(cached, new) tokens of every request."""
    past, new = [], []
    for i in range(case["decodes"] + case["chunks"]):
        f = 1.0 if case["even"] else ((i + 1) * 40503 % 65536) / 65536.0  # multiples of the golden section: well spread
        one = i < case["decodes"]
        lo = case["past"] // 8 if one else 0
        past.append(lo + int(round(f * (case["past"] - lo))))
        new.append(1 if one else max(1, case["chunk"] - int((1.0 - f) * 0.5 * case["chunk"])))
    return past, new


# ---- inputs ------------------------------------------------------------------------------------------
_TYPES = {"f16": torch.float16, "f32": torch.float32}


def _pages(case, g, spare=0):
    """Page numbers of every request in random order, and what is left: (table, free list, pages in all)."""
    past, new = _lengths(case)
    p = case["page"]
    have = [-(-x // p) for x in past]
    want = [-(-(x + y) // p) for x, y in zip(past, new)]
    n = sum(want) + spare
    perm = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    return past, new, have, want, perm, n


def _filled(width, counts, perm):
    """[requests, width] table whose row s holds the next counts[s] entries of perm, -1 behind them."""
    cnt = torch.tensor(counts, device="cuda")
    at = (torch.cumsum(cnt, 0) - cnt)[:, None] + torch.arange(width, device="cuda")
    ok = torch.arange(width, device="cuda") < cnt[:, None]
    return torch.where(ok, perm[at.clamp(max=perm.numel() - 1)], torch.full_like(at, -1).to(torch.int32)).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    st = dict(case=case)
    if case["op"] == "page_plan":
        past, new, have, want, perm, n = _pages(case, g, spare=64)
        held = sum(have)
        tokens = sum(new) + 37  # arrays of a fixed size, a little longer than this step
        st.update(past=ints(past), new=ints(new), table=_filled(max(want) + 8, have, perm[:held]) if held else
                  torch.full((len(past), max(want) + 8), -1, dtype=torch.int32, device="cuda"),
                  free=perm[held:].contiguous(), n_pages=n, cu=torch.zeros(len(past) + 1, dtype=torch.int32, device="cuda"),
                  kv=torch.zeros(len(past), dtype=torch.int32, device="cuda"),
                  pos=torch.zeros(tokens, dtype=torch.int32, device="cuda"),
                  slots=torch.zeros(tokens, dtype=torch.int32, device="cuda"),
                  counts=torch.zeros(3, dtype=torch.int32, device="cuda"))
    elif case["op"] == "qk_norm_rope":
        t, hq, hkv, d, p = case["tokens"], case["hq"], case["hkv"], case["d"], case["page"]
        ty = _TYPES[case["dtype"]]
        qkv = randn(t, (hq + 2 * hkv) * d).to(ty)  # one projection's output, read in place
        rows = 16384
        n = -(-t // p) + 8
        half = case["rot"] // 2
        freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        ang = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * freq
        st.update(q=qkv[:, :hq * d].view(t, hq, d), k=qkv[:, hq * d:(hq + hkv) * d].view(t, hkv, d),
                  v=qkv[:, (hq + hkv) * d:].view(t, hkv, d), cos_sin=torch.cat([ang.cos(), ang.sin()], 1).float().contiguous(),
                  pos=torch.randint(0, rows, (t,), generator=g, device="cuda", dtype=torch.int32),
                  slots=torch.randperm(n * p, generator=g, device="cuda")[:t].to(torch.int32),
                  wq=1.0 - case["bias"] + 0.1 * randn(d) if case["norm"] else None,
                  wk=1.0 - case["bias"] + 0.1 * randn(d) if case["norm"] else None,
                  q_out=torch.zeros((t, hq, d), dtype=_TYPES[case["out"]], device="cuda"),
                  kc=torch.zeros((n, hkv, p, d), dtype=torch.float16, device="cuda"),
                  vc=torch.zeros((n, hkv, p, d), dtype=torch.float16, device="cuda"))
    else:
        hq, hkv, d, p = case["hq"], case["hkv"], case["d"], case["page"]
        past, new, have, want, perm, n = _pages(case, g, spare=8)
        shape = (n, p, hkv, d) if case["seq_major"] else (n, hkv, p, d)
        cu = [0]
        for x in new:
            cu.append(cu[-1] + x)
        q = 1.5 * randn(cu[-1], hq, d)
        kv = lambda: torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)  # noqa: E731
        st.update(q=q.to(_TYPES[case["dtype"]]), kc=kv(), vc=kv(), table=_filled(max(want) + 3, want, perm), cu=ints(cu),
                  kv=ints([x + y for x, y in zip(past, new)]), most_new=max(new), most_kv=max(x + y for x, y in zip(past, new)),
                  out=torch.zeros((cu[-1], hq, d), dtype=_TYPES[case["dtype"]], device="cuda"))
    return st


# ---- plain forms -------------------------------------------------------------------------------------
def _plain_page_plan(st):
    past, new, free, p = st["past"].long(), st["new"].long(), st["free"], st["case"]["page"]
    n, width = st["table"].shape
    had = ((past + p - 1) // p).clamp(max=width)
    want = ((past + new + p - 1) // p).clamp(max=width)
    need = torch.where(new > 0, (want - had).clamp(min=0), 0)
    base = torch.cumsum(need, 0) - need
    col = torch.arange(width, device="cuda")
    at = base[:, None] + col - had[:, None]
    fresh = (col >= had[:, None]) & (col < (had + need)[:, None])
    page = torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1)], -1)
    table = torch.where(fresh, page, st["table"])
    cu = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), torch.cumsum(new, 0)])
    t = torch.arange(st["pos"].numel(), device="cuda")
    s = torch.searchsorted(cu[1:], t, right=True).clamp(max=n - 1)
    pos = past[s] + t - cu[s]
    live = t < cu[-1]
    entry = table[s, (pos // p).clamp(max=width - 1)].long()
    some = live & (pos // p < width) & (entry >= 0) & (entry < st["n_pages"])
    slots = torch.where(some, entry * p + pos % p, -1)
    short = (new > 0) & ((past + new > width * p) | ((need > 0) & (base + need > free.numel())))
    counts = torch.stack([cu[-1], need.sum(), short.sum()])
    i32 = torch.int32
    return dict(table=table, cu=cu.to(i32), kv=(past + new).to(i32), pos=torch.where(live, pos, -1).to(i32), slots=slots.to(i32),
                counts=counts.to(i32))


def _plain_turn(x, w, st):
    """Norm and rotation of [tokens, heads, d] in 32 bits."""
    c = st["case"]
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (w + c["bias"])
    half = c["rot"] // 2
    cs = st["cos_sin"][st["pos"].long()]
    cos, sin = cs[:, None, :half], cs[:, None, half:]
    if c["pairs"]:
        a, b = x[..., 0:c["rot"]:2], x[..., 1:c["rot"]:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:c["rot"]]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., c["rot"]:]], -1)


def _plain_qk_norm_rope(st):
    page, off = st["slots"].long() // st["case"]["page"], st["slots"].long() % st["case"]["page"]
    q = _plain_turn(st["q"], st["wq"], st).to(st["q_out"].dtype)
    st["kc"][page, :, off] = _plain_turn(st["k"], st["wk"], st).half()
    st["vc"][page, :, off] = st["v"].half()
    return dict(q=q, k=st["kc"], v=st["vc"])


def _plain_paged_attention(st):
    c = st["case"]
    hq, hkv, d, p = c["hq"], c["hkv"], c["d"], c["page"]
    g, m, n = hq // hkv, st["most_new"], st["most_kv"]
    cu, kv = st["cu"].long(), st["kv"].long()
    s, new = kv.numel(), cu[1:] - cu[:-1]
    i, key = torch.arange(m, device="cuda"), torch.arange(n, device="cuda")
    row = (cu[:-1, None] + i).clamp(max=st["q"].shape[0] - 1)
    q = st["q"][row].float().view(s, m, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(s, hkv, g * m, d)
    page = st["table"].long()[:, key // p].clamp(min=0)
    off = (key % p).expand(s, n)

    def rows(cache):  # [s, hkv, n, d]
        x = cache[page, off] if c["seq_major"] else cache[page, :, off]
        return x.transpose(1, 2).float().contiguous()

    a = torch.matmul(q, rows(st["kc"]).transpose(2, 3).contiguous()) * d ** -0.5
    if c["softcap"] > 0:
        a = c["softcap"] * torch.tanh(a / c["softcap"])
    pos = (kv - new)[:, None] + i
    sees = (key <= pos[..., None]) & (key < kv[:, None, None])
    if c["window"] > 0:
        sees = sees & (key > pos[..., None] - c["window"])
    a = a.view(s, hkv, g, m, n).masked_fill(~sees[:, None, None], float("-inf"))
    a = torch.exp(a - a.amax(-1, keepdim=True).clamp(min=-1e30))
    a = a / a.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(a.view(s, hkv, g * m, n), rows(st["vc"])).view(s, hkv, g, m, d).permute(0, 3, 1, 2, 4).reshape(s, m, hq, d)
    t = torch.arange(st["q"].shape[0], device="cuda")
    seq = torch.searchsorted(cu[1:], t, right=True)
    return o[seq, t - cu[seq]].to(st["q"].dtype)


def run(state):
    st, c = state, state["case"]
    if not own:
        return {"page_plan": _plain_page_plan, "qk_norm_rope": _plain_qk_norm_rope, "paged_attention": _plain_paged_attention}[c["op"]](st)
    ctx = _context()
    if c["op"] == "page_plan":
        ctx.page_plan(st["past"], st["new"], st["free"], st["table"], c["page"], st["n_pages"], st["cu"], st["kv"], st["pos"], st["slots"],
                      st["counts"])
        return {k: st[k] for k in ("table", "cu", "kv", "pos", "slots", "counts")}
    if c["op"] == "qk_norm_rope":
        ctx.qk_norm_rope(st["q"], st["k"], st["v"], st["pos"], st["cos_sin"], st["q_out"], st["kc"], st["vc"], st["slots"],
                         q_weight=st["wq"], k_weight=st["wk"], eps=1e-6, weight_bias=c["bias"], interleaved=c["pairs"])
        return dict(q=st["q_out"], k=st["kc"], v=st["vc"])
    import argus_hip
    ctx.paged_attention(st["q"], st["kc"], st["vc"], st["table"], st["cu"], st["kv"], st["out"], max_new=st["most_new"],
                        max_kv=st["most_kv"], softcap=c["softcap"], window=c["window"],
                        layout=argus_hip.SEQ_MAJOR if c["seq_major"] else argus_hip.HEAD_MAJOR)
    return st["out"]


# ---- what a pass cannot do without ---------------------------------------------------------------------
def work(case):
    size = {"f16": 2, "f32": 4}
    if case["op"] == "page_plan":
        past, new = _lengths(case)
        p = case["page"]
        fresh = sum(-(-(x + y) // p) - -(-x // p) for x, y in zip(past, new))
        touched = sum((x + y - 1) // p - x // p + 1 for x, y in zip(past, new))
        tokens = sum(new) + 37
        return dict(bytes=16 * len(past) + 4 * touched + 8 * fresh + 8 * tokens + 16, flops=0)
    if case["op"] == "qk_norm_rope":
        t, d = case["tokens"], case["d"]
        e, o = size[case["dtype"]], size[case["out"]]
        heads = case["hq"] + case["hkv"]
        table = min(t, 16384) * case["rot"] * 4
        return dict(bytes=t * d * ((heads + case["hkv"]) * e + case["hq"] * o + case["hkv"] * 4) + table + 8 * t,
                    flops=t * heads * (4 * d * case["norm"] + 3 * case["rot"]))
    past, new = _lengths(case)
    hq, hkv, d, w = case["hq"], case["hkv"], case["d"], case["window"]
    keys = pairs = 0
    for x, y in zip(past, new):
        first = max(0, x - w + 1) if w else 0  # the first key that any row of the request sees
        keys += x + y - first
        if not w:
            pairs += y * x + y * (y + 1) // 2
        else:
            full = max(0, min(y, x + y - w))  # rows whose window is full
            pairs += full * w + sum(range(x + 1, x + 1 + y - full))
    tokens = sum(new)
    return dict(bytes=4 * keys * hkv * d + 2 * tokens * hq * d * size[case["dtype"]] + 4 * sum(-(-(x + y) // case["page"]) for x, y in zip(past, new)),
                flops=4 * hq * d * pairs)


# ---- the definitions in 64 bits ------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "page_plan":
        return None  # whole numbers
    if case["op"] == "qk_norm_rope":
        d, rot = case["d"], case["rot"]
        first = torch.arange(0, rot, 2, device="cuda") if case["pairs"] else torch.arange(rot // 2, device="cuda")
        second = first + (1 if case["pairs"] else rot // 2)
        row = st["cos_sin"].double()[st["pos"].long()]
        angle = torch.complex(row[:, :rot // 2], row[:, rot // 2:])[:, None]

        def turn(x, w):
            x = x.double()
            if w is not None:
                x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / d + 1e-6) * (w.double() + case["bias"])
            z = torch.complex(x[..., first], x[..., second]) * angle
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            return y

        slot = st["slots"].long()
        caches = []
        for x in (turn(st["k"], st["wk"]), st["v"].double()):
            flat = torch.zeros((st["kc"].shape[0] * case["page"], case["hkv"], d), dtype=torch.float64, device="cuda")
            flat[slot] = x
            caches.append(flat.view(-1, case["page"], case["hkv"], d).transpose(1, 2).contiguous())
        return dict(q=turn(st["q"], st["wq"]), k=caches[0], v=caches[1])
    past, new = _lengths(case)
    if work(case)["flops"] > 2e12:
        return None
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    out, at = torch.zeros((sum(new), hq, d), dtype=torch.float64, device="cuda"), 0
    for s, (x, y) in enumerate(zip(past, new)):
        pages = st["table"][s, :-(-(x + y) // case["page"])].long()
        k, v = (c[pages] if case["seq_major"] else c[pages].transpose(1, 2) for c in (st["kc"], st["vc"]))
        k, v = (c.reshape(-1, hkv, d)[:x + y] for c in (k, v))
        for h in range(hq):
            q = st["q"][at:at + y, h].double()
            logit = (q @ k[:, h * hkv // hq].double().T.contiguous()) / d ** 0.5
            if case["softcap"] > 0:
                logit = torch.tanh(logit / case["softcap"]) * case["softcap"]
            age = torch.arange(x, x + y, device="cuda")[:, None] - torch.arange(x + y, device="cuda")
            hidden = (age < 0) | (age >= case["window"]) if case["window"] > 0 else age < 0
            weight = torch.softmax(logit.masked_fill(hidden, -torch.inf), -1)
            out[at:at + y, h] = weight @ v[:, h * hkv // hq].double()
        at += y
    return out
