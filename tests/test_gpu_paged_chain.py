"""The paged-cache operators as a server uses them: plan, norm + rotation + cache write, attention, over
several steps of requests that come, grow and go -- eagerly, and as one captured step that is replayed
with other lengths."""
import numpy as np
import pytest

import paged_util as U
from gpu_util import ctx, dev, host

pytestmark = pytest.mark.gpu


class Server:
    """Host bookkeeping of a small server: pages, lengths and, for the reference, every token's raw rows."""

    def __init__(self, n, hq, hkv, d, page, width, ty, seed, softcap=0.0, window=0):
        import torch
        self.n, self.hq, self.hkv, self.d, self.page, self.width, self.ty = n, hq, hkv, d, page, width, ty
        self.softcap, self.window = softcap, window
        self.rng = np.random.default_rng(seed)
        self.n_pages = n * width
        self.free = list(self.rng.permutation(self.n_pages))
        self.past = [0] * n
        self.rows = [(np.zeros((0, hkv, d)), np.zeros((0, hkv, d))) for _ in range(n)]
        i32 = lambda *s: torch.full(s, -1, dtype=torch.int32, device="cuda")  # noqa: E731
        self.table = i32(n, width)
        self.kc, self.vc = (torch.full((self.n_pages, hkv, page, d), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2))
        ang = self.rng.uniform(0, 6.3, (width * page, d // 2))
        self.cs = np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)
        self.wq, self.wk = ((1 + 0.2 * self.rng.standard_normal(d)).astype(np.float32) for _ in range(2))
        self.cs_d, self.wq_d, self.wk_d = dev(self.cs), dev(self.wq), dev(self.wk)

    def buffers(self, capacity):
        import torch
        i32 = lambda m: torch.zeros(m, dtype=torch.int32, device="cuda")  # noqa: E731
        ty = getattr(torch, {"f16": "float16", "f32": "float32"}[self.ty])
        return dict(past=i32(self.n), new=i32(self.n), free=i32(self.n_pages), cu=i32(self.n + 1), kv=i32(self.n), pos=i32(capacity),
                    slots=i32(capacity), counts=i32(3),
                    x=torch.zeros((capacity, self.hq + 2 * self.hkv, self.d), dtype=ty, device="cuda"),
                    q=torch.zeros((capacity, self.hq, self.d), dtype=ty, device="cuda"),
                    out=torch.zeros((capacity, self.hq, self.d), dtype=ty, device="cuda"))

    def fill(self, b, new):
        """A step's inputs into fixed buffers; returns the raw rows."""
        import torch
        t = sum(new)
        x = self.rng.standard_normal((t, self.hq + 2 * self.hkv, self.d), dtype=np.float32).astype({"f16": np.float16, "f32": np.float32}[self.ty])
        b["past"].copy_(dev(np.array(self.past, np.int32)))
        b["new"].copy_(dev(np.array(new, np.int32)))
        b["free"].fill_(-1)
        b["free"][:len(self.free)] = dev(np.array(self.free, np.int32))
        b["x"].fill_(float("nan"))
        b["x"][:t] = dev(x)
        b["out"].fill_(-9.0)
        torch.cuda.synchronize()
        return x

    def launch(self, b, workspace=None, **hints):
        c, hq, hkv = ctx(), self.hq, self.hkv
        c.page_plan(b["past"], b["new"], b["free"], self.table, self.page, self.n_pages, b["cu"], b["kv"], b["pos"], b["slots"], b["counts"])
        c.qk_norm_rope(b["x"][:, :hq], b["x"][:, hq:hq + hkv], b["x"][:, hq + hkv:], b["pos"], self.cs_d, b["q"], self.kc, self.vc, b["slots"],
                       q_weight=self.wq_d, k_weight=self.wk_d)
        c.paged_attention(b["q"], self.kc, self.vc, self.table, b["cu"], b["kv"], b["out"], softcap=self.softcap, window=self.window,
                          workspace=workspace, **hints)

    def check(self, b, new, x):
        """The step's output against the references; then the host's books."""
        dt = x.dtype.type
        q, out, at = host(b["q"]), host(b["out"]), 0
        counts = host(b["counts"])
        assert counts.tolist()[0] == sum(new) and counts[2] == 0
        self.free = self.free[counts[1]:]
        for s, m in enumerate(new):
            r = x[at:at + m]
            pos = np.arange(self.past[s], self.past[s] + m)
            qr, qtol = U.norm_rope(r[:, :self.hq], self.wq, 0.0, 1e-6, self.cs, pos, False, dt)
            kr, _ = U.norm_rope(r[:, self.hq:self.hq + self.hkv], self.wk, 0.0, 1e-6, self.cs, pos, False, np.float16)
            if m:
                U.within(q[at:at + m], qr, qtol, "queries of request %d" % s)
            # what the cache holds is taken from the cache: its own error is checked above
            have = self.past[s] + m
            pages = host(self.table)[s, :U.ceil_div(have, self.page)]
            k, v = (host(c)[pages].transpose(0, 2, 1, 3).reshape(-1, self.hkv, self.d)[:have] for c in (self.kc, self.vc))
            assert np.array_equal(k[:self.past[s]], self.rows[s][0]), "cached keys of request %d changed" % s
            assert np.abs(k[self.past[s]:].astype(np.float64) - kr).max(initial=0) < 0.02
            assert np.array_equal(v[self.past[s]:], r[:, self.hq + self.hkv:].astype(np.float16))
            if m:
                ref, tol = U.attention(q[at:at + m], (k, v), have, m, self.softcap, self.window, dtype=dt)
                U.within(out[at:at + m], ref, tol, "request %d: %d new of %d" % (s, m, have))
            self.rows[s] = (k, v)
            self.past[s] = have
            at += m
        assert (out[at:] == -9.0).all()

    def end(self, s):
        """The request leaves and its pages are free again."""
        import torch
        n = U.ceil_div(self.past[s], self.page)
        self.free += list(host(self.table)[s, :n])
        self.table[s].fill_(-1)
        self.past[s], self.rows[s] = 0, (np.zeros((0, self.hkv, self.d)), np.zeros((0, self.hkv, self.d)))
        torch.cuda.synchronize()


STEPS = [[5, 40, 0, 1], [1, 1, 33, 1], [1, 1, 1, 70], [4, 1, 0, 1], [1, 1, 1, 1]]


@pytest.mark.parametrize("ty,hq,hkv,d,page,softcap,window", [
    ("f16", 8, 2, 128, 16, 0.0, 0), ("f32", 14, 2, 64, 32, 0.0, 0), ("f16", 4, 2, 256, 16, 50.0, 40), ("f32", 8, 8, 64, 16, 0.0, 17)])
def test_steps_of_a_server(ty, hq, hkv, d, page, softcap, window):
    sv = Server(4, hq, hkv, d, page, 160 // page, ty, 1, softcap, window)
    b = sv.buffers(90)
    for i, new in enumerate(STEPS):
        x = sv.fill(b, new)
        sv.launch(b, max_new=max(new))
        sv.check(b, new, x)
        if i == 2:
            sv.end(1)
            sv.end(3)


@pytest.mark.parametrize("ty", ["f16", "f32"])
def test_a_captured_step_is_replayed_with_other_requests(ty):
    """One graph of the three calls over buffers of fixed size; every replay has other lengths, and equals
    an eager run of the same step bit for bit.  Two graphs live at once, each with its own workspace."""
    import torch
    sv = Server(4, 8, 2, 128, 16, 70, ty, 2)
    graphs = []
    side = torch.cuda.Stream()
    for capacity in (8, 700):
        b = sv.buffers(capacity)
        hints = dict(max_new=1 if capacity == 8 else 0)
        args = (b["q"], sv.kc, sv.vc, sv.table, b["cu"], b["kv"], b["out"])
        need = ctx().paged_attention_workspace(*args, **hints)
        assert need > 0
        ws = torch.full((need,), 0x7f, dtype=torch.uint8, device="cuda")
        side.wait_stream(torch.cuda.current_stream())
        sv.fill(b, [0, 0, 0, 0])
        with torch.cuda.stream(side):
            sv.launch(b, ws, **hints)  # kernels are loaded outside the capture
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            sv.launch(b, ws, **hints)
        graphs.append((g, b, ws, hints))
    # a captured call without a workspace of its own is refused, and the capture goes on
    b = graphs[1][1]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        b["q"].mul_(1.0)
        rc = ctx().paged_attention(b["q"], sv.kc, sv.vc, sv.table, b["cu"], b["kv"], b["out"], check=False)
    assert rc == -1 and "workspace" in ctx().last_error()
    for i, new in enumerate([[600, 3, 0, 90], [1, 1, 0, 1], [1, 300, 20, 1], [1, 1, 1, 1], [0, 1, 2, 1], [1, 1, 1, 1]]):
        small = max(new) == 1
        g, b, ws, hints = graphs[0 if small else 1]
        x = sv.fill(b, new)
        g.replay()
        torch.cuda.synchronize()
        got = b["out"].clone()
        b["out"].fill_(-9.0)
        sv.launch(b, None, **hints)  # the program's own eager work, on the context's workspace
        torch.cuda.synchronize()
        assert torch.equal(got, b["out"]), "step %d" % i
        b["out"].fill_(-9.0)
        ws.fill_(0xff)  # nothing is kept in the workspace from call to call
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, b["out"]), "second replay of step %d" % i
        sv.check(b, new, x)


def test_a_workspace_that_is_too_small_or_misaligned_is_refused():
    import argus_hip as A
    import torch
    sv = Server(2, 8, 2, 128, 16, 100, "f16", 3)
    b = sv.buffers(16)
    sv.fill(b, [0, 0])
    args = (b["q"], sv.kc, sv.vc, sv.table, b["cu"], b["kv"], b["out"])
    need = ctx().paged_attention_workspace(*args)
    ws = torch.zeros(need + 256, dtype=torch.uint8, device="cuda")
    assert ctx().paged_attention(*args, workspace=ws[:need - 1], check=False) == A.ERR_NOMEM
    assert ctx().paged_attention(*args, workspace=ws[1:need + 1], check=False) == A.ERR_INVALID
    assert ctx().paged_attention(*args, workspace=ws[:need], check=False) == A.OK


def test_pages_that_ran_out():
    """A request without a page for its token: the plan says so, the write skips it, nobody else is touched."""
    import torch
    sv = Server(3, 8, 2, 128, 16, 8, "f16", 4)
    b = sv.buffers(60)
    x = sv.fill(b, [16, 20, 5])
    sv.launch(b)
    sv.check(b, [16, 20, 5], x)
    sv.free = []  # request 0 needs a page now, the others do not
    before = host(sv.kc).copy()
    sv.fill(b, [1, 1, 1])
    sv.launch(b)
    assert host(b["counts"]).tolist() == [3, 1, 1] and host(b["slots"])[0] == -1 and (host(b["slots"])[1:3] >= 0).all()
    after = host(sv.kc)
    changed = np.flatnonzero((before.view(np.uint16) != after.view(np.uint16)).reshape(len(before), -1).any(1))
    table = host(sv.table)
    assert sorted(changed) == sorted([table[1, 1], table[2, 0]])
    torch.cuda.synchronize()
