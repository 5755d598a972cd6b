"""CPU checks of the paged-cache entry points: argument structs, refusals that need no device, and the
loop references the GPU tests compare with."""
import ctypes as C
import os
import re

import numpy as np
import pytest

import paged_util as U

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_header_field_order():
    import argus_hip as A
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "argus_hip.h")).read(), flags=re.S)
    for cname, cls in (("argus_hip_page_plan_args", A.PagePlanArgs), ("argus_hip_qk_norm_rope_args", A.QkNormRopeArgs),
                       ("argus_hip_paged_attention_args", A.PagedAttentionArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), text, re.S).group(1)
        kinds = {"int32_t": C.c_int32, "int64_t": C.c_int64, "float": C.c_float, "size_t": C.c_size_t}
        fields = []
        for decl in filter(None, (x.strip() for x in body.split(";"))):
            ty, names = re.match(r"((?:const )?\w+ ?\*?)\s*(.*)", decl, re.S).groups()
            fields += [(n.strip().lstrip("*"), C.c_void_p if "*" in decl else kinds[ty.strip()]) for n in names.split(",")]
        assert fields == list(cls._fields_), cname


def attention_args(**kw):
    import argus_hip as A
    a = dict(n_seqs=4, n_tokens=9, heads_q=8, heads_kv=2, head_dim=128, n_pages=100, page_size=16, table_stride=20, layout=0, dtype=A.F16)
    a.update(kw)
    return A.PagedAttentionArgs(**a)


@pytest.mark.parametrize("kw,code", [
    (dict(), None), (dict(n_seqs=0, n_tokens=0), None), (dict(dtype=0), None), (dict(layout=1), None), (dict(heads_q=24, heads_kv=1), None),
    (dict(n_seqs=-1), -1), (dict(n_tokens=-1), -1), (dict(heads_kv=3), -1), (dict(heads_q=0), -1), (dict(n_pages=0), -1),
    (dict(table_stride=0), -1), (dict(layout=2), -1), (dict(window=-1), -1), (dict(softcap=float("inf")), -1), (dict(scale=float("nan")), -1),
    (dict(min_new=-1), -1), (dict(max_kv=-1), -1), (dict(q_stride=1028), -1), (dict(out_stride=-8), -1),
    (dict(softcap=1e-40), -1), (dict(n_tokens=2 ** 30, heads_q=8, heads_kv=2), -2), (dict(head_dim=96), -2), (dict(page_size=15), -2), (dict(page_size=2048), -2), (dict(dtype=2), -2)])
def test_paged_attention_checks_its_arguments_without_a_device(kw, code):
    # the workspace query makes the checks of the call; without a context it assumes 256 compute units
    import argus_hip as A
    rc = A.lib.argus_hip_paged_attention_workspace(None, C.byref(attention_args(**kw)))
    assert rc >= 0 if code is None else rc == code


def test_null_contexts_and_arguments():
    import argus_hip as A
    for name in ("page_plan", "qk_norm_rope", "paged_attention"):
        assert getattr(A.lib, "argus_hip_" + name)(None, None) == A.ERR_INVALID
    assert A.lib.argus_hip_paged_attention_workspace(None, None) == A.ERR_INVALID


def test_tensors_in_host_memory_are_refused():
    import argus_hip as A
    import torch
    c = A.Context.__new__(A.Context)  # no device needed: the refusal comes before the library
    c.handle, c.device = None, 0
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    f = lambda *s: torch.zeros(s, dtype=torch.float16)  # noqa: E731
    with pytest.raises(ValueError):
        c.page_plan(i(2), i(2), i(4), i(2, 3), 16, 64, i(3), i(2), i(6), i(6), i(3))
    with pytest.raises(ValueError):
        c.qk_norm_rope(f(2, 4, 64), f(2, 2, 64), f(2, 2, 64), i(2), torch.zeros(5, 64), f(2, 4, 64), f(3, 2, 16, 64), f(3, 2, 16, 64), i(2))
    with pytest.raises(ValueError):
        c.paged_attention(f(2, 4, 64), f(3, 2, 16, 64), f(3, 2, 16, 64), i(2, 3), i(3), i(2), f(2, 4, 64))


def test_rows_shared_by_tokens_are_refused():
    import argus_hip as A
    import torch
    c = A.Context.__new__(A.Context)
    c.handle, c.device = None, -1  # host tensors pass for the context's: the refusal comes before the library
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    f = lambda *s: torch.zeros(s, dtype=torch.float16)  # noqa: E731
    one = f(1, 4, 64).expand(2, 4, 64)
    with pytest.raises(ValueError, match="share"):
        c.paged_attention(one, f(3, 2, 16, 64), f(3, 2, 16, 64), i(2, 3), i(3), i(2), f(2, 4, 64))
    with pytest.raises(ValueError, match="share"):
        c.qk_norm_rope(one, f(2, 2, 64), f(2, 2, 64), i(2), torch.zeros(5, 64), f(2, 4, 64), f(3, 2, 16, 64), f(3, 2, 16, 64), i(2))


# ---- the references --------------------------------------------------------------------------------

def test_reference_plan_on_a_step_done_by_hand():
    # pages of 16: request 0 has 20 tokens (2 pages) and brings 1; request 1 is new and brings 33 (3 pages);
    # request 2 is idle; request 3 has 32 (2 pages, full) and brings 2 (1 page).  Four pages are free, 0 is one.
    t = [[5, 6, -1], [-1, -1, -1], [7, -1, -1], [8, 9, -1]]
    r = U.plan([20, 0, 3, 32], [1, 33, 0, 2], [3, 0, 2, 1], t, 16, 10, 38)
    assert r["table"].tolist() == [[5, 6, -1], [3, 0, 2], [7, -1, -1], [8, 9, 1]]
    assert r["cu"].tolist() == [0, 1, 34, 34, 36] and r["kv"].tolist() == [21, 33, 3, 34]
    assert r["pos"].tolist() == [20] + list(range(33)) + [32, 33, -1, -1]
    assert r["slots"].tolist() == [6 * 16 + 4] + list(range(48, 64)) + list(range(16)) + [32] + [16, 17] + [-1, -1]
    assert r["counts"].tolist() == [36, 4, 0]
    r = U.plan([20, 0, 3, 32], [1, 33, 0, 2], [3, 0], t, 16, 10, 36)  # two pages short
    assert r["counts"].tolist() == [36, 4, 2] and r["slots"][33] == -1 and (r["slots"][34:] == -1).all()


def test_reference_rotation_turns_a_pair_by_its_angle():
    x = np.zeros((1, 1, 8))
    x[0, 0, 1] = 2.0
    ang = np.array([[0.3, 0.7, 1.1, 2.0]])
    cs = np.concatenate([np.cos(ang), np.sin(ang)], 1)
    y, _ = U.norm_rope(x, None, 0.0, 0.0, cs, np.array([0]), False, np.float32)
    assert np.allclose(y[0, 0, [1, 5]], [2 * np.cos(0.7), 2 * np.sin(0.7)]) and np.count_nonzero(y) == 2
    y, _ = U.norm_rope(x, None, 0.0, 0.0, cs, np.array([0]), True, np.float32)  # second of the first pair
    assert np.allclose(y[0, 0, :2], [-2 * np.sin(0.3), 2 * np.cos(0.3)]) and np.count_nonzero(y) == 2
    x = np.arange(1.0, 9.0).reshape(1, 1, 8)
    y, _ = U.norm_rope(x, np.ones(8), 1.0, 0.0, None, None, False, np.float32)
    assert np.allclose((y * y).mean(), 4.0)  # weight 1 + bias 1


def test_reference_attention_against_closed_forms():
    rng = np.random.default_rng(0)
    k, v = np.zeros((9, 1, 64)), rng.standard_normal((9, 1, 64))
    out, _ = U.attention(np.ones((3, 2, 64)), (k, v), 9, 3)  # equal logits: the mean of what is seen
    for i in range(3):
        assert np.allclose(out[i, 0], v[:7 + i, 0].mean(0)) and np.allclose(out[i, 1], out[i, 0])
    out, _ = U.attention(np.ones((3, 2, 64)), (k, v), 9, 3, window=1)
    assert np.allclose(out[:, 0], v[6:, 0])
    out, _ = U.attention(np.ones((3, 2, 64)), (k[:2], v[:2]), 2, 3)  # the first row stands before position 0
    assert (out[0] == 0).all() and np.allclose(out[1, 0], v[0, 0])


def test_the_tolerance_notices_a_wrong_reference():
    rng = np.random.default_rng(1)
    k, v = rng.standard_normal((40, 1, 64)).astype(np.float16), rng.standard_normal((40, 1, 64)).astype(np.float16)
    q = rng.standard_normal((2, 1, 64)).astype(np.float16)
    out, tol = U.attention(q, (k, v), 40, 2)
    wrong, _ = U.attention(q, (k[:39], v[:39]), 39, 2)  # one key late
    with pytest.raises(AssertionError):
        U.within(wrong, out, tol)
    with pytest.raises(AssertionError):
        U.within(out * (1 + 2.0 ** -7), out, tol)
