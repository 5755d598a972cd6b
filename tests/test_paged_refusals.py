"""Calls of the paged-cache operators that are refused because their outputs would overwrite each other or
what is still being read."""
import ctypes as C

import pytest

from test_paged_args import attention_args


@pytest.mark.parametrize("kw,code", [
    (dict(out_stride=1024), None), (dict(out_stride=2048), None), (dict(out_stride=8, n_tokens=1), None), (dict(q_stride=512), None),
    (dict(out_stride=1016), -1), (dict(out_stride=8), -1)])
def test_rows_of_out_do_not_overlap(kw, code):
    import argus_hip as A
    rc = A.lib.argus_hip_paged_attention_workspace(None, C.byref(attention_args(**kw)))
    assert rc >= 0 if code is None else rc == code


@pytest.mark.gpu
def test_overlapping_rows_are_refused_by_the_calls():
    import argus_hip as A
    import torch
    from gpu_util import ctx
    f = lambda *s: torch.zeros(s, dtype=torch.float16, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    rows = torch.as_strided(f(4096), (4, 4, 64), (128, 64, 1))
    assert ctx().paged_attention(f(4, 4, 64), f(3, 2, 16, 64), f(3, 2, 16, 64), i(2, 3), i(3), i(2), rows, check=False) == A.ERR_INVALID
    rope = lambda q, out: ctx().qk_norm_rope(q, f(4, 2, 64), f(4, 2, 64), None, None, out, f(3, 2, 16, 64), f(3, 2, 16, 64),  # noqa: E731
                                             torch.arange(4, dtype=torch.int32, device="cuda"), check=False)
    assert rope(f(4, 4, 64), rows) == A.ERR_INVALID
    assert rope(rows, f(4, 4, 64)) == A.OK  # reading a row twice is no harm


@pytest.mark.gpu
def test_queries_in_place_keep_their_type_and_stride():
    import argus_hip as A
    import torch
    from gpu_util import ctx
    f = lambda *s, ty=torch.float16: torch.zeros(s, dtype=ty, device="cuda")  # noqa: E731
    wide = f(4, 8, 64)
    same = wide.view(4, 8, 64)[:, :4]
    rope = lambda q, out, n=4: ctx().qk_norm_rope(q, f(n, 2, 64, ty=q.dtype), f(n, 2, 64, ty=q.dtype), None, None, out, f(3, 2, 16, 64),  # noqa: E731
                                                  f(3, 2, 16, 64), torch.arange(n, dtype=torch.int32, device="cuda"), check=False)
    assert rope(same, same) == A.OK
    assert rope(same, wide.view(-1)[:1024].view(4, 4, 64)) == A.ERR_INVALID
    assert rope(same, wide.view(-1)[:2048].view(torch.float32).view(4, 4, 64)) == A.ERR_INVALID
    assert rope(same[:1], wide.view(-1)[:256].view(1, 4, 64), 1) == A.OK  # one token has no stride
