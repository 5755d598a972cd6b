"""page_plan on the GPU against a loop over requests and tokens: all results are whole numbers and have
to be equal."""
import numpy as np
import pytest

import paged_util as U
from gpu_util import ctx, dev, host

pytestmark = pytest.mark.gpu


def run(past, new, free, table, page, n_pages, capacity, twice=True):
    import torch
    n = len(past)
    t = dict(past=dev(np.array(past, np.int32)), new=dev(np.array(new, np.int32)), free=dev(np.array(free, np.int32)),
             table=dev(np.array(table, np.int32)))
    out = {k: torch.full((m,), -77, dtype=torch.int32, device="cuda")
           for k, m in (("cu", n + 1), ("kv", n), ("pos", capacity), ("slots", capacity), ("counts", 3))}
    for _ in range(2 if twice else 1):  # the same call again gives the same tables
        rc = ctx().page_plan(t["past"], t["new"], t["free"], t["table"], page, n_pages, out["cu"], out["kv"], out["pos"], out["slots"],
                             out["counts"])
        assert rc == 0
        got = {k: host(v) for k, v in out.items()}
        got["table"] = host(t["table"])
        ref = U.plan(past, new, free, table, page, n_pages, capacity)
        for k in ref:
            assert np.array_equal(got[k], ref[k]), (k, got[k][:20], ref[k][:20])


def case(rng, n, page, width, most_past, most_new, idle=0.2):
    past = rng.integers(0, most_past + 1, n)
    new = np.where(rng.random(n) < idle, 0, rng.integers(1, most_new + 1, n))
    have = [min(U.ceil_div(int(x), page), width) for x in past]
    need = sum(U.ceil_div(int(x + y), page) - U.ceil_div(int(x), page) for x, y in zip(past, new))
    n_pages = sum(have) + need + 5
    order = rng.permutation(n_pages)
    table = np.full((n, width), -1, np.int32)
    at = 0
    for s, h in enumerate(have):
        table[s, :h] = order[at:at + h]
        at += h
    return past, new, order[at:], table, n_pages


@pytest.mark.parametrize("n,page,width,most_past,most_new", [
    (1, 16, 4, 0, 1), (1, 16, 70, 1000, 100), (3, 16, 40, 500, 33), (64, 16, 260, 4000, 1), (65, 32, 40, 1000, 200),
    (511, 64, 20, 1000, 5), (2048, 16, 30, 300, 2), (2049, 128, 8, 900, 3), (5000, 1024, 3, 2000, 4)])
def test_against_loops(n, page, width, most_past, most_new):
    rng = np.random.default_rng(n * page)
    past, new, free, table, n_pages = case(rng, n, page, width, most_past, most_new)
    run(past, new, free, table, page, n_pages, int(new.sum()) + 13)


def test_most_requests_a_call_takes():
    rng = np.random.default_rng(4)
    past, new, free, table, n_pages = case(rng, 16384, 16, 3, 30, 2)
    run(past, new, free, table, 16, n_pages, int(new.sum()))


@pytest.mark.parametrize("seed", range(4))
def test_short_of_pages_of_table_or_of_rows(seed):
    rng = np.random.default_rng(seed)
    past, new, free, table, n_pages = case(rng, 37, 16, 9, 200, 60)  # some past + new exceed 9 pages of 16
    run(past, new, free[:11], table, 16, n_pages, int(new.sum()) + 5)
    run(past, new, free[:0], table, 16, n_pages, int(new.sum()))
    run(past, new, free, table, 16, n_pages, int(new.sum()) // 2)  # fewer rows than tokens
    run(past, new, free, table, 16, n_pages, 0)


def test_numbers_outside_the_pool_and_negative_lengths():
    rng = np.random.default_rng(9)
    past, new, free, table, n_pages = case(rng, 20, 32, 12, 200, 100)
    free = np.array(free)
    free[1::3] = [n_pages + 1, -5, 1 << 30][0]
    table[::4, 0] = n_pages + 7
    past, new = np.array(past), np.array(new)
    past[3], new[5] = -4, -1
    run(past, new, free, table, 32, n_pages, int(np.maximum(new, 0).sum()) + 3)


def test_no_requests_and_all_idle():
    run([], [], [1, 2, 3], np.zeros((0, 4), np.int32), 16, 8, 5)
    run([17, 0, 3], [0, 0, 0], [1, 2], np.full((3, 4), 6, np.int32), 16, 8, 7)


def test_lengths_whose_sum_passes_31_bits():
    # sums saturate; the tokens that have a row are those of the first request
    big = 2 ** 31 - 1
    import torch
    past, new = np.array([0, big, 5], np.int32), np.array([40, big, 3], np.int32)
    table = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    i32 = lambda *s: torch.full(s, -77, dtype=torch.int32, device="cuda")  # noqa: E731
    cu, kv, pos, slots, counts = i32(4), i32(3), i32(40), i32(40), i32(3)
    ctx().page_plan(dev(past), dev(new), dev(np.arange(8, dtype=np.int32)), table, 16, 8, cu, kv, pos, slots, counts)
    assert host(cu).tolist() == [0, 40, big, big] and host(kv).tolist() == [40, big, 8]
    assert host(pos).tolist() == list(range(40)) and host(slots).tolist() == list(range(40))
    assert host(counts)[0] == big and host(counts)[2] == 1  # the second request: past its table
    assert host(table)[0].tolist() == [0, 1, 2, -1]


def test_refusals():
    import argus_hip as A
    import torch
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731

    def call(page=16, n_pages=64, table=None, n=2, check=False):
        return ctx().page_plan(z(n), z(n), z(4), z(n, 3) if table is None else table, page, n_pages, z(n + 1), z(n), z(6), z(6), z(3), check=check)

    assert call() == A.OK
    assert call(page=24) == A.ERR_UNSUPPORTED and call(page=8) == A.ERR_UNSUPPORTED and call(page=2048) == A.ERR_UNSUPPORTED
    assert call(n_pages=0) == A.ERR_INVALID and call(n_pages=1 << 27) == A.ERR_INVALID
    assert call(n=16385) == A.ERR_UNSUPPORTED and "16384" in ctx().last_error()
    assert call(table=z(2, 0)) == A.ERR_INVALID
    past = z(2)
    assert ctx().page_plan(past, z(2), z(4), z(2, 3), 16, 64, z(3), past, z(6), z(6), z(3), check=False) == A.ERR_INVALID
    whole = z(4)
    assert ctx().page_plan(z(2), whole[2:], z(4), z(2, 3), 16, 64, whole[:3], z(2), z(6), z(6), z(3), check=False) == A.ERR_INVALID
    with pytest.raises(ValueError):
        call(table=z(3, 3))
    with pytest.raises(TypeError):
        ctx().page_plan(z(2).long(), z(2), z(4), z(2, 3), 16, 64, z(3), z(2), z(6), z(6), z(3))
