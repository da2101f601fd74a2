"""Eviction by attention mass against the definition written with Python lists. Everything is exact: rows, counts, masses and
the moved values are compared bit for bit."""

from __future__ import annotations

import math

import pytest
import torch

from kv_skill_v2_b200 import _native as N
from kv_skill_v2_b200 import ops

pytestmark = pytest.mark.gpu


def reference(table, valid, mass, keep, *, chunks=None, per_library=False, floor=1, M=None):
    """(new n_valid, kept rows per page) from lists."""
    P, rows_of = len(mass), len(mass[0])
    M = rows_of if M is None else M
    chunks = chunks or [len(t) for t in table]
    live = [[(c, p, min(n, rows_of)) for c, (p, n) in enumerate(zip(t, v))][:k] for t, v, k in zip(table, valid, chunks)]
    live = [[(c, p, n) for c, p, n in e if 0 <= p < P] for e in live]
    rows = [max([0] + [n for e in live for _, q, n in e if q == p]) for p in range(P)]
    weight = lambda p, i: -math.inf if math.isnan(mass[p][i]) else mass[p][i]  # noqa: E731
    nan_last = lambda p, i: math.isnan(mass[p][i])  # noqa: E731
    ranked = [sorted(range(rows[p]), key=lambda i: (nan_last(p, i), -weight(p, i) if weight(p, i) != -math.inf else math.inf, i))
              for p in range(P)]
    if per_library:
        stays = [set(r[: min(floor, M)]) for r in ranked]
        first = [set(s) for s in stays]
        for lib, e in enumerate(live):
            left = keep[lib] - sum(sum(i < n for i in first[p]) for _, p, n in e)
            others = sorted((nan_last(p, i), -weight(p, i) if weight(p, i) != -math.inf else math.inf, c, i, p)
                            for c, p, n in e for i in ranked[p][floor:M] if i < n)
            for *_, i, p in others[: max(0, left)]:
                stays[p].add(i)
    else:
        most = [max([0] + [keep[lib][c] for lib, e in enumerate(live) for c, q, _ in e if q == p]) for p in range(P)]
        stays = [set(ranked[p][: min(M, max(floor, most[p]))]) for p in range(P)]
    counts = [[0] * len(t) for t in table]
    for lib, e in enumerate(live):
        for c, p, n in e:
            counts[lib][c] = sum(i < n for i in stays[p])
    return counts, [sorted(s) for s in stays], rows


def case(seed, n_lib, C, P, rows, d, dtypes, ragged=True, zeros=0.3, bad=False):
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(P, generator=g)[: n_lib * C].view(n_lib, C)
    order[:, 0] = order[0, 0]
    page_of = order.to(torch.int32)
    n_valid = torch.full((n_lib, C), rows, dtype=torch.int32)
    if ragged:
        n_valid = torch.randint(1, rows + 1, (n_lib, C), generator=g, dtype=torch.int32)
    mass = torch.randint(0, 9, (P, rows), generator=g).float() / 8  # many ties
    mass[torch.rand(P, rows, generator=g) < zeros] = 0.0
    mass[0, 0], mass[-1, -1] = -0.0, -1.5
    if bad:
        page_of[-1, -1] = P + 3
    pools = [torch.randn(P, rows, d, generator=g).to(t).cuda() for t in dtypes]
    return pools, page_of.cuda(), n_valid.cuda(), mass.cuda()


def check(pools, page_of, n_valid, mass, keep, klist, *, M=None, nco=None, per_library=False, floor=1):
    before = [p.clone() for p in pools]
    chunks = None if nco is None else nco.tolist()
    counts, stays, rows = reference(page_of.tolist(), n_valid.tolist(), mass.tolist(), klist, chunks=chunks,
                                    per_library=per_library, floor=floor, M=M)
    nv, new_mass, kept, out = ops.pages_evict(pools, page_of, n_valid, mass, keep, n_chunks_of=nco,
                                              per_library=per_library, floor=floor, page_rows=M)
    P, R = mass.shape
    m = R if M is None else M
    assert nv.tolist() == counts
    want_kept = [s + [-1] * (m - len(s)) for s in stays]
    assert kept.tolist() == want_kept
    idx = kept.clamp(min=0).long()
    want_mass = torch.where(kept >= 0, mass.gather(1, idx), 0.0)
    assert torch.equal(new_mass.view(torch.int32), want_mass.view(torch.int32))  # (the bits: a NaN may stay)
    for b, o, p in zip(before, out, pools):
        want = torch.zeros(P, m, b.shape[2], dtype=b.dtype, device="cuda") if M is not None else b.clone()
        for q, s in enumerate(stays):
            if M is None:
                want[q, : rows[q]] = 0
            want[q, : len(s)] = b[q, s]
        assert torch.equal(o, want)
        assert (o.data_ptr() == p.data_ptr()) == (M is None)
        if M is not None:
            assert torch.equal(p, b)
    return nv


F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
SHAPES = [(1, 1, 1, 1, 8, [F16]), (2, 3, 9, 17, 24, [F16, F16]), (4, 6, 40, 64, 256, [F16, F16, F16]),
          (3, 5, 15, 200, 136, [BF16, F32]), (2, 4, 12, 33, 7, [F16, F32]), (1, 7, 9, 513, 40, [F16]),
          (5, 2, 30, 31, 1, [BF16])]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("new", [None, 0.3, 1.0])
def test_budget_per_chunk(shape, new):
    n_lib, C, P, rows, d, dtypes = shape
    for i, k in enumerate((1, max(1, rows // 4), rows)):
        a = case(i, *shape)
        M = None if new is None else max(1, int(new * rows))
        check(*a, k, [[k] * C] * n_lib, M=M)
    keep = torch.randint(0, rows + 2, (n_lib, C), generator=torch.Generator().manual_seed(9), dtype=torch.int32)
    check(*case(7, *shape), keep.cuda(), keep.tolist(), M=None if new is None else max(1, int(new * rows)), floor=2)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("new", [None, 0.5])
@pytest.mark.parametrize("floor", [0, 1, 3])
def test_budget_per_library(shape, new, floor):
    n_lib, C, P, rows, d, dtypes = shape
    for i, k in enumerate((0, C, max(1, rows * C // 3), rows * C, 2**31 - 1)):
        a = case(10 + i, *shape, ragged=i % 2 == 0)
        check(*a, k, [k] * n_lib, M=None if new is None else max(1, int(new * rows)), per_library=True, floor=floor)
    keep = torch.randint(0, rows * C + 1, (n_lib,), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    check(*case(21, *shape), keep.cuda(), keep.tolist(), per_library=True, floor=floor)


@pytest.mark.parametrize("per_library", [False, True])
def test_ragged_tables_long_pages_and_odd_masses(per_library):
    # chunk counts per Library, a page of 4096 rows (the most), NaN, infinities, equal masses everywhere
    pools, page_of, n_valid, mass = case(30, 2, 3, 6, 4096, 8, [F16])
    mass[:, 5], mass[:, 9], mass[:, 11], mass[:, 13] = math.nan, math.inf, -math.inf, -math.nan
    mass[2] = 0.25
    nco = torch.tensor([3, 2], dtype=torch.int32, device="cuda")
    k = 700 if not per_library else 1900
    check(pools, page_of, n_valid, mass, k, [k] * 2 if per_library else [[k] * 3] * 2, nco=nco, M=1000,
          per_library=per_library)


def test_many_chunks_of_one_library():
    # more positions than one round of the CTA takes, in every pass; ties that run over many chunks
    for seed in range(3):
        a = case(40 + seed, 1, 150, 150, 96, 8, [F16], zeros=0.9)
        check(*a, 2000 + 777 * seed, [2000 + 777 * seed], per_library=True, M=60)


@pytest.mark.parametrize("per_library", [False, True])
def test_long_tables(per_library):
    # too long for every page's CTA to look through, and too many rows of a Library for shared memory
    a = case(45, 4, 300, 1250, 200, 8, [F16])
    k = 9000 if per_library else 37
    check(*a, k, [k] * 4 if per_library else [[k] * 300] * 4, per_library=per_library, M=90)


def test_a_chunk_without_rows_and_a_page_outside_the_pool():
    pools, page_of, n_valid, mass = case(50, 2, 4, 12, 20, 16, [F16])
    n_valid[1, 2] = 0
    check(pools, page_of, n_valid, mass, 5, [[5] * 4] * 2, M=8)
    pools, page_of, n_valid, mass = case(51, 2, 4, 12, 20, 16, [F16], bad=True)
    ops.device_status(torch.device("cuda:0"))
    nv = check(pools, page_of, n_valid, mass, 5, [[5] * 4] * 2, M=8)
    assert int(nv[-1, -1]) == 0 and ops.device_status(torch.device("cuda:0")) & N.DEV_BADPAGE
    nv = check(pools, page_of, n_valid, mass, 30, [30] * 2, M=8, per_library=True)
    assert int(nv[-1, -1]) == 0 and ops.device_status(torch.device("cuda:0")) & N.DEV_BADPAGE
    n_valid[0, 1] = 25  # more than the page holds
    check(pools, page_of, n_valid, mass, 5, [[5] * 4] * 2)
    assert ops.device_status(torch.device("cuda:0")) & N.DEV_CLAMPED


def test_captured_and_repeated():
    pools, page_of, n_valid, mass = case(60, 4, 6, 40, 64, 256, [F16, F16])
    want = ops.pages_evict(pools, page_of, n_valid, mass, 100, per_library=True, page_rows=40)
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros_like(mass)
    with torch.cuda.graph(graph):
        got = ops.pages_evict(pools, page_of, n_valid, x, 100, per_library=True, page_rows=40)
    x.copy_(mass)
    for _ in range(3):
        graph.replay()
        for a, b in zip([*want[:3], *want[3]], [*got[:3], *got[3]]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("per_library", [False, True])
def test_one_library_one_page_twice_and_keeps_below_zero(per_library):
    a = case(80, 1, 6, 7, 40, 24, [F16, F16])
    a[1][0, 3] = a[1][0, 1]
    k = 50 if per_library else 9
    check(*a, k, [k] if per_library else [[k] * 6], per_library=per_library, M=30)
    keep = torch.tensor([-3] if per_library else [[-1, 0, 5, -7, 40, 41]], dtype=torch.int32)
    check(*a, keep.cuda(), keep.tolist(), per_library=per_library, floor=0)
    check(*a, keep.cuda(), keep.tolist(), per_library=per_library, floor=40, M=12)


@pytest.mark.parametrize("per_library", [False, True])
def test_the_least_keep_there_is(per_library):
    # a budget below zero is one of nothing, also where the floor's rows would take it below what 32 bits hold
    a = case(86, 3, 4, 12, 40, 24, [F16])
    least = -2**31
    keep = torch.full((3,) if per_library else (3, 4), least, dtype=torch.int32)
    keep[1] = least + 3
    for floor in (0, 2):
        check(*a, keep.cuda(), keep.tolist(), per_library=per_library, floor=floor, M=30)


def test_more_pools_than_one_launch_moves():
    dtypes = [F16, BF16, F32] * 25
    check(*case(81, 2, 3, 8, 20, 16, dtypes), 7, [[7] * 3] * 2, M=9)
    check(*case(82, 2, 3, 8, 20, 16, dtypes), 7, [[7] * 3] * 2)


def test_two_streams_at_once():
    a, b = case(83, 4, 6, 40, 64, 256, [F16, F16]), case(84, 2, 30, 70, 128, 64, [F16])
    run = [lambda x=x, k=k: ops.pages_evict(*x, k, per_library=True, page_rows=40) for x, k in ((a, 100), (b, 700))]
    want = [r() for r in run]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for s, r in zip(streams, run):
            with torch.cuda.stream(s):
                got.append(r())
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            for x, y in zip([*w[:3], *w[3]], [*g[:3], *g[3]]):
                assert torch.equal(x, y)


def test_refusals():
    pools, page_of, n_valid, mass = case(70, 2, 3, 9, 16, 8, [F16])
    with pytest.raises(ValueError, match="mass"):
        ops.pages_evict(pools, page_of, n_valid, mass.half(), 3)
    with pytest.raises(ValueError, match="mass"):
        ops.pages_evict(pools, page_of, n_valid, mass[:, :8].contiguous(), 3)
    with pytest.raises(ValueError, match="keep"):
        ops.pages_evict(pools, page_of, n_valid, mass, torch.ones(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="keep"):
        ops.pages_evict(pools, page_of, n_valid, mass, torch.ones(2, 3, dtype=torch.int32, device="cuda"), per_library=True)
    with pytest.raises(ValueError, match="page_rows"):
        ops.pages_evict(pools, page_of, n_valid, mass, 3, page_rows=17)
    with pytest.raises(ValueError, match="page_rows"):
        ops.pages_evict(pools, page_of, n_valid, mass, 3, page_rows=0)
    with pytest.raises(ValueError, match="floor"):
        ops.pages_evict(pools, page_of, n_valid, mass, 3, floor=-1)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.pages_evict(pools, page_of, n_valid, mass.cpu(), 3)
    with pytest.raises(ValueError, match="overlaps"):  # in place the same pool twice would move twice
        ops.pages_evict([*pools, pools[0]], page_of, n_valid, mass, 3)
    big = torch.zeros(1, 4100, 8, dtype=F16, device="cuda")
    one = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    with pytest.raises(NotImplementedError, match="4096"):
        ops.pages_evict([big], one, one + 1, torch.zeros(1, 4100, device="cuda"), 3)
