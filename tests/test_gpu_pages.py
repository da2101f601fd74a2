"""Page operators: forks that share pages, compaction, against a host restatement (copies are exact)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def _state(dev, seed, n_lib, C, P, rows, widths, dtype, ragged_chunks=False):
    g = torch.Generator().manual_seed(seed)
    pools = [torch.randn(P, rows, d, generator=g).to(dtype) for d in widths]
    page_of = torch.randperm(P, generator=g)[: n_lib * C].view(n_lib, C).to(torch.int32)
    page_of[:, 0] = page_of[0, 0]
    n_valid = torch.randint(0, rows + 1, (n_lib, C), generator=g, dtype=torch.int32)
    nco = torch.randint(1, C + 1, (n_lib,), generator=g, dtype=torch.int32) if ragged_chunks else None
    return pools, page_of, n_valid, nco


def _live(page_of, nco):
    t = page_of.tolist()
    return sorted({p for i, row in enumerate(t) for c, p in enumerate(row) if nco is None or c < int(nco[i])})


def _copy(pools, moves):
    out = [p.clone() for p in pools]
    for src, dst, rows in moves:
        for new, old in zip(out, pools):
            new[dst, :rows] = old[src, :rows]
            new[dst, rows:] = 0
    return out


def _fork(pools, page_of, n_valid, nco, parents, own_from):
    P, C = pools[0].shape[0], page_of.shape[1]
    live = set(_live(page_of, nco))
    free = [p for p in range(P) if p not in live]
    child, moves, missing = [], [], 0
    for parent, own in zip(parents.tolist(), own_from.tolist()):
        row = []
        for c in range(C):
            if nco is not None and c >= int(nco[parent]):
                row.append(0)
            elif c < own:
                row.append(int(page_of[parent, c]))
            elif free:
                row.append(free.pop(0))
                moves.append((int(page_of[parent, c]), row[-1], int(n_valid[parent, c])))
            else:
                row.append(-1)
                missing += 1
        child.append(row)
    return torch.tensor(child, dtype=torch.int32), missing, _copy(pools, moves)


def _compact(pools, page_of, n_valid, nco):
    live = _live(page_of, nco)
    n = len(live)
    holes = [p for p in range(n) if p not in set(live)]
    to, moves = {}, []
    for p in live:
        to[p] = p if p < n else holes.pop(0)
        if p >= n:
            rows = max(int(n_valid[i, c]) for i in range(page_of.shape[0]) for c in range(page_of.shape[1])
                       if int(page_of[i, c]) == p and (nco is None or c < int(nco[i])))
            moves.append((p, to[p], rows))
    table = [[0 if nco is not None and c >= int(nco[i]) else to[int(p)] for c, p in enumerate(row)]
             for i, row in enumerate(page_of.tolist())]
    return torch.tensor(table, dtype=torch.int32), n, _copy(pools, moves)


def _to(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]


# one page per Library up to a few hundred pages; row sizes that break 16-byte units; one pool and many
CASES = [
    (1, 1, 2, 1, [8], torch.float16, False),
    (3, 4, 40, 17, [24, 24], torch.float16, False),
    (5, 7, 100, 33, [12, 20], torch.bfloat16, True),
    (2, 3, 33, 5, [7], torch.float16, True),        # 14-byte rows: 2-byte units
    (4, 16, 1100, 3, [16], torch.float32, True),    # more pages than plan threads
    (2, 5, 64, 9, [8] * 40, torch.float16, False),  # more pools than one launch takes
    (8, 6, 96, 128, [256], torch.float16, True),
]


@pytest.mark.parametrize("n_lib,C,P,rows,widths,dtype,ragged", CASES)
@pytest.mark.parametrize("own", [0, 1, 99])
def test_fork(dev, n_lib, C, P, rows, widths, dtype, ragged, own):
    from kv_skill_v2_b200 import ops
    pools, page_of, n_valid, nco = _state(dev, 7 * C + own, n_lib, C, P, rows, widths, dtype, ragged)
    parents = torch.tensor([n_lib - 1, 0, n_lib // 2], dtype=torch.int32)
    own_from = torch.tensor([max(0, C - own), 0, C], dtype=torch.int32)
    child, missing, want = _fork(pools, page_of, n_valid, nco, parents, own_from)
    d_pools = [p.to(dev) for p in pools]
    d_of, d_nv, d_nco, d_par, d_own = _to(dev, page_of, n_valid, nco, parents, own_from)
    got, short = ops.pages_fork(d_pools, d_of, d_nv, d_par, d_own, n_chunks_of=d_nco)
    assert torch.equal(got.cpu(), child)
    assert int(short) == missing
    for g, w in zip(d_pools, want):
        assert torch.equal(g.cpu(), w)
    assert torch.equal(d_of.cpu(), page_of)  # the parents' table is left alone
    assert ops.device_status(dev) == 0


@pytest.mark.parametrize("n_lib,C,P,rows,widths,dtype,ragged", CASES)
def test_compact(dev, n_lib, C, P, rows, widths, dtype, ragged):
    from kv_skill_v2_b200 import ops
    pools, page_of, n_valid, nco = _state(dev, 11 * C, n_lib, C, P, rows, widths, dtype, ragged)
    table, n, want = _compact(pools, page_of, n_valid, nco)
    d_pools = [p.to(dev) for p in pools]
    d_of, d_nv, d_nco = _to(dev, page_of, n_valid, nco)
    got, n_live = ops.pages_compact(d_pools, d_of, d_nv, n_chunks_of=d_nco)
    assert torch.equal(got.cpu(), table)
    assert int(n_live) == n
    for g, w in zip(d_pools, want):
        assert torch.equal(g[:n].cpu(), w[:n])
    # compacting what is compact moves nothing
    before = [p.clone() for p in d_pools]
    again, n2 = ops.pages_compact(d_pools, got, d_nv, n_chunks_of=d_nco)
    assert torch.equal(again, got) and int(n2) == n
    assert all(torch.equal(a, b) for a, b in zip(before, d_pools))
    assert ops.device_status(dev) == 0


def test_no_children(dev):
    from kv_skill_v2_b200 import ops
    pools, page_of, n_valid, _ = _state(dev, 1, 2, 3, 10, 4, [8], torch.float16)
    none = torch.empty(0, dtype=torch.int32, device=dev)
    child, short = ops.pages_fork([pools[0].to(dev)], page_of.to(dev), n_valid.to(dev), none, none)
    assert child.shape == (0, 3) and int(short) == 0


def test_bad_entries_are_flagged(dev):
    from kv_skill_v2_b200 import _native as N
    from kv_skill_v2_b200 import ops
    pools, page_of, n_valid, _ = _state(dev, 2, 3, 4, 30, 4, [8], torch.float16)
    page_of[1, 2] = 30   # one past the pool
    page_of[2, 1] = -5
    pool = pools[0].to(dev)
    par = torch.tensor([1, 2, 3, -1], dtype=torch.int32, device=dev)  # two of them are no Library
    own = torch.tensor([0, 4, 0, 0], dtype=torch.int32, device=dev)
    child, short = ops.pages_fork([pool], page_of.to(dev), n_valid.to(dev), par, own)
    assert int(child[0, 2]) == -1 and int(child[1, 1]) == -1
    assert (child[2:] == -1).all() and int(short) == 0
    assert ops.device_status(dev) & N.DEV_BADPAGE
    table, _ = ops.pages_compact([pool], page_of.to(dev), n_valid.to(dev))
    assert int(table[1, 2]) == 30 and int(table[2, 1]) == -5
    assert ops.device_status(dev) & N.DEV_BADPAGE


def test_valid_rows_beyond_the_page_are_clamped(dev):
    from kv_skill_v2_b200 import _native as N
    from kv_skill_v2_b200 import ops
    pools, page_of, n_valid, _ = _state(dev, 3, 1, 2, 8, 4, [8], torch.float16)
    n_valid[0, 1] = 1000
    pool = pools[0].to(dev)
    one = torch.zeros(1, dtype=torch.int32, device=dev)
    child, _ = ops.pages_fork([pool], page_of.to(dev), n_valid.to(dev), one, one)
    assert torch.equal(pool[int(child[0, 1])], pool[int(page_of[0, 1])])
    assert ops.device_status(dev) & N.DEV_CLAMPED


def test_captured_and_on_another_stream(dev):
    from kv_skill_v2_b200 import ops
    pools, page_of, n_valid, _ = _state(dev, 4, 4, 6, 64, 32, [64, 64], torch.float16)
    par, own = torch.tensor([2, 0], dtype=torch.int32), torch.tensor([4, 5], dtype=torch.int32)
    child, _, want = _fork(pools, page_of, n_valid, None, par, own)
    d_pools = [p.to(dev) for p in pools]
    d_of, d_nv, d_par, d_own = _to(dev, page_of, n_valid, par, own)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got, _ = ops.pages_fork(d_pools, d_of, d_nv, d_par, d_own)
    side.synchronize()
    assert torch.equal(got.cpu(), child)
    for p, q in zip(d_pools, pools):
        p.copy_(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, _ = ops.pages_fork(d_pools, d_of, d_nv, d_par, d_own)
    for p, q in zip(d_pools, pools):
        p.copy_(q)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got.cpu(), child)
    for g, w in zip(d_pools, want):
        assert torch.equal(g.cpu(), w)
