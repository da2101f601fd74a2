"""Attention mass against its definition in 64 bits.

Tolerance: a float32 q takes part with 22 bits, so a score near 1 is off by at most 2^-21, times read_temp = 12 that is 6e-6
of a weight, and the sums are float32: the house bound for float32 results, 2e-5 of the largest mass, holds both. With bf16
slots q keeps 16 bits: each of its d_s products is off by up to 2^-17 of itself, which random signs leave at 2^-17 |q| |k| /
sqrt(d_s) of a score, 12 times that of a weight; 1e-4 of the largest mass allows for d_s = 8 and more."""

from __future__ import annotations

import pytest
import torch

from kv_skill_v2_b200 import _native as N
from kv_skill_v2_b200 import ops

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TEMP = 12.0


def tol(q, slots):
    return 1e-4 if q.dtype is not BF16 and slots.dtype is BF16 else 2e-5


def unit(x):
    return x / x.norm(dim=-1, keepdim=True)


def case(seed, n_lib, T, shared, private, rows, d, k, slots=F16, q=F32, ragged=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    C, P = shared + private, shared + n_lib * private
    order = torch.randperm(P, generator=g, device="cuda")
    common = torch.arange(shared, device="cuda").expand(n_lib, shared)
    mine = shared + torch.arange(n_lib * private, device="cuda").view(n_lib, private)
    page_of = order[torch.cat([common, mine], 1)].to(torch.int32).contiguous()
    n_valid = torch.full((n_lib, C), rows, dtype=torch.int32, device="cuda")
    if ragged:
        n_valid = torch.randint(1, rows + 1, (n_lib, C), generator=g, device="cuda", dtype=torch.int32)
    pool = unit(torch.randn(P, rows, d, generator=g, device="cuda")).to(slots)
    R = n_lib * T
    near = torch.randint(0, P * rows, (R,), generator=g, device="cuda")
    qv = unit(unit(torch.randn(R, d, generator=g, device="cuda")) + 0.6 * pool.view(-1, d)[near].float()).to(q)
    idx = torch.stack([torch.randperm(C, generator=g, device="cuda")[:k] for _ in range(R)]).to(torch.int32)
    wk = torch.rand(R, k, generator=g, device="cuda")
    pages = ops.Pages(slots=pool, page_of=page_of, n_valid=n_valid, S=torch.zeros(n_lib, C, d, device="cuda"))
    return qv, pages, idx, wk, T


def reference(q, pages, idx, wk, T, temp=TEMP, prior=None, decay=1.0):
    P, rows, d = pages.slots.shape
    out = torch.zeros(P, rows, dtype=torch.float64, device="cuda") if prior is None else decay * prior.double()
    po, nv = pages.page_of.tolist(), pages.n_valid.tolist()
    for lib in range(len(po)):
        sl = slice(lib * T, (lib + 1) * T)
        for c, (p, n) in enumerate(zip(po[lib], nv[lib])):
            n = min(n, rows)
            w = (wk[sl].double() * (idx[sl] == c)).sum(1)
            reads = w.nonzero().view(-1)
            if not reads.numel() or n <= 0 or not 0 <= p < P:
                continue
            a = torch.softmax(temp * (q[sl][reads].double() @ pages.slots[p, :n].double().t()), -1)
            out[p, :n] += w[reads] @ a
    return out


def close(got, want, bound):
    assert got.dtype == F32 and got.shape == want.shape
    err = float((got.double() - want).abs().max() / want.abs().max().clamp(min=1e-300))
    assert err < bound, err


SHAPES = [
    # n_lib, rows a Library, shared, private, page_rows, d_s, k
    (1, 1, 1, 0, 1, 8, 1), (1, 1, 3, 0, 17, 72, 2), (1, 4, 8, 0, 96, 256, 2), (2, 3, 2, 2, 255, 136, 4),
    (1, 64, 16, 0, 256, 512, 4), (3, 5, 3, 2, 257, 1032, 3), (1, 130, 2, 0, 512, 192, 1), (2, 200, 3, 1, 300, 64, 2),
    (1, 257, 1, 0, 33, 2560, 1), (4, 40, 6, 3, 700, 264, 5), (1, 20, 4, 0, 1025, 128, 2), (2, 3, 2, 1, 2048, 64, 2),
    (1, 600, 40, 0, 64, 128, 30), (5, 1, 0, 7, 512, 2048, 7), (1, 3000, 12, 0, 130, 64, 6),
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("slots,q", [(F16, F32), (F16, BF16), (F16, F16), (BF16, F32), (BF16, BF16), (BF16, F16)])
def test_mass(shape, slots, q):
    a = case(1, *shape, slots=slots, q=q)
    got = ops.read_mass(*a[:4], rows_per_lib=a[4])
    close(got, reference(*a), tol(a[0], a[1].slots))
    assert torch.equal(got, ops.read_mass(*a[:4], rows_per_lib=a[4]))  # the order of atomics does not show
    assert not ops.device_status(torch.device("cuda:0"))


@pytest.mark.parametrize("shape", [(1, 1, 1, 0, 300, 512, 1), (1, 1, 4, 0, 700, 2560, 1), (1, 4, 20, 0, 96, 256, 2),
                                   (3, 20, 20, 4, 100, 64, 3), (2, 30, 20, 4, 300, 512, 4), (1, 40, 1, 0, 520, 64, 1),
                                   (1, 1, 2, 0, 2048, 72, 2), (1, 90, 2, 0, 257, 40, 2), (1, 150, 2, 0, 64, 24, 1),
                                   (1, 700, 8, 0, 90, 64, 2), (4, 300, 6, 2, 260, 128, 4)])
@pytest.mark.parametrize("slots", [F16, BF16])
def test_a_float32_query_keeps_its_precision(shape, slots):
    """In norm: 22 or 24 bits of q are next to nothing (2e-7 of a weight), 16 are 4.4e-7 where a call has as many pairs a page
    as it must have for them, float32 scores and sums 2e-7 or so: 1e-6 bounds it, whatever the slots' type."""
    a = case(13, *shape, slots=slots)
    want = reference(*a)
    off = float((ops.read_mass(*a[:4], rows_per_lib=a[4]).double() - want).norm() / want.norm())
    assert off < 1e-6, off


@pytest.mark.parametrize("shape", [(1, 165, 1, 0, 520, 24, 1), (1, 660, 4, 0, 260, 24, 1), (2, 500, 10, 5, 700, 16, 3),
                                   (1, 33, 2, 0, 1300, 104, 1), (3, 400, 40, 30, 40, 48, 7)])
def test_three_terms_over_several_tiles(shape):
    # bf16 slots and few columns: pages of more pairs than a tile holds, with more and fewer than fit one operand in the last
    a = case(14, *shape, slots=BF16)
    prior = torch.rand(a[1].slots.shape[:2], device="cuda")
    got = ops.read_mass(*a[:4], rows_per_lib=a[4], mass=prior, decay=0.5)
    want = reference(*a, prior=prior, decay=0.5)
    close(got, want, 2e-5)
    assert float((got.double() - want).norm() / want.norm()) < 1e-6
    assert torch.equal(got, ops.read_mass(*a[:4], rows_per_lib=a[4], mass=prior, decay=0.5))
    assert not ops.device_status(torch.device("cuda:0"))


def test_prior_decay_and_in_place():
    a = case(2, 2, 9, 4, 3, 100, 128, 3)
    prior = torch.rand(a[1].slots.shape[:2], device="cuda")
    want = reference(*a, prior=prior, decay=0.75)
    keep = prior.clone()
    got = ops.read_mass(*a[:4], rows_per_lib=9, mass=prior, decay=0.75)
    close(got, want, 2e-5)
    assert torch.equal(prior, keep)
    out = ops.read_mass(*a[:4], rows_per_lib=9, mass=prior, decay=0.75, out=prior)
    assert out is prior and torch.equal(out, got)
    # pages that nothing reads keep decay * prior
    a[3].zero_()
    assert torch.equal(ops.read_mass(*a[:4], rows_per_lib=9, mass=keep, decay=0.75), keep * 0.75)


def test_pairs_that_read_nothing_and_pages_read_twice():
    q, pages, idx, wk, T = case(3, 2, 30, 6, 2, 90, 64, 4)
    wk[3] = 0.0
    idx[5, 2] = -1
    idx[7, 1] = idx[7, 0]           # the same chunk twice in a row
    pages.n_valid[1, 4] = 0          # an empty chunk
    pages.page_of[0, 1] = pages.page_of[0, 0]  # one page under two chunks
    close(ops.read_mass(q, pages, idx, wk, rows_per_lib=T), reference(q, pages, idx, wk, T), 2e-5)


def test_what_lies_behind_the_valid_slots_does_not_matter():
    q, pages, idx, wk, T = case(4, 2, 20, 3, 1, 140, 96, 3)
    # the readers of a page agree on n_valid here, so that what lies behind it is read by none
    for p in range(pages.slots.shape[0]):
        pages.n_valid[pages.page_of == p] = 7 * p + 5
    want = ops.read_mass(q, pages, idx, wk, rows_per_lib=T)
    for p in range(pages.slots.shape[0]):
        pages.slots[p, 7 * p + 5:] = float("nan") if p % 2 else float("inf")
    got = ops.read_mass(q, pages, idx, wk, rows_per_lib=T)
    assert torch.equal(got, want) and bool(got.isfinite().all())


def test_a_row_that_is_not_finite_reaches_only_what_it_reads():
    q, pages, idx, wk, T = case(5, 1, 200, 8, 0, 64, 64, 1, ragged=False)
    want = ops.read_mass(q, pages, idx, wk, rows_per_lib=T)
    q2 = q.clone()
    q2[17, 3] = float("nan")
    got = ops.read_mass(q2, pages, idx, wk, rows_per_lib=T)
    page = int(pages.page_of[0, int(idx[17, 0])])
    assert bool(got[page].isnan().all())
    others = [p for p in range(8) if p != page]
    assert torch.equal(got[others], want[others])


@pytest.mark.parametrize("T", [40, 300])
def test_pairs_whose_weight_is_nan_read_nothing(T):
    q, pages, idx, wk, T = case(12, 1, T, 6, 0, 64, 64, 3)  # (with and without a plan)
    wk[5], wk[7, 1], q[5] = float("nan"), -float("nan"), float("nan")
    mass = torch.rand(6, 64, device="cuda")
    got = ops.read_mass(q, pages, idx, wk, rows_per_lib=T, mass=mass, decay=0.5)
    assert bool(got.isfinite().all())
    clean = torch.nan_to_num(wk, nan=0.0)
    assert torch.equal(got, ops.read_mass(q, pages, idx, clean, rows_per_lib=T, mass=mass, decay=0.5))
    close(got, reference(q, pages, idx, clean, T, prior=mass, decay=0.5), 2e-5)


def test_rows_of_any_size():
    # a power of two of q is taken out row by row. Scores of up to 2^6 are off by 2^-22 of that, 12 times that is 2e-4 of a
    # weight on either side of the softmax; scores of next to nothing by nothing
    q, pages, idx, wk, T = case(6, 1, 50, 3, 0, 64, 128, 2)
    q = q * torch.exp2(torch.randint(-20, 7, (50, 1), device="cuda").float())
    close(ops.read_mass(q, pages, idx, wk, rows_per_lib=T), reference(q, pages, idx, wk, T), 1e-3)
    small = q[:, :] * 2.0 ** -40
    close(ops.read_mass(small, pages, idx, wk, rows_per_lib=T), reference(small, pages, idx, wk, T), 2e-5)


def test_a_page_outside_the_pool_and_too_many_valid_slots():
    q, pages, idx, wk, T = case(7, 1, 10, 5, 0, 40, 64, 5)
    dev = torch.device("cuda:0")
    pages.page_of[0, 2] = 99
    close(ops.read_mass(q, pages, idx, wk, rows_per_lib=T), reference(q, pages, idx, wk, T), 2e-5)
    assert ops.device_status(dev) == N.DEV_BADPAGE
    pages.page_of[0, 2] = 0
    pages.n_valid[0, 1] = 41
    close(ops.read_mass(q, pages, idx, wk, rows_per_lib=T), reference(q, pages, idx, wk, T), 2e-5)
    assert ops.device_status(dev) == N.DEV_CLAMPED


def test_a_pool_of_more_than_four_gigabytes():
    P, rows, d = 2200, 512, 2048
    pool = torch.zeros(P, rows, d, dtype=F16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(8)
    used = [0, 1029, P - 1]
    for p in used:
        pool[p] = unit(torch.randn(rows, d, generator=g, device="cuda")).half()
    pages = ops.Pages(slots=pool, page_of=torch.tensor([used], dtype=torch.int32, device="cuda"),
                      n_valid=torch.full((1, 3), rows, dtype=torch.int32, device="cuda"), S=torch.zeros(1, 3, d, device="cuda"))
    q = unit(torch.randn(5, d, generator=g, device="cuda"))
    idx = torch.tensor([[0, 1, 2]] * 5, dtype=torch.int32, device="cuda")
    wk = torch.rand(5, 3, generator=g, device="cuda")
    got = ops.read_mass(q, pages, idx, wk, rows_per_lib=5)
    close(got, reference(q, pages, idx, wk, 5), 2e-5)


def test_captured_and_on_two_streams():
    a = case(9, 2, 100, 6, 2, 512, 256, 4)
    b = case(10, 1, 33, 9, 0, 300, 512, 3)
    want_a, want_b = ops.read_mass(*a[:4], rows_per_lib=100), ops.read_mass(*b[:4], rows_per_lib=33)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            x = ops.read_mass(*a[:4], rows_per_lib=100)
        with torch.cuda.stream(s2):
            y = ops.read_mass(*b[:4], rows_per_lib=33)
        torch.cuda.synchronize()
        assert torch.equal(x, want_a) and torch.equal(y, want_b)
    graph = torch.cuda.CUDAGraph()
    q = a[0].clone()
    mass = torch.zeros_like(want_a)
    with torch.cuda.graph(graph):
        ops.read_mass(q, *a[1:4], rows_per_lib=100, mass=mass, out=mass)
    mass.zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    close(mass, 3 * reference(*a), 2e-5)


def test_refusals():
    q, pages, idx, wk, T = case(11, 1, 4, 3, 0, 16, 64, 2)
    f = lambda **k: ops.read_mass(k.get("q", q), k.get("pages", pages), k.get("idx", idx), k.get("wk", wk),  # noqa: E731
                                  rows_per_lib=k.get("T", T), mass=k.get("mass"), out=k.get("out"))
    with pytest.raises(ValueError, match="q must be"):
        f(q=q[:, :32].contiguous())
    with pytest.raises(ValueError, match="idx"):
        f(idx=idx.long())
    with pytest.raises(ValueError, match="wk"):
        f(wk=wk.half())
    with pytest.raises(ValueError, match="Libraries"):
        f(T=2)
    with pytest.raises(ValueError, match="mass must"):
        f(mass=torch.zeros(3, 15, device="cuda"))
    with pytest.raises(ValueError, match="out must"):
        f(out=torch.zeros(3, 16, device="cuda", dtype=torch.float64))
    with pytest.raises(ValueError, match="page_of"):
        f(pages=ops.Pages(pages.slots, pages.page_of.long(), pages.n_valid, pages.S))
    with pytest.raises(NotImplementedError):
        f(pages=ops.Pages(pages.slots.float(), pages.page_of, pages.n_valid, pages.S))
    with pytest.raises(NotImplementedError):
        ops.read_mass(q[:, :60].contiguous(), ops.Pages(pages.slots[..., :60].contiguous(), pages.page_of, pages.n_valid, pages.S),
                      idx, wk, rows_per_lib=T)
    with pytest.raises(NotImplementedError, match="2048"):
        big = torch.zeros(3, 2049, 64, dtype=F16, device="cuda")
        f(pages=ops.Pages(big, pages.page_of, pages.n_valid, pages.S))
    with pytest.raises(RuntimeError, match="CUDA"):
        f(wk=wk.cpu())
