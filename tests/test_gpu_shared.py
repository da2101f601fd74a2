"""Shared read against the definition in 64 bits.

Tolerance, per output element: with u the rounding of an operand (q and P; half a step of f16 2^-11 or bf16 2^-8, squared
where they enter as hi + lo pairs) and e the tensor core's accumulation (2^-23 per 16 terms), the scores are off by
at most (u + e d/16) |q| |k|, which the softmax turns into twice read_temp times that, relative; P adds u + e N/16.
These multiply A = sum_c w_c sum_n a_n |v_n|; in the linear read the scores' error multiplies sum_n |v_n| / sqrt(n)
itself. The result is rounded once (half a step). Errors add with random signs, so the 2-norm is held to far less:
1e-5 for float32 results from f16 slots, 3e-5 from bf16 slots (u^2 = 2^-16, mean-square 0.29 of it, over 2 roundings),
and for 16-bit results the output's half step plus P's and q's."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TEMP = 12.0


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def make(dev, seed, n_lib=1, rows=4, shared=4, private=0, page_rows=32, d_s=64, k=2, slots=torch.float16, untied=False,
         q_dtype=torch.float32, full=False):
    from kv_skill_v2_b200 import ops
    g = torch.Generator(device=dev).manual_seed(seed)
    P, C = shared + n_lib * private + 3, shared + private
    order = torch.randperm(P, generator=g, device=dev)
    lib = torch.arange(n_lib, device=dev)[:, None]
    page_of = torch.cat([torch.arange(shared, device=dev).expand(n_lib, shared),
                         shared + lib * private + torch.arange(private, device=dev)], 1)
    page_of = order[page_of].to(torch.int32).contiguous()
    rows_of = torch.randint(1, page_rows + 1, (P,), generator=g, device=dev, dtype=torch.int32)
    if full:
        rows_of[:] = page_rows
    n_valid = rows_of[page_of.long()].contiguous()
    pool = [torch.nn.functional.normalize(torch.randn(P, page_rows, d_s, generator=g, device=dev), dim=-1).to(slots)
            for _ in range(2 if untied else 1)]
    for p in pool:  # nothing behind the valid rows is read
        p.masked_fill_((torch.arange(page_rows, device=dev) >= rows_of[:, None])[..., None], float("nan"))
    R = n_lib * rows
    q = torch.randn(R, d_s, generator=g, device=dev) * d_s ** -0.5
    near = pool[0][page_of[torch.arange(R, device=dev) // rows, 0].long(), 0].float()
    q = torch.nn.functional.normalize(q + 0.5 * torch.rand(R, 1, generator=g, device=dev) * near, dim=-1).to(q_dtype)
    k = C if k == 0 else k
    idx = torch.stack([torch.randperm(C, generator=g, device=dev)[:k] for _ in range(R)]).to(torch.int32)
    wk = torch.rand(R, k, generator=g, device=dev)
    pages = ops.Pages(slots=pool[0], page_of=page_of, n_valid=n_valid, S=torch.zeros(n_lib, C, d_s, device=dev),
                      vslots=pool[1] if untied else None)
    return pages, q, idx.contiguous(), wk


def reference(pages, q, idx, wk, rows, softmax=True, temp=TEMP):
    """(r, bound's A for the scores, A for P) in 64 bits."""
    V = pages.slots if pages.vslots is None else pages.vslots
    r = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mag_s, mag_p = r.clone(), r.clone()
    qd, w = q.double(), wk.double()
    for lib in range(pages.n_lib):
        for c in range(pages.n_chunks):
            sel = slice(lib * rows, (lib + 1) * rows)
            weight = torch.where((idx[sel] == c) & (wk[sel] != 0), w[sel], torch.zeros_like(w[sel])).sum(1)
            mag_w = torch.where(idx[sel] == c, w[sel].abs(), torch.zeros_like(w[sel])).sum(1)
            n = min(int(pages.n_valid[lib, c]), pages.page_rows)
            hit = mag_w.nonzero().view(-1)
            if n <= 0 or hit.numel() == 0:
                continue
            p = int(pages.page_of[lib, c])
            if not 0 <= p < pages.slots.shape[0]:
                continue
            K, Vp = pages.slots[p, :n].double(), V[p, :n].double()
            s = qd[sel][hit] @ K.t()
            a = torch.softmax(temp * s, -1) if softmax else s / math.sqrt(n)
            size = qd[sel][hit].norm(dim=-1, keepdim=True) * K.norm(dim=-1).max()
            r[sel][hit] += weight[hit, None] * (a @ Vp)
            mag_p[sel][hit] += mag_w[hit, None] * (a.abs() @ Vp.abs())
            wide = 2 * abs(temp) * (a @ Vp.abs()) if softmax else Vp.abs().sum(0) / math.sqrt(n)
            mag_s[sel][hit] += mag_w[hit, None] * size * wide
    return r, mag_s, mag_p


def check(got, pages, q, idx, wk, rows, out=torch.float32, softmax=True, temp=TEMP, norm=True):
    want, mag_s, mag_p = reference(pages, q, idx, wk, rows, softmax, temp)
    u = HALF[pages.slots.dtype]
    if out == torch.float32:
        u = 2 * u * u
    e = 2.0 ** -23
    bound = (u + e * (q.shape[1] / 16 + 4)) * mag_s + (u + e * (min(512, pages.page_rows) / 16 + 8)) * mag_p
    bound = bound + HALF[out] * want.abs() + 1e-30
    diff = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (diff <= bound).all(), float((diff / bound).max())
    if norm and float(want.norm()) > 0:
        rel = float((got.double() - want).norm() / want.norm())
        limit = 1e-5 if pages.slots.dtype == torch.float16 else 3e-5
        if out != torch.float32:
            limit = HALF[out] + 2 * HALF[pages.slots.dtype]
        assert rel <= limit, rel


CASES = [
    dict(),
    dict(rows=1, shared=1, k=1, page_rows=1, d_s=8),
    dict(rows=1, shared=3, k=0, page_rows=17, d_s=200),
    dict(rows=37, shared=5, k=3, page_rows=77, d_s=256),
    dict(rows=64, shared=6, k=4, page_rows=512, d_s=512, full=True),
    dict(n_lib=5, rows=2, shared=4, private=3, k=0, page_rows=130, d_s=264),
    dict(n_lib=3, rows=33, shared=2, private=1, k=2, page_rows=513, d_s=72),       # two segments
    dict(n_lib=2, rows=5, shared=3, private=2, k=3, page_rows=1300, d_s=136),      # three
    dict(rows=300, shared=3, k=2, page_rows=257, d_s=1000),                        # many tiles a page
    dict(rows=9, shared=4, k=2, page_rows=384, d_s=2048),
    dict(rows=7, shared=3, k=2, page_rows=300, d_s=2560),                          # clusters of 8
    dict(n_lib=2, rows=40, shared=2, private=1, k=0, page_rows=600, d_s=4096),
    dict(n_lib=40, rows=1, shared=30, private=10, k=0, page_rows=64, d_s=128),     # 1600 pairs
    dict(n_lib=2, rows=700, shared=20, private=4, k=6, page_rows=40, d_s=64),      # the plan in three kernels
    dict(rows=16, shared=4, k=2, page_rows=100, d_s=320, untied=True),
    dict(n_lib=3, rows=20, shared=2, private=2, k=0, page_rows=520, d_s=96, untied=True),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("slots", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("out", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("softmax", [True, False])
def test_against_the_definition(dev, case, slots, out, softmax):
    from kv_skill_v2_b200 import ops
    c = CASES[case]
    rows = c.get("rows", 4)
    pages, q, idx, wk = make(dev, 100 + case, slots=slots, **c)
    got = ops.read_shared(q, pages, idx, wk, rows_per_lib=rows, read_temp=TEMP, read_softmax=softmax, out_dtype=out)
    assert got.dtype == out and got.shape == q.shape
    # the linear read of many slots cancels: its 2-norm is judged by the element bound alone
    check(got, pages, q, idx, wk, rows, out, softmax, norm=softmax)
    assert ops.device_status(dev) == 0


@pytest.mark.parametrize("q_dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_half_queries(dev, q_dtype, out):
    from kv_skill_v2_b200 import ops
    pages, q, idx, wk = make(dev, 3, rows=20, shared=5, k=3, page_rows=90, d_s=512, q_dtype=q_dtype)
    check(ops.read_shared(q, pages, idx, wk, rows_per_lib=20, out_dtype=out), pages, q, idx, wk, 20, out)


@pytest.mark.parametrize("size", [1e-6, 1e4])
def test_queries_of_any_size(dev, size):
    from kv_skill_v2_b200 import ops
    pages, q, idx, wk = make(dev, 4, rows=20, shared=5, k=3, page_rows=90, d_s=512)
    q = q * size
    temp = TEMP / size
    check(ops.read_shared(q, pages, idx, wk, rows_per_lib=20, read_temp=temp), pages, q, idx, wk, 20, temp=temp)


def test_same_as_the_decode_read(dev):
    """read_decode rounds q and P to f16 once: both are within its 2e-3 of the definition."""
    from kv_skill_v2_b200 import ops
    pages, q, idx, wk = make(dev, 5, n_lib=4, rows=3, shared=6, private=2, k=4, page_rows=200, d_s=1024, full=True)
    a = ops.read_shared(q, pages, idx, wk, rows_per_lib=3)
    b = ops.read_decode(q, pages, idx, wk, rows_per_lib=3)
    assert float((a - b).abs().max() / b.abs().max()) <= 2e-3


def test_rows_that_read_nothing(dev):
    from kv_skill_v2_b200 import ops
    pages, q, idx, wk = make(dev, 6, rows=12, shared=5, k=3, page_rows=50, d_s=128)
    idx[2], wk[3], idx[4, 1], wk[5, 2] = -1, 0.0, -1, 0.0
    pages.n_valid[0, 4] = 0
    r = ops.read_shared(q, pages, idx, wk, rows_per_lib=12)
    wk2 = torch.where(idx < 0, torch.zeros_like(wk), wk)
    check(r, pages, q, idx.clamp(min=0), wk2, 12)
    assert (r[2] == 0).all() and (r[3] == 0).all()
    idx[:] = -1
    assert (ops.read_shared(q, pages, idx, wk, rows_per_lib=12) == 0).all()
    assert ops.device_status(dev) == 0


def test_a_chunk_twice_in_a_row_and_signed_weights(dev):
    from kv_skill_v2_b200 import ops
    pages, q, idx, wk = make(dev, 7, rows=70, shared=4, k=4, page_rows=50, d_s=128)
    idx[:, 2] = idx[:, 0]
    wk[:, 1] *= -1
    check(ops.read_shared(q, pages, idx, wk, rows_per_lib=70), pages, q, idx, wk, 70)


@pytest.mark.parametrize("page_rows", [100, 700])
def test_libraries_that_disagree_on_a_page(dev, page_rows):
    from kv_skill_v2_b200 import ops
    pages, q, idx, wk = make(dev, 8, n_lib=6, rows=3, shared=3, k=0, page_rows=page_rows, d_s=256, full=True)
    g = torch.Generator(device=dev).manual_seed(1)
    pages.n_valid.copy_(torch.randint(0, page_rows + 1, pages.n_valid.shape, generator=g, device=dev))
    check(ops.read_shared(q, pages, idx, wk, rows_per_lib=3), pages, q, idx, wk, 3)


def test_the_result_does_not_depend_on_the_other_rows(dev):
    from kv_skill_v2_b200 import ops
    pages, q, idx, wk = make(dev, 9, rows=150, shared=4, k=2, page_rows=300, d_s=512)
    whole = ops.read_shared(q, pages, idx, wk, rows_per_lib=150)
    for _ in range(3):
        assert torch.equal(whole, ops.read_shared(q, pages, idx, wk, rows_per_lib=150))
    few = torch.tensor([0, 77, 149], device=dev)
    part = ops.read_shared(q[few].contiguous(), pages, idx[few].contiguous(), wk[few].contiguous(), rows_per_lib=3)
    assert torch.equal(whole[few], part)


def test_a_row_that_is_not_finite_spoils_only_itself(dev):
    from kv_skill_v2_b200 import ops
    pages, q, idx, wk = make(dev, 10, rows=40, shared=2, k=2, page_rows=120, d_s=256)
    clean = ops.read_shared(q, pages, idx, wk, rows_per_lib=40)
    q[7, 3] = float("nan")
    r = ops.read_shared(q, pages, idx, wk, rows_per_lib=40)
    rest = torch.arange(40, device=dev) != 7
    assert torch.equal(r[rest], clean[rest]) and torch.isnan(r[7]).all()


def test_bad_entries_are_flagged(dev):
    from kv_skill_v2_b200 import _native as N
    from kv_skill_v2_b200 import ops
    pages, q, idx, wk = make(dev, 11, rows=8, shared=4, k=2, page_rows=50, d_s=128, full=True)
    good = ops.read_shared(q, pages, idx, wk, rows_per_lib=8)
    assert ops.device_status(dev) == 0
    idx[3, 0] = 4  # one past the Library's chunks
    r = ops.read_shared(q, pages, idx, wk, rows_per_lib=8)
    assert ops.device_status(dev) & N.DEV_BADPAGE
    rest = torch.arange(8, device=dev) != 3
    assert torch.equal(r[rest], good[rest])
    idx[3, 0] = 0
    pages.page_of[0, 1] = pages.slots.shape[0]
    r = ops.read_shared(q, pages, idx, wk, rows_per_lib=8)
    assert ops.device_status(dev) & N.DEV_BADPAGE and torch.isfinite(r).all()
    pages.page_of[0, 1] = 0
    pages.n_valid[0, 2] = 1000
    ops.read_shared(q, pages, idx, wk, rows_per_lib=8)
    assert ops.device_status(dev) & N.DEV_CLAMPED


def test_streams_and_graphs(dev):
    from kv_skill_v2_b200 import ops
    pages, q, idx, wk = make(dev, 12, n_lib=2, rows=30, shared=4, private=2, k=3, page_rows=200, d_s=512)
    want = ops.read_shared(q, pages, idx, wk, rows_per_lib=30)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = []
    for s in streams:  # two calls at once
        with torch.cuda.stream(s):
            got.append(ops.read_shared(q, pages, idx, wk, rows_per_lib=30))
    torch.cuda.synchronize()
    assert all(torch.equal(want, g) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.read_shared(q, pages, idx, wk, rows_per_lib=30)
        flat = ops.read_shared(q, pages, idx, wk, rows_per_lib=30, read_softmax=False)
    idx2 = idx.flip(0).contiguous()
    want2 = ops.read_shared(q, pages, idx2, wk, rows_per_lib=30)
    flat2 = ops.read_shared(q, pages, idx2, wk, rows_per_lib=30, read_softmax=False)
    for now, a in ((idx2, want2), (None, want2)):
        if now is not None:
            idx.copy_(now)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, a) and torch.equal(flat, flat2)


def test_refusals(dev):
    from kv_skill_v2_b200 import ops
    pages, q, idx, wk = make(dev, 13, rows=4, shared=4, k=2, page_rows=8, d_s=64)
    for bad in (dict(q=q[:, :56].contiguous()), dict(q=q[:3]), dict(idx=idx.long()), dict(idx=idx[:, :1]),
                dict(wk=wk.double()), dict(out_dtype=torch.float64), dict(q=q.double()), dict(rows_per_lib=0),
                dict(rows_per_lib=1), dict(idx=idx[:, :0], wk=wk[:, :0])):
        a = dict(q=q, idx=idx, wk=wk, rows_per_lib=4, out_dtype=torch.float32) | bad
        with pytest.raises(ValueError):
            ops.read_shared(a.pop("q"), pages, a.pop("idx"), a.pop("wk"), **a)
    for slots, d in ((pages.slots.float(), 64), (pages.slots[:, :, :60].contiguous(), 60)):
        p = ops.Pages(slots=slots, page_of=pages.page_of, n_valid=pages.n_valid, S=pages.S)
        with pytest.raises(NotImplementedError):
            ops.read_shared(q[:, :d].contiguous(), p, idx, wk, rows_per_lib=4)
    with pytest.raises(RuntimeError):
        ops.read_shared(q.cpu(), pages, idx, wk, rows_per_lib=4)


@pytest.mark.parametrize("d_s,page_rows", [(2048, 512), (1024, 300), (256, 130)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_pages_of_few_and_of_many_pairs_in_turn(dev, d_s, page_rows, out):
    """Each cluster meets units of both kinds, several of them, in a random order."""
    from kv_skill_v2_b200 import ops
    C, R = 220, 260
    pages, q, idx, wk = make(dev, 21, rows=R, shared=C, k=6, page_rows=page_rows, d_s=d_s)
    g = torch.Generator(device=dev).manual_seed(5)
    busy = torch.randperm(C, generator=g, device=dev)[:60]
    many = torch.rand(R, 6, generator=g, device=dev) < 0.7  # most pairs go to a few pages
    idx = torch.where(many, busy[torch.randint(0, 60, (R, 6), generator=g, device=dev)].to(torch.int32), idx)
    idx = idx.contiguous()
    got = ops.read_shared(q, pages, idx, wk, rows_per_lib=R, out_dtype=out)
    check(got, pages, q, idx, wk, R, out)
    assert ops.device_status(dev) == 0


@pytest.mark.parametrize("slots,out", [(torch.float16, torch.float32), (torch.bfloat16, torch.float32),
                                       (torch.float16, torch.bfloat16)])
@pytest.mark.parametrize("d_s,page_rows", [(2048, 512), (1024, 300), (256, 1100)])
def test_the_tail_of_a_page_gives_the_same_bits(dev, d_s, page_rows, slots, out):
    """A page's last few pairs take another form of the read, and which pairs those are is up to the order of the
    count: the result is the same to the bit, run after run and with a row alone."""
    from kv_skill_v2_b200 import ops
    R = 69  # 64 + 5, 2 * 32 + 5
    pages, q, idx, wk = make(dev, 31, rows=R, shared=3, k=0, page_rows=page_rows, d_s=d_s, slots=slots)
    whole = ops.read_shared(q, pages, idx, wk, rows_per_lib=R, out_dtype=out)
    for _ in range(5):
        assert torch.equal(whole, ops.read_shared(q, pages, idx, wk, rows_per_lib=R, out_dtype=out))
    for row in (0, 33, 68):
        one = ops.read_shared(q[row:row + 1].contiguous(), pages, idx[row:row + 1].contiguous(),
                              wk[row:row + 1].contiguous(), rows_per_lib=1, out_dtype=out)
        assert torch.equal(whole[row:row + 1], one)


@pytest.mark.parametrize("slots", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("softmax,size,temp", [(True, 1e-34, TEMP), (True, 1e-36, TEMP), (True, 1e-34, TEMP / 1e-34),
                                               (False, 1e-34, TEMP), (False, 1e-30, TEMP)])
def test_queries_near_the_smallest_floats(dev, slots, out, softmax, size, temp):
    """2^15 over the row's largest value is no float32 from 2^-112 down: the row's scale stops at 2^126. The linear read
    is compared in units of `size` (its bound has an absolute part); its coefficient 1 / (2^126 sqrt(n)) keeps 20 bits,
    half a step of which (2^-21) is below the bound's 2^-23 (d_s / 16)."""
    from kv_skill_v2_b200 import ops
    pages, q, idx, wk = make(dev, 14, rows=40, shared=5, k=3, page_rows=90, d_s=512, slots=slots)
    q = q * size
    q[:, ::7] = 0.0
    q[3] = 0.0
    got = ops.read_shared(q, pages, idx, wk, rows_per_lib=40, read_temp=temp, read_softmax=softmax, out_dtype=out)
    if softmax:
        check(got, pages, q, idx, wk, 40, out, temp=temp)
    else:
        check(got.double() / size, pages, q.double() / size, idx, wk, 40, out, softmax=False, norm=False)
    assert ops.device_status(dev) == 0


@pytest.mark.parametrize("case", [dict(rows=70, shared=5, k=3, page_rows=200, d_s=256),
                                  dict(n_lib=7, rows=9, shared=3, private=2, k=0, page_rows=600, d_s=128),
                                  dict(n_lib=3, rows=41, shared=4, private=1, k=4, page_rows=90, d_s=512)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_slices_give_the_same_bits(dev, case, out):
    """A workspace limit cuts the rows into slices: within Libraries, at their borders, down to one row each."""
    from kv_skill_v2_b200 import ops
    rows = case["rows"]
    pages, q, idx, wk = make(dev, 16, **case)
    whole = ops.read_shared(q, pages, idx, wk, rows_per_lib=rows, out_dtype=out)
    need = ops.shared_workspace(pages, q.shape[0], idx.shape[1], out)
    for limit in (need // 2, need // 5, need // 30, 1):
        got = ops.read_shared(q, pages, idx, wk, rows_per_lib=rows, out_dtype=out, max_workspace=limit)
        assert torch.equal(got, whole)
    # a last Library that is cut, and more rows than Libraries
    cut = ops.read_shared(q[:-2], pages, idx[:-2], wk[:-2], rows_per_lib=rows, out_dtype=out, max_workspace=need // 5)
    assert torch.equal(cut, whole[:-2])
    with pytest.raises(ValueError):
        ops.read_shared(q, pages, idx, wk, rows_per_lib=rows - 1, out_dtype=out, max_workspace=need // 5)
    assert ops.device_status(dev) == 0


@pytest.mark.parametrize("d_s,page_rows", [(256, 100), (2048, 300), (2560, 90), (256, 700)])
@pytest.mark.parametrize("slots", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("softmax", [True, False])
def test_a_slot_that_is_not_finite_reaches_only_its_readers(dev, d_s, page_rows, slots, softmax):
    """Libraries that name one page with different n_valid: NaN in the slots that only some of them read."""
    from kv_skill_v2_b200 import ops
    n_lib, rows = 5, 8
    pages, q, idx, wk = make(dev, 15, n_lib=n_lib, rows=rows, shared=3, k=0, page_rows=page_rows, d_s=d_s, slots=slots,
                             full=True)
    few = page_rows * 2 // 3
    pages.n_valid[:3] = few
    pages.n_valid[4] = few - 20
    pages.slots[pages.page_of[0, 1].long(), few:] = float("nan")
    r = ops.read_shared(q, pages, idx, wk, rows_per_lib=rows, read_softmax=softmax)
    keep = torch.arange(n_lib * rows, device=dev) // rows != 3
    assert torch.isnan(r[~keep]).all()
    want, mag_s, mag_p = reference(pages, q, idx, wk, rows, softmax)
    e, u = 2.0 ** -23, 2 * HALF[slots] ** 2
    bound = (u + e * (d_s / 16 + 4)) * mag_s + (u + e * 40) * mag_p + 2.0 ** -24 * want.abs() + 1e-30
    assert ((r.double() - want).abs() <= bound)[keep].all()
    # the same bits as from a call that nobody else is part of
    one = ops.Pages(slots=pages.slots, page_of=pages.page_of[4:5].contiguous(),
                    n_valid=pages.n_valid[4:5].contiguous(), S=pages.S[4:5])
    at = slice(4 * rows, 5 * rows)
    alone = ops.read_shared(q[at].contiguous(), one, idx[at].contiguous(), wk[at].contiguous(), rows_per_lib=rows,
                            read_softmax=softmax)
    assert torch.equal(r[at], alone)


def test_a_slot_that_is_not_finite_among_many_pairs(dev):
    """The same where the plan takes several launches (more than 4096 pairs) and pages have several tiles; the page of
    another chunk only has another length."""
    from kv_skill_v2_b200 import ops
    n_lib, rows = 5, 300
    pages, q, idx, wk = make(dev, 17, n_lib=n_lib, rows=rows, shared=6, k=3, page_rows=80, d_s=64, full=True)
    pages.n_valid[:2, 1] = 50
    pages.n_valid[2, 4] = 60
    pages.slots[pages.page_of[0, 1].long(), 70, 5] = float("inf")
    r = ops.read_shared(q, pages, idx, wk, rows_per_lib=rows)
    reads = ((idx == 1) & (torch.arange(n_lib * rows, device=dev) // rows >= 2)[:, None]).any(1)
    want, mag_s, mag_p = reference(pages, q, idx, wk, rows)
    bound = (2.0 ** -21 + 2.0 ** -23 * 8) * mag_s + (2.0 ** -21 + 2.0 ** -23 * 13) * mag_p + 2.0 ** -24 * want.abs() + 1e-30
    assert ((r.double() - want).abs() <= bound)[~reads].all() and torch.isfinite(r[~reads]).all()
    assert not torch.isfinite(r[reads]).all(-1).any()
    assert ops.device_status(dev) == 0
