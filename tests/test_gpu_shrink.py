"""A served Library that shrinks, as a server runs it: prompts record the attention that the slots get, the Library is
evicted by it, the steps that follow read what is left, and the interface's projections run in 8 bits -- against the
definitions in 64 bits."""

from __future__ import annotations

import pytest
import torch

from kv_skill_v2_b200 import LayerSelector, LibraryInjector, PagedLibrary, make_interface, ops
from kv_skill_v2_b200.interface import LinearInterface
from tests._fixtures import TOL, TinyReader, rel_err

pytestmark = pytest.mark.gpu
D_M, D_S, LAYERS = 96, 64, [1, 3]
DEV = torch.device("cuda:0")


def library(seed=0, n_lib=3, C=5, rows=24, untied=False, ragged=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pools = {li: torch.nn.functional.normalize(torch.randn(n_lib * C, rows, D_S, generator=g, device="cuda"), dim=-1).half()
             for li in LAYERS}
    vals = {li: torch.randn_like(p) for li, p in pools.items()} if untied else None
    page_of = torch.randperm(n_lib * C, generator=g, device="cuda").view(n_lib, C).to(torch.int32)
    n_valid = torch.randint(rows // 2, rows + 1, (n_lib, C), generator=g, device="cuda", dtype=torch.int32)
    nco = torch.tensor([C, C - 2, C - 1], dtype=torch.int32, device="cuda")[:n_lib] if ragged else None
    return PagedLibrary.from_pool(pools, page_of, n_valid, nco, layer_vslots=vals)


def interface(seed, layers=LAYERS):
    g = torch.Generator(device="cuda").manual_seed(seed)
    W_in = torch.randn(D_M, D_S, generator=g, device="cuda") * D_M ** -0.5
    W_out = torch.randn(D_S, D_M, generator=g, device="cuda") * 0.2
    return LinearInterface(W_in, W_out, layers).cuda().requires_grad_(False)


def chunks(lib, b):
    nco = lib.pages(LAYERS[0]).n_chunks_of
    return lib.n_chunks if nco is None else int(nco[b])


def e4m3(x):
    """x [n, k] float64 in blocks of 128 columns as the 8-bit format holds them."""
    n, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % 128)).view(n, -1, 128)
    mx = x.abs().amax(-1, keepdim=True)
    two = torch.exp2(torch.ceil(torch.log2(mx.clamp(min=1e-300) / 448.0)))
    v = x / torch.where(mx > 0, two, 1.0)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step * two).view(n, -1)[:, :k]


def step(h, itf, lib, li, top_k, fp8=False, live=None):
    """(delta, mass by page) of one read in 64 bits: q by the interface's map, softmax routing and read."""
    p = lib.pages(li)
    P, N = p.slots.shape[:2]
    mass = torch.zeros(P, N, dtype=torch.float64, device="cuda")
    w_in, w_out = itf.w_in.double(), itf.w_out.double()
    if fp8:
        w_in, w_out = e4m3(w_in), e4m3(w_out)
    V = p.slots if p.vslots is None else p.vslots
    out = torch.zeros(h.shape, dtype=torch.float64, device="cuda")
    for b in range(h.shape[0]):
        x = h[b].double()
        q = (e4m3(x) if fp8 else x) @ w_in.t() * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6)
        q = q / (q.norm(dim=-1, keepdim=True) + 1e-6)
        n = chunks(lib, b)
        logits = q @ p.S[b, :n].double().t() * 10.0
        k = top_k if 0 < top_k < n else n
        top, idx = logits.topk(k, dim=-1)
        w = torch.softmax(top, -1)
        r = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        for t in range(q.shape[0]):
            for j in range(k):
                page, nv = int(p.page_of[b, int(idx[t, j])]), int(p.n_valid[b, int(idx[t, j])])
                a = w[t, j] * torch.softmax(12.0 * p.slots[page, :nv].double() @ q[t], 0)
                r[t] += a @ V[page, :nv].double()
                if live is None or bool(live[b, t]):
                    mass[page, :nv] += a
        out[b] = (e4m3(r.float().double()) if fp8 else r) @ w_out.t()
    return out, mass


def close(got, want, tol):
    assert float((got.double() - want).abs().max()) <= tol * float(want.abs().max())


@pytest.mark.parametrize("share", [False, True])
@pytest.mark.parametrize("top_k", [2, 0])
def test_reads_record_the_attention_of_their_slots(share, top_k):
    lib = library(1).reserve(4).fork([0, 2], own_from=[3, 2])
    inj = LibraryInjector(TinyReader(D_M, 5).cuda(), itf := interface(2), top_k=top_k, share_pages=share)
    inj.load_library(lib)
    g = torch.Generator(device="cuda").manual_seed(3)
    want = {li: 0.0 for li in LAYERS}
    inj.record_mass, inj.mass_decay = True, 0.5
    with torch.no_grad():
        for T in (40, 1, 1):
            h = torch.randn(lib.n_lib, T, D_M, generator=g, device="cuda")
            for li in LAYERS:
                got, _ = inj._inject(h, li)
                delta, mass = step(h, itf, lib, li, top_k)
                assert rel_err(got - h, delta) <= TOL
                want[li] = 0.5 * want[li] + mass
    for li in LAYERS:  # (q is float32: its 2e-6 reach the weights twelvefold)
        close(inj.slot_mass[li], want[li], 1e-4)
    inj.load_library(lib)
    assert inj.slot_mass == {}
    inj.detach()


def test_a_captured_step_records():
    lib = library(40)
    inj = LibraryInjector(TinyReader(D_M, 5).cuda(), itf := interface(41), top_k=2)
    inj.load_library(lib)
    inj.record_mass = inj.gemm_fp8 = True
    g = torch.Generator(device="cuda").manual_seed(42)
    x, h = torch.zeros(3, 1, D_M, device="cuda"), torch.randn(3, 1, D_M, generator=g, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="before it is captured"):  # nothing there yet that replays could add to
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                inj._inject(x, 1)
        inj._inject(h, 1)
        first = inj.slot_mass[1].clone()
        with torch.cuda.graph(graph):
            inj._inject(x, 1)
    inj.slot_mass[1].zero_()
    x.copy_(h)
    for _ in range(3):
        graph.replay()
    close(inj.slot_mass[1], 3 * first.double(), 1e-6)
    close(first, step(h, itf, lib, 1, 2, fp8=True)[1], 1e-3)
    inj.detach()


def test_a_weight_first_used_in_a_capture():
    lib, itf = library(43), interface(44)
    h = torch.randn(3, 2, D_M, generator=torch.Generator(device="cuda").manual_seed(45), device="cuda")
    inj = LibraryInjector(TinyReader(D_M, 5).cuda(), itf, top_k=2)
    inj.load_library(lib)
    inj.gemm_fp8 = True
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        with torch.cuda.graph(graph):
            got = inj._inject(h, 1)[0]
        want = inj._inject(h, 1)[0].clone()  # before any replay: not with what the graph has yet to write
        graph.replay()
        assert torch.equal(got, want) and not torch.equal(want, h)
        assert rel_err(want - h, step(h, itf, lib, 1, 2, fp8=True)[0]) <= 2e-2
    inj.detach()


def test_masked_positions_give_no_attention():
    """A padded batch: the position mask's zeros are not counted."""
    lib = library(4)
    inj = LibraryInjector(TinyReader(D_M, 5).cuda(), itf := interface(5), top_k=2)
    inj.load_library(lib)
    inj.record_mass = True
    h = torch.randn(3, 9, D_M, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    live = torch.ones(3, 9, device="cuda")
    live[0, :4], live[2, 1:] = 0, 0
    inj.pos_mask = live
    with torch.no_grad():
        inj._inject(h, 1)
    close(inj.slot_mass[1], step(h, itf, lib, 1, 2, live=live)[1], 1e-4)
    inj.detach()


@pytest.mark.parametrize("untied", [False, True])
@pytest.mark.parametrize("new_rows", [None, 10])
@pytest.mark.parametrize("per_library", [False, True])
def test_an_evicted_library_reads_what_is_left(untied, new_rows, per_library):
    lib = library(7, untied=untied)
    g = torch.Generator(device="cuda").manual_seed(8)
    P, rows = lib.pages(1).slots.shape[:2]
    mass = {li: torch.rand(P, rows, generator=g, device="cuda") for li in LAYERS}
    total = mass[1] + mass[3]
    old = {li: (lib.pages(li).slots.clone(), None if not untied else lib.pages(li).vslots.clone()) for li in LAYERS}
    n_old, S_old = lib.pages(1).n_valid.clone(), {li: lib.pages(li).S.clone() for li in LAYERS}
    keep = 22 if per_library else 7
    small, left = lib.evict(mass, keep, per_library=per_library, page_rows=new_rows)
    p = small.pages(1)
    assert p.page_rows == (new_rows or rows) and tuple(left.shape) == (P, p.page_rows)
    for b in range(3):
        n = chunks(small, b)
        if per_library:
            assert int(p.n_valid[b, :n].sum()) == min(keep, int(n_old[b, :n].clamp(max=p.page_rows).sum()))
        for c in range(n):
            page, nv = int(p.page_of[b, c]), int(p.n_valid[b, c])
            if not per_library:
                assert nv == min(keep, int(n_old[b, c]))
            kept = total[page, : int(n_old[b, c])].topk(nv).indices.sort().values
            for li in LAYERS:
                assert torch.equal(small.pages(li).slots[page, :nv], old[li][0][page, kept])
                if untied:
                    assert torch.equal(small.pages(li).vslots[page, :nv], old[li][1][page, kept])
                assert torch.equal(small.pages(li).S, S_old[li])
            close(left[page, :nv], total[page, kept].double(), 1e-6)
    inj = LibraryInjector(TinyReader(D_M, 5).cuda(), itf := interface(9), top_k=2)
    inj.load_library(small)
    h = torch.randn(3, 4, D_M, generator=g, device="cuda")
    with torch.no_grad():
        for li in LAYERS:
            for _ in range(2):
                assert rel_err(inj._inject(h, li)[0] - h, step(h, itf, small, li, 2)[0]) <= TOL
    inj.detach()
    # it is forked and compacted as any other
    grown, _ = small.reserve(3).fork([0], own_from=[2]).compact()
    q = grown.pages(3)
    for c in range(chunks(grown, 3)):
        a, b, nv = int(q.page_of[3, c]), int(q.page_of[0, c]), int(q.n_valid[0, c])
        assert torch.equal(q.slots[a, :nv], q.slots[b, :nv])


def test_a_chunk_that_would_be_empty_is_refused():
    lib = library(10, ragged=False).fork([0])
    nv = lib.pages(1).n_valid
    nv[0, 0], nv[3, 0] = 24, 2  # the fork reads two rows of a page that its parent reads whole
    mass = torch.zeros(lib.pages(1).slots.shape[:2], device="cuda")
    mass[int(lib.pages(1).page_of[0, 0]), 20:] = 1.0
    with pytest.raises(RuntimeError, match="empty chunk"):
        lib.evict(mass, 4, page_rows=8)
    with pytest.raises(ValueError, match="at least one layer"):
        lib.evict({}, 4)


def test_prompt_evict_decode_in_8_bits():
    """The whole of it: a prompt records, its Library is evicted, steps with 8-bit projections read the rest."""
    lib = library(11, rows=40)
    itf = interface(12)
    inj = LibraryInjector(TinyReader(D_M, 5).cuda(), itf, top_k=3, share_pages=True)
    inj.load_library(lib)
    g = torch.Generator(device="cuda").manual_seed(13)
    prompt = torch.randn(3, 60, D_M, generator=g, device="cuda")
    inj.record_mass = True
    inj.gemm_fp8 = True
    with torch.no_grad():
        for li in LAYERS:
            inj._inject(prompt, li)
    small, _ = lib.evict(inj.slot_mass, 12, page_rows=12)
    inj.record_mass = False
    inj.load_library(small)
    with torch.no_grad():
        for T in (1, 1, 7):
            h = torch.randn(3, T, D_M, generator=g, device="cuda")
            for li in LAYERS:
                want = step(h, itf, small, li, 3, fp8=True)[0]
                for _ in range(3):  # eager, captured, replayed. (r's rounding to 8 bits may fall on the other side of a tie:
                    # one step of e4m3 of one value of r in 64, an eighth of it against the whole sum)
                    assert rel_err(inj._inject(h, li)[0] - h, want) <= 2e-2
    assert ops.device_status(DEV) == 0
    inj.detach()


@pytest.mark.parametrize("kind", ["linear", "model", "low-rank", "selector"])
@pytest.mark.parametrize("T", [1, 50])
def test_hooked_projections_in_8_bits(kind, T):
    """An injector with gemm_fp8 is one whose interface holds the 8-bit values, with rows rounded too: against the same
    injector on float32 weights it is off by the roundings of e4m3 (2^-4 of a value, random over 64 and more of a sum)."""
    g = torch.Generator(device="cuda").manual_seed(20)
    sel = None
    if kind == "linear":
        itf = interface(21)
    else:
        itf = make_interface(D_M, D_S, LAYERS, rank=32 if kind == "low-rank" else 0).cuda()
        with torch.no_grad():
            for m in [*(itf.A if kind == "low-rank" else [itf.A]), itf.B]:
                m.weight.copy_(torch.randn(m.weight.shape, generator=g, device="cuda") * m.weight.shape[1] ** -0.5)
            itf.gate_w.copy_(torch.randn(D_M, generator=g, device="cuda") * 0.1)
        itf = itf.requires_grad_(False)
    if kind == "selector":
        sel = LayerSelector(D_M, LAYERS, k=1, alpha_init=0.05).cuda().requires_grad_(False)
        sel.u.weight.copy_(torch.randn(sel.u.weight.shape, generator=g, device="cuda"))
    reader = TinyReader(D_M, 5).cuda().eval().requires_grad_(False)
    lib = library(22)
    x = torch.randn(3, T, D_M, generator=g, device="cuda")
    outs = []
    with torch.no_grad():
        bare = reader(x)
        for fp8 in (False, True):
            inj = LibraryInjector(reader, itf, top_k=0, selector=sel)
            inj.gemm_fp8 = fp8
            inj.load_library(lib)
            first = reader(x)
            assert torch.equal(reader(x), first) or sel is not None
            outs.append(first - bare)
            inj.detach()
    off = float((outs[1] - outs[0]).norm() / outs[0].norm())
    assert 1e-4 < off < 0.1, off


def test_refusals():
    reader = TinyReader(D_M, 5).cuda()
    lib = library(30)
    h = torch.randn(3, 2, D_M, device="cuda")
    inj = LibraryInjector(reader, interface(31), read_softmax=False)
    inj.load_library(lib)
    inj.record_mass = True
    with torch.no_grad(), pytest.raises(ValueError, match="linear read"):
        inj._inject(h, 1)
    inj.detach()
    inj = LibraryInjector(reader, interface(31), top_k=2)
    inj.load_library(lib)
    inj.gemm_fp8 = True
    inj.set_adapters(ops.Adapters(torch.zeros(1, 2, D_M, device="cuda"), torch.zeros(1, D_S, 2, device="cuda")), None,
                     torch.zeros(3, dtype=torch.int32, device="cuda"))
    with torch.no_grad(), pytest.raises(NotImplementedError, match="adapters"):
        inj._inject(h, 1)
    inj.detach()
