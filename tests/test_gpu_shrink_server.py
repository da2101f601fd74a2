"""What a server does around a Library that shrinks: evictions that are refused leave it whole, one bad request does not
spoil the attention that others recorded, recorded attention goes with the pages when they are forked, moved or evicted."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from kv_skill_v2_b200 import LayerSelector, Library, LibraryInjector, ops
from tests._fixtures import TinyReader
from tests.test_gpu_shrink import D_M, D_S, DEV, LAYERS, chunks, close, interface, library, step

pytestmark = pytest.mark.gpu


def shared_short_fork():
    """Three Libraries and a fork that reads two rows of a page that its parent reads whole, with the attention behind them."""
    lib = library(10, ragged=False).fork([0])
    nv = lib.pages(1).n_valid
    nv[0, 0], nv[3, 0] = 24, 2
    mass = torch.rand(lib.pages(1).slots.shape[:2], generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") * 0.1
    page = int(lib.pages(1).page_of[0, 0])
    mass[page, 20:], mass[page, :2] = 1.0, 0.0
    return lib, mass


@pytest.mark.parametrize("per_library", [False, True])
@pytest.mark.parametrize("new_rows", [None, 8])
def test_an_eviction_that_would_empty_a_chunk_moves_nothing(per_library, new_rows):
    lib, mass = shared_short_fork()
    before = {li: lib.pages(li).slots.clone() for li in LAYERS}
    was = mass.clone()
    with pytest.raises(RuntimeError, match="empty chunk"):
        lib.evict(mass, 5 if per_library else 4, per_library=per_library, page_rows=new_rows)
    with pytest.raises(RuntimeError, match="empty chunk"):
        lib.evict({1: mass}, 0, per_library=per_library, floor=0, page_rows=new_rows)
    for li in LAYERS:
        assert torch.equal(lib.pages(li).slots, before[li])
    assert torch.equal(mass, was)
    # what every reader has some of goes as ever, and can be loaded
    mass[int(lib.pages(1).page_of[0, 0]), 0] = 2.0
    small, _ = lib.evict(mass, 20 if per_library else 4, per_library=per_library, page_rows=new_rows)
    assert int(small.pages(1).n_valid.min()) >= 1
    inj = LibraryInjector(TinyReader(D_M, 5).cuda(), interface(2), top_k=2)
    inj.load_library(small)
    inj.detach()


def test_an_eviction_is_not_captured():
    lib, mass = shared_short_fork()
    for new_rows in (None, 8):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                lib.evict(mass, 4, page_rows=new_rows)
    assert ops.device_status(DEV) == 0


@pytest.mark.parametrize("share", [False, True])
@pytest.mark.parametrize("top_k", [2, 0])
@pytest.mark.parametrize("T", [1, 9])
def test_a_request_that_is_not_finite_leaves_no_trace_in_the_mass(share, top_k, T):
    """Three Libraries and forks that share their pages: one request of the batch goes wrong, then the next steps run."""
    lib = library(1).reserve(4).fork([0, 2], own_from=[3, 2])
    g = torch.Generator(device="cuda").manual_seed(50)
    steps = [torch.randn(lib.n_lib, T, D_M, generator=g, device="cuda") for _ in range(3)]
    bad = [x.clone() for x in steps]
    bad[0][3, -1, 5], bad[1][0, 0] = float("nan"), float("inf")
    live = [torch.ones(lib.n_lib, T, device="cuda") for _ in steps]
    live[0][3, -1], live[1][0, 0] = 0, 0
    got = []
    for rows, masks in ((bad, None), (steps, live)):  # the same rows taken out by a position mask
        inj = LibraryInjector(TinyReader(D_M, 5).cuda(), interface(2), top_k=top_k, share_pages=share)
        inj.load_library(lib)
        inj.record_mass, inj.mass_decay = True, 0.5
        with torch.no_grad():
            for i, h in enumerate(rows):
                inj.pos_mask = None if masks is None else masks[i]
                for li in LAYERS:
                    inj._inject(h, li)
        got.append(inj.slot_mass)
        inj.detach()
    for li in LAYERS:
        assert bool(got[0][li].isfinite().all()) and float(got[0][li].sum()) > 0
        assert torch.equal(got[0][li], got[1][li])
    assert ops.device_status(DEV) == 0


def test_summary_keys_that_are_not_finite_leave_no_trace_in_the_mass():
    """The routing of one Library is NaN: it shares pages with a fork whose routing is not."""
    lib = library(1).fork([0])
    inj = LibraryInjector(TinyReader(D_M, 5).cuda(), interface(2), top_k=0)
    inj.load_library(lib)
    inj.record_mass = True
    h = torch.randn(lib.n_lib, 4, D_M, generator=torch.Generator(device="cuda").manual_seed(51), device="cuda")
    lib.pages(1).S[3, 1] = float("nan")
    with torch.no_grad():
        inj._inject(h, 1)
    assert bool(inj.slot_mass[1].isfinite().all())
    live = torch.ones(lib.n_lib, 4, device="cuda")
    live[3] = 0
    got, inj.slot_mass, inj.pos_mask = inj.slot_mass[1], {}, live
    with torch.no_grad():
        inj._inject(h, 1)
    assert torch.equal(got, inj.slot_mass[1])
    inj.detach()


@pytest.mark.parametrize("fp8", [False, True])
def test_a_weight_prepared_on_another_stream(fp8):
    lib, h = library(60), torch.randn(3, 2, D_M, generator=torch.Generator(device="cuda").manual_seed(61), device="cuda")
    outs = []
    for late in (False, True):
        inj = LibraryInjector(TinyReader(D_M, 5).cuda(), interface(62), top_k=2, cuda_graphs=False)
        inj.load_library(lib)
        inj.gemm_fp8 = fp8
        one, two = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.no_grad():
            if late:  # the weights are written 20 ms from now, in memory that held NaN
                with torch.cuda.stream(one):
                    for n in (64 * 128, 96 * 128, 1 << 20):
                        torch.full((n,), float("nan"), device="cuda")
                    torch.cuda._sleep(40_000_000)
                    inj._inject(h, 1)
            with torch.cuda.stream(two):
                outs.append(inj._inject(h, 1)[0])
        torch.cuda.synchronize()
        inj.detach()
    assert torch.equal(outs[0], outs[1]) and not torch.equal(outs[0], h)


@pytest.mark.parametrize("fp8", [False, True])
def test_a_weight_first_used_in_a_callers_capture(fp8):
    lib, h = library(63), torch.randn(3, 2, D_M, generator=torch.Generator(device="cuda").manual_seed(64), device="cuda")
    itf, outs = interface(65), []
    for captured in (False, True):
        inj = LibraryInjector(TinyReader(D_M, 5).cuda(), itf, top_k=2, cuda_graphs=False)
        inj.load_library(lib)
        inj.gemm_fp8 = fp8
        graph = torch.cuda.CUDAGraph()
        with torch.no_grad():
            if captured:
                with torch.cuda.graph(graph):
                    inj._inject(h, 1)
            outs.append(inj._inject(h, 1)[0])  # before any replay
        inj.detach()
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("fp8", [False, True])
def test_a_captured_step_keeps_its_weights(fp8):
    """A caller's graph reads the prepared weights in place: others that come later do not push them out."""
    lib, h = library(66), torch.randn(3, 2, D_M, generator=torch.Generator(device="cuda").manual_seed(67), device="cuda")
    inj = LibraryInjector(TinyReader(D_M, 5).cuda(), interface(68), top_k=2, cuda_graphs=False)
    inj.load_library(lib)
    inj.gemm_fp8 = fp8
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        want = inj._inject(h, 1)[0]
        with torch.cuda.graph(graph):
            got = inj._inject(h, 1)[0]
        others = [torch.full((D_S, D_M), float(i), device="cuda") for i in range(100)]
        for W in others:
            inj._weight(W)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
    assert torch.equal(got, want) and not torch.equal(want, h)
    inj.detach()


def of_slots(lib):
    """A mass that says which slot it belongs to, another for every layer."""
    return {li: lib.pages(li).slots[..., li].float().contiguous() for li in LAYERS}


def belongs(mass, lib):
    """Every valid slot's mass is its own."""
    for li in LAYERS:
        p = lib.pages(li)
        assert tuple(mass[li].shape) == tuple(p.slots.shape[:2])
        for b in range(lib.n_lib):
            for c in range(chunks(lib, b)):
                page, nv = int(p.page_of[b, c]), int(p.n_valid[b, c])
                assert nv > 0 and torch.equal(mass[li][page, :nv], p.slots[page, :nv, li].float())


@pytest.mark.parametrize("new_rows", [None, 9])
@pytest.mark.parametrize("ragged", [False, True])
def test_recorded_attention_goes_with_its_pages(new_rows, ragged):
    """reserve, fork, drop, compact, evict and load_library, as requests join and leave."""
    lib = library(70, ragged=ragged)
    inj = LibraryInjector(TinyReader(D_M, 5).cuda(), interface(71), top_k=2)
    mass = of_slots(lib)
    lib = lib.reserve(9)
    inj.load_library(lib, slot_mass=mass)
    mass = inj.slot_mass
    belongs(mass, lib)
    held = {li: mass[li].data_ptr() for li in LAYERS}
    for m in mass.values():
        m[15:] = 7.0  # what is left in free pages by those that were there
    lib = lib.fork([0, 2], own_from=[1, 2], mass=mass)
    belongs(mass, lib)
    lib = lib.drop([0, 1])
    lib, n_live = lib.compact(mass=mass)
    belongs(mass, lib)
    assert n_live < 15 and {li: mass[li].data_ptr() for li in LAYERS} == held
    lib, mass = lib.evict(mass, 8, page_rows=new_rows, per_layer=True)
    belongs(mass, lib)
    inj.load_library(lib, slot_mass=mass)
    # recording goes on from there
    inj.record_mass = True
    h = torch.randn(lib.n_lib, 3, D_M, generator=torch.Generator(device="cuda").manual_seed(72), device="cuda")
    before = mass[1].double()
    with torch.no_grad():
        inj._inject(h, 1)
    want = before + step(h, inj.itf, lib, 1, 2)[1]
    assert inj.slot_mass[1] is mass[1] and float((mass[1] - want).abs().max()) <= 1e-4 * float(want.abs().max())
    inj.detach()


def test_one_mass_for_all_layers_goes_with_its_pages():
    lib = library(73, rows=203).reserve(4)  # 203 floats: rows of no 16 bytes
    mass = of_slots(lib)[1]
    lib = lib.fork([0], own_from=[3], mass=mass).drop([1])
    lib, _ = lib.compact(mass=mass)
    p = lib.pages(1)
    for b in range(lib.n_lib):
        for c in range(chunks(lib, b)):
            page, nv = int(p.page_of[b, c]), int(p.n_valid[b, c])
            assert torch.equal(mass[page, :nv], p.slots[page, :nv, 1].float())


def test_masses_that_do_not_fit_are_refused():
    lib = library(74).reserve(3)
    P, N = lib.pages(1).slots.shape[:2]
    inj = LibraryInjector(TinyReader(D_M, 5).cuda(), interface(75), top_k=2)
    table, slots = lib.pages(1).page_of.clone(), lib.pages(1).slots.clone()
    for bad in (torch.zeros(P - 1, N, device="cuda"), torch.zeros(P, N, device="cuda", dtype=torch.float64),
                torch.zeros(N, P, device="cuda").t(), torch.zeros(P, N)):
        for call in (lambda: lib.fork([0], own_from=4, mass=bad), lambda: lib.compact(mass={1: bad})):
            with pytest.raises(ValueError, match="mass must be"):
                call()
    for bad in (torch.zeros(P + 1, N, device="cuda"), torch.zeros(P, N + 1, device="cuda"), torch.zeros(P, N, device="cuda").half()):
        with pytest.raises(ValueError, match="slot_mass of layer 3"):
            inj.load_library(lib, slot_mass={3: bad})
    with pytest.raises(ValueError, match="each layer"):
        lib.evict(torch.zeros(P, N, device="cuda"), 4, per_layer=True)
    assert torch.equal(lib.pages(1).page_of, table) and torch.equal(lib.pages(1).slots, slots)
    inj.detach()


@pytest.mark.parametrize("k", [1, 2])
@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("share", [False, True])
def test_rows_that_a_selector_drops_give_no_attention(k, T, share):
    """A LayerSelector's rows count in full at the layers that have a weight for them, not at the others."""
    g = torch.Generator(device="cuda").manual_seed(80)
    lib, itf = library(81), interface(82)
    sel = LayerSelector(D_M, LAYERS, k=k, alpha_init=0.05).cuda().requires_grad_(False)
    sel.u.weight.copy_(torch.randn(sel.u.weight.shape, generator=g, device="cuda"))
    inj = LibraryInjector(TinyReader(D_M, 5).cuda(), itf, top_k=2, selector=sel, share_pages=share)
    inj.load_library(lib)
    inj.record_mass = True
    h = torch.randn(3, T, D_M, generator=g, device="cuda")
    with torch.no_grad():
        for i, li in enumerate(LAYERS):
            inj._inject(h, li)
            w = sel.weights()[..., i]
            assert bool(((w > 0) & (w < 1)).any()) == (k == 2)
            close(inj.slot_mass[li], step(h, itf, lib, li, 2, live=w != 0)[1], 1e-4)
    assert abs(float(sum(m.sum() for m in inj.slot_mass.values())) - 3 * T * k) < 1e-3 * T
    inj.detach()


def test_a_library_of_its_own_and_the_last_tokens_attention():
    """record_mass on a Library that is not paged, alone and beside record_attn."""
    g = torch.Generator(device="cuda").manual_seed(83)
    unit = lambda n: torch.nn.functional.normalize(torch.randn(n, D_S, generator=g, device="cuda"), dim=-1).half().float()  # noqa: E731
    lib = Library([{"K": {0.25: unit(n), 0.75: unit(n)}} for n in (17, 30, 5, 24)], LAYERS, [0.25, 0.75])
    itf = interface(84)
    h = torch.randn(2, 5, D_M, generator=g, device="cuda")
    got, attn = [], []
    for mass, last in ((True, False), (True, True), (False, True)):
        inj = LibraryInjector(TinyReader(D_M, 5).cuda(), itf, top_k=2)
        inj.load_library(lib)
        inj.record_mass, inj.record_attn = mass, last
        with torch.no_grad():
            for li in LAYERS:
                inj._inject(h, li)
        got.append(inj.slot_mass)
        attn.append(inj.last_attn)
        inj.detach()
    paged = SimpleNamespace(pages=lambda li: lib.pages(li, DEV), n_chunks=lib.n_chunks)
    for li in LAYERS:
        close(got[0][li], step(h.view(1, 10, D_M), itf, paged, li, 2)[1], 1e-4)
        assert torch.equal(got[1][li], got[0][li]) and torch.equal(attn[1][li], attn[2][li])
    assert got[2] == {}
