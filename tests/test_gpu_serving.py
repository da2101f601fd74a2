"""Many requests over shared documents, as a server runs them: Libraries forked for requests, their pages compacted, the
batch read with every shared page fetched once, and an adapter of its own per request -- against the definition in 64
bits, and against itself after pages moved (results do not depend on where a page lies)."""

from __future__ import annotations

import pytest
import torch

from tests._fixtures import TOL, TinyReader, rel_err

pytestmark = pytest.mark.gpu

D_M, D_S, LAYER = 96, 64, 1


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def _library(dev, seed=0, n_lib=3, C=5, rows=20, ragged=True, untied=False):
    from kv_skill_v2_b200 import PagedLibrary
    g = torch.Generator(device=dev).manual_seed(seed)
    pools = {li: torch.nn.functional.normalize(torch.randn(n_lib * C, rows, D_S, generator=g, device=dev), dim=-1).half()
             for li in (LAYER, 3)}
    vals = {li: torch.randn_like(p) for li, p in pools.items()} if untied else None
    page_of = torch.randperm(n_lib * C, generator=g, device=dev).view(n_lib, C).to(torch.int32)
    n_valid = torch.randint(1, rows + 1, (n_lib, C), generator=g, device=dev, dtype=torch.int32)
    nco = torch.tensor([C, C - 2, C - 1], dtype=torch.int32, device=dev)[:n_lib] if ragged else None
    return PagedLibrary.from_pool(pools, page_of, n_valid, nco, layer_vslots=vals)


def _content(lib, li, row, c):
    p = lib.pages(li)
    return p.slots[int(p.page_of[row, c]), :int(p.n_valid[row, c])]


def _chunks(lib, row):
    nco = lib.pages(LAYER).n_chunks_of
    return lib.n_chunks if nco is None else int(nco[row])


@pytest.mark.parametrize("ragged,untied", [(False, False), (True, False), (True, True)])
def test_fork_drop_compact_keep_every_library(dev, ragged, untied):
    lib = _library(dev, ragged=ragged, untied=untied)
    before = {(li, r, c): _content(lib, li, r, c).clone() for li in lib.layers for r in range(3)
              for c in range(_chunks(lib, r))}
    with pytest.raises(RuntimeError, match="free pages too few"):
        lib.fork([0, 0, 0, 0, 0, 0, 0, 0], own_from=0)
    lib = lib.reserve(8)
    parents, own = [0, 1, 0, 2], [5, 2, 3, 4]
    lib = lib.fork(parents, own)
    assert lib.n_lib == 7
    origin = [0, 1, 2] + parents

    def same(lib, origin):
        for i, o in enumerate(origin):
            for li in lib.layers:
                for c in range(_chunks(lib, i)):
                    assert torch.equal(_content(lib, li, i, c), before[li, o, c])

    same(lib, origin)
    t = lib.pages(LAYER).page_of
    taken = {int(t[r, c]) for r in range(3) for c in range(_chunks(lib, r))}  # (entries past a Library's chunks name nothing)
    for i, (par, o) in enumerate(zip(parents, own)):
        n = _chunks(lib, par)
        assert torch.equal(t[3 + i, :min(o, n)], t[par, :min(o, n)])
        assert not set(t[3 + i, o:n].tolist()) & taken
    # rewriting a fork's own chunk reaches nobody else
    p = lib.pages(LAYER)
    mine = int(p.page_of[5, 4]) if _chunks(lib, 5) == 5 else int(p.page_of[5, 3])
    kept = p.slots[mine].clone()
    p.slots[mine].fill_(0.25)
    same(lib.select([0, 1, 2, 3, 4, 6]), [0, 1, 2, 0, 1, 2])
    p.slots[mine].copy_(kept)
    lib = lib.drop([1, 4])
    lib, n = lib.compact()
    origin = [0, 2, 0, 0, 2]
    same(lib, origin)
    live = set()
    for i in range(lib.n_lib):
        live |= set(lib.pages(LAYER).page_of[i, :_chunks(lib, i)].tolist())
    assert live == set(range(n))
    with pytest.raises(ValueError):
        lib.select([9])
    with pytest.raises(ValueError):
        lib.fork([0], own_from=[1, 2])


def _reference(h, W_in, W_out, lib, li, ad_in, ad_out, of, top_k, route_temp, read_temp):
    """delta of every token in 64 bits (single linear maps, no gate)."""
    out = torch.zeros(h.shape, dtype=torch.float64, device=h.device)
    p = lib.pages(li)
    for b in range(h.shape[0]):
        x = h[b].double()
        x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6)
        q = x @ W_in.double()
        a = int(of[b])
        if a >= 0:
            q = q + ad_in.scale[a].double() * (x @ ad_in.a[a].double().t()) @ ad_in.b[a].double().t()
        q = q / (q.norm(dim=-1, keepdim=True) + 1e-6)
        n = _chunks(lib, b)
        logits = q @ p.S[b, :n].double().t() * route_temp
        k = top_k if 0 < top_k < n else n
        top, idx = logits.topk(k, dim=-1)
        w = torch.softmax(top, -1)
        r = torch.zeros(q.shape, dtype=torch.float64, device=h.device)
        for t in range(q.shape[0]):
            for j in range(k):
                K = _content(lib, li, b, int(idx[t, j])).double()
                r[t] += w[t, j] * (torch.softmax(read_temp * K @ q[t], 0) @ K)
        y = r @ W_out.double()
        if a >= 0:
            y = y + ad_out.scale[a].double() * (r @ ad_out.a[a].double().t()) @ ad_out.b[a].double().t()
        out[b] = y
    return out


@pytest.mark.parametrize("T", [1, 5, 70])
@pytest.mark.parametrize("graphs", [True, False])
def test_requests_with_adapters_over_forked_libraries(dev, T, graphs):
    from kv_skill_v2_b200 import LibraryInjector, ops
    from kv_skill_v2_b200.interface import LinearInterface
    g = torch.Generator(device=dev).manual_seed(3)
    W_in = torch.randn(D_M, D_S, generator=g, device=dev) * D_M ** -0.5
    W_out = torch.randn(D_S, D_M, generator=g, device=dev) * 0.2
    whole = _library(dev, seed=4).reserve(6).fork([0, 0, 1, 2], own_from=[4, 3, 2, 9])
    lib = whole.select([3, 4, 5, 6, 0])
    B = lib.n_lib
    of = torch.tensor([2, -1, 0, 2, 1], dtype=torch.int32, device=dev)

    def adapters(d_in, d_out):
        return ops.Adapters(a=torch.randn(3, 4, d_in, generator=g, device=dev) * d_in ** -0.5,
                            b=torch.randn(3, d_out, 4, generator=g, device=dev) * 0.2,
                            scale=torch.rand(3, generator=g, device=dev) + 0.5)

    ad_in, ad_out = adapters(D_M, D_S), adapters(D_S, D_M)
    reader = TinyReader(D_M, 4).to(dev)
    itf = LinearInterface(W_in, W_out, [LAYER]).to(dev).requires_grad_(False)
    inj = LibraryInjector(reader, itf, top_k=2, cuda_graphs=graphs, share_pages=True)
    inj.load_library(lib)
    inj.set_adapters(ad_in, ad_out, of)
    h = torch.randn(B, T, D_M, generator=g, device=dev)
    with torch.no_grad():
        want = _reference(h, W_in, W_out, lib, LAYER, ad_in, ad_out, of, 2, 10.0, 12.0)
        for _ in range(3):  # eager, captured, replayed
            got, _ = inj._inject(h, LAYER)
            assert rel_err(got - h, want) <= TOL
        first = got.clone()
        # another assignment of adapters, in place and then as another tensor
        of.copy_(of.flip(0))
        want2 = _reference(h, W_in, W_out, lib, LAYER, ad_in, ad_out, of, 2, 10.0, 12.0)
        assert rel_err(inj._inject(h, LAYER)[0] - h, want2) <= TOL
        inj.set_adapters(ad_in, ad_out, of.flip(0).contiguous())
        assert torch.equal(inj._inject(h, LAYER)[0], first)
        # the pages move: the same bits
        moved, _ = whole.compact()
        inj.load_library(moved.select([3, 4, 5, 6, 0]))
        assert torch.equal(inj._inject(h, LAYER)[0], first)
        # without adapters and page sharing: the path of read_decode
        inj.set_adapters()
        inj.share_pages = False
        plain, _ = inj._inject(h, LAYER)
        none = torch.full((B,), -1, dtype=torch.int32, device=dev)
        ref = _reference(h, W_in, W_out, moved.select([3, 4, 5, 6, 0]), LAYER, ad_in, ad_out, none, 2, 10.0, 12.0)
        assert rel_err(plain - h, ref) <= TOL
    assert ops.device_status(dev) == 0
    inj.detach()


def test_adapter_refusals(dev):
    from kv_skill_v2_b200 import LibraryInjector, make_interface, ops
    reader = TinyReader(D_M, 4).to(dev)
    low = make_interface(D_M, D_S, [LAYER], rank=8).to(dev).requires_grad_(False)
    inj = LibraryInjector(reader, low, top_k=2)
    inj.load_library(_library(dev, ragged=False))
    ad = ops.Adapters(a=torch.zeros(1, 2, D_M, device=dev), b=torch.zeros(1, D_S, 2, device=dev))
    with pytest.raises(ValueError):
        inj.set_adapters(ad)
    inj.set_adapters(ad, None, torch.zeros(3, dtype=torch.int32, device=dev))
    h = torch.randn(3, 1, D_M, device=dev)
    with torch.no_grad(), pytest.raises(NotImplementedError):
        inj._inject(h, LAYER)
    inj.set_adapters(ad, None, torch.zeros(2, dtype=torch.int32, device=dev))
    with torch.no_grad(), pytest.raises(ValueError):
        inj._inject(h, LAYER)
    inj.detach()


def test_captured_steps_of_earlier_adapters_do_not_pile_up(dev):
    """Requests join and leave: every step brings other adapter tensors."""
    from kv_skill_v2_b200 import LibraryInjector, ops
    from kv_skill_v2_b200.interface import LinearInterface
    g = torch.Generator(device=dev).manual_seed(8)
    W_in = torch.randn(D_M, D_S, generator=g, device=dev) * D_M ** -0.5
    W_out = torch.randn(D_S, D_M, generator=g, device=dev) * 0.2
    lib = _library(dev, seed=9, ragged=False)
    itf = LinearInterface(W_in, W_out, [LAYER]).to(dev).requires_grad_(False)
    inj = LibraryInjector(TinyReader(D_M, 4).to(dev), itf, top_k=2)
    inj.load_library(lib)
    h = torch.randn(3, 1, D_M, generator=g, device=dev)
    kept, sizes = [], []
    with torch.no_grad():
        inj._inject(h, LAYER)
        plain = inj._inject(h, LAYER)[0]
        for step in range(24):
            ad = ops.Adapters(a=torch.randn(2, 4, D_M, generator=g, device=dev) * D_M ** -0.5,
                              b=torch.randn(2, D_S, 4, generator=g, device=dev) * 0.2, scale=torch.ones(2, device=dev))
            of = torch.randint(-1, 2, (3,), generator=g, device=dev, dtype=torch.int32)
            inj.set_adapters(ad, None, of)
            kept.append(ad)  # (the caller keeps them: no address comes back)
            for _ in range(2):
                got = inj._inject(h, LAYER)[0]
            want = _reference(h, W_in, W_out, lib, LAYER, ad, ops.Adapters(a=torch.zeros(2, 1, D_S, device=dev),
                              b=torch.zeros(2, D_M, 1, device=dev), scale=torch.zeros(2, device=dev)), of, 2, 10.0, 12.0)
            assert rel_err(got - h, want) <= TOL
            sizes.append(len(inj._graphs))
        inj.set_adapters()
        assert torch.equal(inj._inject(h, LAYER)[0], plain)
    assert max(sizes) <= 8 and max(sizes[12:]) == max(sizes[:12]), sizes
    inj.detach()


@pytest.mark.parametrize("top_k", [0, 2])
def test_a_prompt_over_shared_pages_keeps_no_workspace(dev, monkeypatch, top_k):
    """A shared read above the workspace limits runs in slices and is not captured; the rows are the same."""
    import kv_skill_v2_b200.injector as module
    from kv_skill_v2_b200 import LibraryInjector, ops
    from kv_skill_v2_b200.interface import LinearInterface
    g = torch.Generator(device=dev).manual_seed(12)
    W_in = torch.randn(D_M, D_S, generator=g, device=dev) * D_M ** -0.5
    W_out = torch.randn(D_S, D_M, generator=g, device=dev) * 0.2
    lib = _library(dev, seed=13, ragged=False)
    inj = LibraryInjector(TinyReader(D_M, 4).to(dev), LinearInterface(W_in, W_out, [LAYER]).to(dev).requires_grad_(False),
                          top_k=top_k, share_pages=True)
    inj.load_library(lib)
    h = torch.randn(3, 200, D_M, generator=g, device=dev)
    with torch.no_grad():
        whole = inj._inject(h, LAYER)[0]
        assert torch.equal(inj._inject(h, LAYER)[0], whole) and len(inj._graphs) == 1
        need = ops.shared_workspace(lib.pages(LAYER), 600, top_k or 5)
        monkeypatch.setattr(module, "_GRAPH_WORKSPACE", need - 1)
        monkeypatch.setattr(ops.read_shared, "__kwdefaults__", {**ops.read_shared.__kwdefaults__, "max_workspace": need // 4})
        inj._graphs.clear()
        before = torch.cuda.memory_allocated()
        for _ in range(3):
            again = inj._inject(h, LAYER)[0]
        assert torch.equal(again, whole) and not inj._graphs
        torch.cuda.synchronize()
        assert torch.cuda.memory_allocated() - before <= 3 * h.numel() * 4
        inj._inject(h[:, :20].contiguous(), LAYER)
        assert len(inj._graphs) == 1  # (a smaller step is captured as before)
    inj.detach()


def _merged(itf, ad_in, ad_out, a):
    """A copy of the interface whose maps hold adapter a (negative: none)."""
    import copy
    m = copy.deepcopy(itf)
    if a >= 0:
        with torch.no_grad():
            m.A.weight += ad_in.scale[a] * ad_in.b[a] @ ad_in.a[a]
            m.B.weight += ad_out.scale[a] * ad_out.b[a] @ ad_out.a[a]
    return m


def _model_interface(dev, g, layers):
    from kv_skill_v2_b200 import ModelInterface
    itf = ModelInterface(D_M, D_S, layers)
    with torch.no_grad():
        itf.A.weight.copy_(torch.randn(D_S, D_M, generator=g, device=dev) * D_M ** -0.5)
        itf.B.weight.copy_(torch.randn(D_M, D_S, generator=g, device=dev) * 0.2)
        itf.gate_w.copy_(torch.randn(D_M, generator=g, device=dev) * 0.1)
        itf.gate_b.copy_(torch.randn(len(layers), generator=g, device=dev))
        itf.log_gain.copy_(torch.randn(len(layers), generator=g, device=dev) * 0.3)
    ads = [ops_adapters(dev, g, d_in, d_out) for d_in, d_out in ((D_M, D_S), (D_S, D_M))]
    return itf.to(dev).requires_grad_(False), ads


def ops_adapters(dev, g, d_in, d_out):
    from kv_skill_v2_b200 import ops
    return ops.Adapters(a=torch.randn(3, 4, d_in, generator=g, device=dev) * d_in ** -0.5,
                        b=torch.randn(3, d_out, 4, generator=g, device=dev) * 0.2,
                        scale=torch.rand(3, generator=g, device=dev) + 0.5)


@pytest.mark.parametrize("selector", [False, True])
@pytest.mark.parametrize("T", [1, 90])
def test_a_hooked_reader_with_adapters_is_one_of_merged_weights(dev, T, selector):
    """ModelInterface (gate, gain) at two depths, with and without a LayerSelector, over forks that share pages: each
    request's tokens come out as from a reader whose interface holds its adapter in the weights."""
    from kv_skill_v2_b200 import LayerSelector, LibraryInjector, ops
    g = torch.Generator(device=dev).manual_seed(21)
    layers = [LAYER, 3]
    itf, (ad_in, ad_out) = _model_interface(dev, g, layers)
    lib = _library(dev, seed=22).reserve(4).fork([0, 2, 0], own_from=[4, 3, 9]).select([3, 4, 5, 1])
    sel = None
    if selector:
        sel = LayerSelector(D_M, layers, k=1, alpha_init=0.05).to(dev).requires_grad_(False)
        sel.u.weight.copy_(torch.randn(sel.u.weight.shape, generator=g, device=dev))
    of = torch.tensor([1, -1, 2, 1], dtype=torch.int32, device=dev)
    reader = TinyReader(D_M, 5).to(dev).eval().requires_grad_(False)
    x = torch.randn(4, T, D_M, generator=g, device=dev)
    inj = LibraryInjector(reader, itf, top_k=2, selector=sel, share_pages=True)
    inj.load_library(lib)
    inj.set_adapters(ad_in, ad_out, of)
    with torch.no_grad():
        for _ in range(2):
            got = reader(x)
        inj.detach()
        bare = reader(x)
        for b in range(4):
            one = LibraryInjector(reader, _merged(itf, ad_in, ad_out, int(of[b])), top_k=2, selector=sel)
            one.load_library(lib.select([b]))
            want = reader(x[b:b + 1])
            one.detach()
            assert rel_err(got[b:b + 1] - bare[b:b + 1], want - bare[b:b + 1]) <= 2 * TOL  # (both are within TOL)
    assert ops.device_status(dev) == 0


def test_a_single_skill_with_adapters_is_one_of_merged_weights(dev):
    from kv_skill_v2_b200 import KVSkill, XEncInjector
    g = torch.Generator(device=dev).manual_seed(23)
    itf, (ad_in, ad_out) = _model_interface(dev, g, [LAYER])
    K = torch.nn.functional.normalize(torch.randn(50, D_S, generator=g, device=dev), dim=-1).half().float()
    reader = TinyReader(D_M, 4).to(dev)
    h = torch.randn(3, 7, D_M, generator=g, device=dev)
    of = torch.tensor([2, -1, 0], dtype=torch.int32, device=dev)

    def branch(interface, rows, **adapters):
        inj = XEncInjector(reader, interface)
        inj.load(KVSkill({LAYER: K}, {LAYER: K}, D_S))
        if adapters:
            inj.set_adapters(**adapters)
        with torch.no_grad():
            out = inj._branch(rows, LAYER)
        inj.detach()
        return out

    got = branch(itf, h, adapters_in=ad_in, adapters_out=ad_out, adapter_of=of)
    for b in range(3):
        want = branch(_merged(itf, ad_in, ad_out, int(of[b])), h[b:b + 1])
        assert rel_err(got[b:b + 1], want) <= 2 * TOL
