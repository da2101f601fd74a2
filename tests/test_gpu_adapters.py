"""Projections with low-rank adapters against the formula in 64 bits.

Tolerance. The 3xF16 / 3xTF32 GEMM is held to 1e-5 of the largest output (as the plain projections are); the low-rank
term is a float32 dot of d_in products, at most d_in / 32 + 5 roundings long per lane, each 2^-24 of the running sum:
with random signs under sqrt(165) * 2^-24 < 1e-6 for d_in <= 5120, and the second product adds rank more. Twice 1e-5
holds both. 16-bit outputs are rounded once: half a step of the value besides."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = 2e-5
HALF = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def _inputs(dev, seed, R, rpa, n, rank, d_in, d_out, h_dtype, ad_dtype):
    g = torch.Generator(device=dev).manual_seed(seed)
    n_of = -(-R // rpa)
    of = torch.randint(0, n, (n_of,), generator=g, device=dev, dtype=torch.int32)
    if n_of > 2:
        of[1] = -1
    return dict(
        h=torch.randn(R, d_in, generator=g, device=dev).to(h_dtype), of=of,
        w=torch.randn(d_out, d_in, generator=g, device=dev) * d_in ** -0.5,
        bias=torch.randn(d_out, generator=g, device=dev) * 0.1,
        a=(torch.randn(n, rank, d_in, generator=g, device=dev) * d_in ** -0.5).to(ad_dtype),
        b=(torch.randn(n, d_out, rank, generator=g, device=dev) * 0.2).to(ad_dtype),
        scale=torch.rand(n, generator=g, device=dev) * 2)


def _ref(x, s, rpa, scale=True):
    """x W^T + s_a (x A^T) B^T in 64 bits, row by row."""
    x = x.double()
    y = x @ s["w"].double().t()
    for i, a in enumerate(s["of"].tolist()):
        if a >= 0:
            rows = slice(i * rpa, min(x.shape[0], (i + 1) * rpa))
            low = (x[rows] @ s["a"][a].double().t()) @ s["b"][a].double().t()
            y[rows] += low * (s["scale"][a].double() if scale else 1.0)
    return y


def _close(got, want, dtype):
    want = want.to(got.device)
    bound = TOL * want.abs().max() + HALF[dtype] * want.abs()
    assert ((got.double() - want).abs() <= bound).all(), float(((got.double() - want).abs() - bound).max())


# R, rows per adapter, adapters, rank, d_in, d_out: one token, odd ranks, a last group that is cut, prompts
SHAPES = [
    (1, 1, 1, 1, 64, 64),
    (5, 2, 3, 7, 260, 132),
    (64, 1, 64, 16, 1024, 512),
    (70, 1, 5, 33, 512, 1028),
    (300, 128, 2, 8, 520, 256),
    (257, 300, 4, 64, 256, 260),
    (96, 8, 7, 256, 136, 72),
    (33, 1, 2, 12, 70, 128),      # d_in that no tensor-core path takes
    (3, 1, 2, 4, 128, 6400),      # wider than one CTA's row
]


@pytest.mark.parametrize("R,rpa,n,rank,d_in,d_out", SHAPES)
@pytest.mark.parametrize("h_dtype,ad_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
                                              (torch.float16, torch.bfloat16), (torch.float32, torch.float16)])
def test_project_in(dev, R, rpa, n, rank, d_in, d_out, h_dtype, ad_dtype):
    from kv_skill_v2_b200 import ops
    s = _inputs(dev, R + rank, R, rpa, n, rank, d_in, d_out, h_dtype, ad_dtype)
    ad = ops.Adapters(s["a"], s["b"], s["scale"])
    more = dict(adapters=ad, adapter_of=s["of"], rows_per_adapter=rpa)
    x = s["h"].double()
    x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6)
    want = _ref(x, s, rpa) + s["bias"].double()
    q, _, _, _ = ops.project_in(s["h"], s["w"], s["bias"], l2=False, **more)
    _close(q, want, torch.float32)
    unit = want / (want.norm(dim=-1, keepdim=True) + 1e-6)
    prep = ops.weights_prep(s["w"]) if d_in % 8 == 0 else None
    q, _, _, _ = ops.project_in(s["h"], s["w"], s["bias"], w_prep=prep, **more)
    _close(q, unit, torch.float32)


@pytest.mark.parametrize("R,rpa,n,rank,d_in,d_out", SHAPES)
@pytest.mark.parametrize("h_dtype", [torch.bfloat16, torch.float32])
def test_project_out(dev, R, rpa, n, rank, d_in, d_out, h_dtype):
    from kv_skill_v2_b200 import ops
    s = _inputs(dev, 3 * R + rank, R, rpa, n, rank, d_in, d_out, torch.float32, torch.bfloat16)
    g = torch.Generator(device=dev).manual_seed(9)
    h = torch.randn(R, d_out, generator=g, device=dev).to(h_dtype)
    gate = torch.rand(R, generator=g, device=dev)
    prep = ops.weights_prep(s["w"]) if d_in % 8 == 0 else None
    delta, _, rel = ops.project_out(s["h"], s["w"], h, b_out=s["bias"], gate=gate, scale=1.5, want_rel=True,
                                    w_prep=prep, adapters=ops.Adapters(s["a"], s["b"]), adapter_of=s["of"],
                                    rows_per_adapter=rpa)
    want = (_ref(s["h"], s, rpa, scale=False) + s["bias"].double()) * gate.double()[:, None] * 1.5
    _close(delta, want, h_dtype)
    ratio = delta.double().norm(dim=-1) / (h.double().norm(dim=-1) + 1e-6)
    assert torch.allclose(rel.double(), ratio, rtol=1e-5)


def test_rows_without_an_adapter_are_the_plain_projection(dev):
    from kv_skill_v2_b200 import ops
    s = _inputs(dev, 5, 40, 1, 3, 8, 256, 128, torch.bfloat16, torch.bfloat16)
    none = torch.full_like(s["of"], -1)
    plain = ops.project_in(s["h"], s["w"])[0]
    got = ops.project_in(s["h"], s["w"], adapters=ops.Adapters(s["a"], s["b"]), adapter_of=none)[0]
    assert torch.equal(plain, got)


def test_gate_and_selector_are_not_adapted(dev):
    from kv_skill_v2_b200 import ops
    s = _inputs(dev, 6, 12, 1, 3, 8, 256, 128, torch.float32, torch.float32)
    g = torch.Generator(device=dev).manual_seed(2)
    gw, sw = torch.randn(256, generator=g, device=dev), torch.randn(8, 256, generator=g, device=dev)
    _, gate, rstd, z = ops.project_in(s["h"], s["w"], gate_w=gw, gate_b=0.3, sel_w=sw)
    _, gate2, rstd2, z2 = ops.project_in(s["h"], s["w"], gate_w=gw, gate_b=0.3, sel_w=sw,
                                         adapters=ops.Adapters(s["a"], s["b"], s["scale"]), adapter_of=s["of"])
    assert torch.equal(gate, gate2) and torch.equal(rstd, rstd2) and torch.equal(z, z2)


def test_non_finite_adapters_reach_only_their_rows(dev):
    from kv_skill_v2_b200 import ops
    s = _inputs(dev, 7, 20, 1, 4, 8, 256, 128, torch.bfloat16, torch.bfloat16)
    s["a"][2] = float("nan")
    s["b"][3] = float("inf")
    q = ops.project_in(s["h"], s["w"], adapters=ops.Adapters(s["a"], s["b"]), adapter_of=s["of"])[0]
    hit = (s["of"] == 2) | (s["of"] == 3)
    assert torch.isfinite(q[~hit]).all()
    assert hit.any() and not torch.isfinite(q[hit]).any(-1).all()


def test_index_past_the_last_adapter_is_flagged(dev):
    from kv_skill_v2_b200 import _native as N
    from kv_skill_v2_b200 import ops
    s = _inputs(dev, 8, 6, 1, 2, 4, 64, 64, torch.float32, torch.float32)
    of = torch.tensor([0, 1, 2, 7, -1, 0], dtype=torch.int32, device=dev)
    q = ops.project_in(s["h"], s["w"], adapters=ops.Adapters(s["a"], s["b"]), adapter_of=of)[0]
    assert ops.device_status(dev) & N.DEV_BADADAPTER
    assert torch.equal(q[2:5], ops.project_in(s["h"], s["w"])[0][2:5])


def test_refusals(dev):
    from kv_skill_v2_b200 import ops
    s = _inputs(dev, 8, 6, 1, 2, 4, 64, 64, torch.float32, torch.float32)
    ad = ops.Adapters(s["a"], s["b"])
    for bad in (dict(adapters=ad), dict(adapters=ad, adapter_of=s["of"][:5]),
                dict(adapters=ad, adapter_of=s["of"].long()),
                dict(adapters=ad, adapter_of=s["of"], rows_per_adapter=0),
                dict(adapters=ad, adapter_of=s["of"], rows_per_adapter=2),
                dict(adapters=ops.Adapters(s["a"], s["b"].half()), adapter_of=s["of"]),
                dict(adapters=ops.Adapters(s["a"][:, :, :60], s["b"]), adapter_of=s["of"]),
                dict(adapters=ops.Adapters(s["a"], s["b"], s["scale"][:1]), adapter_of=s["of"]),
                dict(adapters=ops.Adapters(s["a"].repeat(1, 65, 1), s["b"].repeat(1, 1, 65)), adapter_of=s["of"])):
        with pytest.raises(ValueError):
            ops.project_in(s["h"], s["w"], **bad)
    with pytest.raises(RuntimeError):
        ops.project_in(s["h"], s["w"], adapters=ops.Adapters(s["a"].cpu(), s["b"].cpu()), adapter_of=s["of"])


def test_captured_calls_with_their_own_workspaces(dev):
    from kv_skill_v2_b200 import ops
    s = _inputs(dev, 10, 16, 1, 4, 8, 256, 128, torch.bfloat16, torch.bfloat16)
    ad = ops.Adapters(s["a"], s["b"], s["scale"])
    prep = ops.weights_prep(s["w"])
    eager = ops.project_in(s["h"], s["w"], w_prep=prep, adapters=ad, adapter_of=s["of"])[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q1 = ops.project_in(s["h"], s["w"], w_prep=prep, adapters=ad, adapter_of=s["of"])[0]
        q2 = ops.project_in(s["h"], s["w"], w_prep=prep, adapters=ad, adapter_of=s["of"].flip(0).contiguous())[0]
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(q1, eager) and not torch.equal(q2, eager)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("R,rpa,n,rank,d_in,d_out", [(16, 16, 1, 1, 8, 64), (200, 70, 3, 33, 2056, 256),
                                                     (130, 17, 9, 40, 1000, 132), (64, 64, 1, 256, 5120, 128)])
def test_tiles_of_one_16_bit_type(dev, dtype, R, rpa, n, rank, d_in, d_out):
    """Rows and adapters of one 16-bit type, in tiles of rows that end inside a warp's 16 and ranks inside its 32."""
    from kv_skill_v2_b200 import ops
    s = _inputs(dev, 41, R, rpa, n, rank, d_in, d_out, dtype, dtype)
    ad = ops.Adapters(a=s["a"], b=s["b"], scale=s["scale"])
    q = ops.project_in(s["h"], s["w"], l2=False, rms=False, adapters=ad, adapter_of=s["of"], rows_per_adapter=rpa)[0]
    of = s["of"].long().repeat_interleave(rpa)[:R]
    low = torch.einsum("tk,trk->tr", s["h"].double(), s["a"].double()[of.clamp(min=0)])
    low = torch.einsum("tr,tnr->tn", low, s["b"].double()[of.clamp(min=0)]) * s["scale"].double()[of.clamp(min=0)][:, None]
    want = s["h"].double() @ s["w"].double().t() + low * (of >= 0)[:, None]
    assert float((q.double() - want).abs().max()) <= TOL * float(want.abs().max())


# Plans that would run all of d_in in one split, and are given one per 1280 columns: many output tiles, long rows.
FORCED = [(2048, 512, 4, 32, 2600, 2048), (1999, 512, 4, 7, 5120, 2048), (1100, 1, 5, 16, 2568, 4096)]


@pytest.mark.parametrize("R,rpa,n,rank,d_in,d_out", FORCED)
@pytest.mark.parametrize("prepared", [True, False])
@pytest.mark.parametrize("h_dtype", [torch.bfloat16, torch.float32])
def test_long_rows_with_many_output_tiles(dev, R, rpa, n, rank, d_in, d_out, prepared, h_dtype):
    """Both projections, called through the C entries with exactly the workspace that the query gives and a guard behind
    it. 2-norm: the accumulator loses up to 2^-23 of itself at each product it adds, always towards zero, half of that on
    average. 1280 columns are 80 steps of three products (3xF16; 160 steps as 3xTF32), over which the running sum grows
    like a square root, 2/3 of its end on average: 240 x 2^-24 x 2/3 = 1e-5 (2e-5). The loss is in proportion to the
    columns of a split, so rows without an adapter are at most 0.6 as far off as in the plain projection's one split of
    them all (a third or a quarter, and the operands' own 1e-7)."""
    from kv_skill_v2_b200 import _native as N
    from kv_skill_v2_b200 import ops
    s = _inputs(dev, R + d_in, R, rpa, n, rank, d_in, d_out, h_dtype, torch.bfloat16)
    s["of"][0] = -1
    prep = ops.weights_prep(s["w"]) if prepared else None
    want = _ref(s["h"], s, rpa)
    y = torch.empty(R, d_out, device=dev)
    ptr, st = ops._ptr, ops._stream(dev)
    adapt = (ptr(s["a"]), ptr(s["b"]), N.BF16, ptr(s["scale"]), n, rank, ptr(s["of"]), rpa)
    guard = 32 << 20

    def workspace(size):
        assert size > 0
        ws = torch.full((size + guard,), 0x5A, dtype=torch.uint8, device=dev)
        return ws, size

    def judge(ws, size):
        torch.cuda.synchronize()
        assert (ws[size:] == 0x5A).all()
        assert float((y.double() - want).norm() / want.norm()) <= (1e-5 if prepared else 2e-5)
        _close(y, want, torch.float32)

    ws, size = workspace(N.lib().xencb_project_in_adapted_workspace(R, d_in, d_out, rank))
    N.call("xencb_project_in_adapted", ptr(s["h"]), ops._hdt(s["h"], "h"), R, d_in, ptr(s["w"]), ptr(prep), None, d_out, 0,
           None, 0.0, None, None, None, 0, 1e-6, ptr(y), None, None, None, *adapt, ptr(ws), size, st)
    judge(ws, size)
    if prepared:
        plain = ops.project_in(s["h"], s["w"], w_prep=prep, rms=False, l2=False)[0].double()
        bare = s["h"].double() @ s["w"].double().t()
        none = torch.full_like(s["of"], -1)
        split = ops.project_in(s["h"], s["w"], w_prep=prep, rms=False, l2=False, adapter_of=none, rows_per_adapter=rpa,
                               adapters=ops.Adapters(s["a"], s["b"], s["scale"]))[0].double()
        assert float((split - bare).norm()) <= 0.6 * float((plain - bare).norm())
    if h_dtype == torch.float32:
        y.fill_(7.0)
        zero = torch.zeros(R, d_out, device=dev)
        ws, size = workspace(N.lib().xencb_project_out_adapted_workspace(R, d_in, d_out, rank))
        N.call("xencb_project_out_adapted", ptr(s["h"]), R, d_in, ptr(s["w"]), ptr(prep), None, d_out, 1.0, None, None,
               None, 0.0, None, None, ptr(zero), N.F32, ptr(y), None, None, *adapt, ptr(ws), size, st)
        judge(ws, size)
    assert ops.device_status(dev) == 0


@pytest.mark.parametrize("R,d_in,d_out", [(2048, 5120, 2048), (1999, 2600, 2048), (64, 2048, 4096), (5, 3440, 1544),
                                          (1, 4096, 2048), (130, 1280, 4096)])
def test_only_the_large_products_lose_to_the_accumulator(dev, R, d_in, d_out):
    """2-norm of float32 results with prepared weights. hi*hi alone is summed in the accumulator that holds the result, 80
    steps at most in a split of 1280 columns, each of which loses half of 2^-23 of a running sum on average, 2/3 of its end
    (it grows like a square root): 80 x 2^-24 x 2/3 = 3.2e-6. The operands' 22 bits and the float32 additions stay below
    2e-7 beside it."""
    from kv_skill_v2_b200 import ops
    s = _inputs(dev, R + d_in, R, 1, 3, 4, d_in, d_out, torch.float32, torch.bfloat16)
    x = s["h"] / s["h"].norm(dim=-1, keepdim=True)
    want = _ref(x, s, 1)
    more = dict(w_prep=ops.weights_prep(s["w"]), adapters=ops.Adapters(s["a"], s["b"], s["scale"]), adapter_of=s["of"])
    steps = min(80, -(-d_in // 16))
    for got in (ops.project_out(x, s["w"], torch.zeros(R, d_out, device=dev), **more)[0],
                ops.project_in(x, s["w"], rms=False, l2=False, **more)[0]):
        assert float((got.double() - want).norm() / want.norm()) <= steps * 2.0 ** -24 * 2 / 3 + 2e-7
