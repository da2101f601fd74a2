"""The projections in 8-bit floating point against their definition in 64 bits: the same rounding to e4m3 with a power of
two per (row, 128 columns), then the product, 1/rms, bias, L2 norm, gate and epilogue exactly.

Tolerance: the operands are the same numbers on both sides (the quantisation is exact up to its own rounding, which is
part of the definition), so what differs is float32 accumulation: the house bound for float32 results, 2e-5 of the
largest value; 16-bit results add half a unit in the last place."""

from __future__ import annotations

import math

import pytest
import torch

from kv_skill_v2_b200 import _native as N
from kv_skill_v2_b200 import ops

pytestmark = pytest.mark.gpu
TOL = 2e-5


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows(n, k, seed, spread=3, dtype=torch.float32):
    """Rows whose blocks of 128 columns have magnitudes 2^-spread .. 2^spread, another for every row and block."""
    g = gen(seed)
    nb = -(-k // 128)
    e = torch.randint(-spread, spread + 1, (n, nb), generator=g, device="cuda")
    x = torch.randn(n, k, generator=g, device="cuda") * torch.exp2(e.float()).repeat_interleave(128, 1)[:, :k]
    return x.to(dtype)


def quantised(x):
    """(e4m3 values [n, 128 B] float64, exponents [n, B]) of x [n, k] from comparisons with powers of two."""
    n, k = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -k % 128)).view(n, -1, 128)
    mx = x.abs().amax(-1)
    e = torch.full(mx.shape, -127, device=x.device)
    for t in range(-127, 127):  # the smallest e with mx <= 448 2^e
        e += (mx > 448.0 * 2.0 ** t).to(e.dtype)
    e = torch.where(mx == 0, 0, e)
    v = x / torch.exp2(e.double())[..., None]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).view(n, -1), e


def values(x):
    v, e = quantised(x)
    return (v.view(v.shape[0], -1, 128) * torch.exp2(e.double())[..., None]).view(v.shape[0], -1)[:, : x.shape[1]]


def rel(got, want):
    return float((got.double() - want).abs().max() / want.abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 8), (5, 127), (7, 128), (2, 129), (130, 516), (33, 4096)])
def test_weights_fp8_bits(n, k, dtype):
    x = rows(n, k, 1, spread=10 if dtype == torch.float16 else 30, dtype=dtype)
    if n > 2:
        x[1] = 0
    w = ops.weights_fp8(x)
    v, e = quantised(x)
    assert w.shape == (n, k) and tuple(w.w.shape) == (n, -(-k // 128) * 128)
    assert torch.equal(w.scale.int() - 127, e.int())
    assert torch.equal(w.w.double(), v)


def test_weights_fp8_borders():
    # 448 is the largest value of e4m3, 448 + one step the first that takes the next power of two; ties round to even
    x = torch.zeros(6, 128, device="cuda")
    x[0, 0], x[1, 0], x[2, 0] = 448.0, 448.00003, 224.0
    x[3, :3] = torch.tensor([448.0, 17.0, 19.0])     # 16 .. 32 in steps of 2: 17 and 19 lie between
    x[4, :2] = torch.tensor([3.0e38, -1.0])
    x[5, :2] = torch.tensor([1.0e-38, 0.0])
    w = ops.weights_fp8(x)
    assert w.scale[:, 0].tolist()[:3] == [127, 128, 126]
    assert w.w[3].float()[:3].tolist() == [448.0, 16.0, 20.0]
    v, e = quantised(x)
    assert torch.equal(w.scale.int() - 127, e.int()) and torch.equal(w.w.double(), v)


def test_weights_fp8_not_finite():
    x = rows(3, 256, 2)
    x[0, 5], x[1, 200] = float("inf"), float("nan")
    w = ops.weights_fp8(x)
    assert w.w[0].float().isnan().nonzero().view(-1).tolist() == [5]
    assert w.w[1].float().isnan().nonzero().view(-1).tolist() == [200]
    y = x.clone()
    y[0, 5], y[1, 200] = 0, 0
    v, e = quantised(y)
    keep = ~w.w.float().isnan()
    assert torch.equal(w.scale.int() - 127, e.int()) and torch.equal(w.w.double()[keep], v[keep])


@pytest.mark.parametrize("R,d_in,d_out,dtype", [
    (1, 4096, 2048, torch.bfloat16), (1, 8, 4, torch.float32), (2, 130, 132, torch.float16), (5, 1000, 328, torch.float32),
    (63, 520, 256, torch.bfloat16), (64, 4096, 2048, torch.float16), (65, 777, 260, torch.float32),
    (127, 384, 516, torch.bfloat16), (128, 1024, 512, torch.float32), (129, 1024, 1024, torch.bfloat16),
    (300, 512, 2048, torch.float32), (513, 2048, 384, torch.float16), (1000, 5120, 640, torch.bfloat16),
    (2048, 5120, 2048, torch.bfloat16), (1111, 700, 2052, torch.float32), (19000, 130, 132, torch.float16),
    (4, 40000, 8, torch.float32), (200, 12000, 16, torch.bfloat16), (3, 256, 7000, torch.float32),
    # 2, 3, 5, 6, 7 and 8 tiles of 256 features, several turns of a CTA, odd ends
    (12345, 136, 260, torch.bfloat16), (9000, 130, 516, torch.float32), (4100, 1000, 1156, torch.float16),
    (5000, 264, 1284, torch.bfloat16), (6001, 72, 1796, torch.float32), (2500, 512, 1800, torch.bfloat16)])
def test_project_in(R, d_in, d_out, dtype):
    h, W = rows(R, d_in, 3, dtype=dtype), rows(d_out, d_in, 4) * d_in ** -0.5
    g = gen(5)
    b, gate_w = torch.randn(d_out, generator=g, device="cuda"), torch.randn(d_in, generator=g, device="cuda") * 0.02
    sel_w = torch.randn(3, d_in, generator=g, device="cuda") * 0.02
    w8 = ops.weights_fp8(W)
    q, gate, rstd, z = ops.project_in(h, w8, b, gate_w=gate_w, gate_b=0.3, sel_w=sel_w)
    hd = h.double()
    rs = 1 / torch.sqrt(hd.pow(2).mean(-1, keepdim=True) + 1e-6)
    y = values(h) @ values(W).t() * rs + b.double()
    assert rel(q, y / (y.norm(dim=-1, keepdim=True) + 1e-6)) < TOL
    # what does not go through the 8-bit product is what it is with a float32 weight, bit for bit
    _, gate32, rstd32, z32 = ops.project_in(h, W, b, gate_w=gate_w, gate_b=0.3, sel_w=sel_w)
    assert torch.equal(gate, gate32) and torch.equal(rstd, rstd32) and torch.equal(z, z32)
    # without a selector calls of many rows take 1/rms and the gate in another order of float32 sums
    q2, gate2, rstd2, _ = ops.project_in(h, w8, b, gate_w=gate_w, gate_b=0.3)
    assert rel(q2, y / (y.norm(dim=-1, keepdim=True) + 1e-6)) < TOL
    assert rel(rstd2, rs[:, 0]) < 1e-6
    assert rel(gate2, torch.sigmoid((hd @ gate_w.double()) * rs[:, 0] + 0.3)) < TOL
    raw = ops.project_in(h, w8, rms=False, l2=False)[0]
    assert rel(raw, values(h) @ values(W).t()) < TOL


@pytest.mark.parametrize("R,d_in,d_out,dtype", [
    (1, 2048, 4096, torch.bfloat16), (5, 328, 1000, torch.float32), (64, 2048, 4096, torch.float16), (70, 96, 512, torch.float32),
    (128, 640, 260, torch.bfloat16), (257, 2048, 1024, torch.bfloat16), (700, 1032, 512, torch.float32),
    (2, 128, 8192, torch.float32), (2048, 2048, 4096, torch.bfloat16), (1500, 520, 2052, torch.float16),
    (10001, 264, 260, torch.float32)])
def test_project_out(R, d_in, d_out, dtype):
    r, W = rows(R, d_in, 6), rows(d_out, d_in, 7) * d_in ** -0.5
    g = gen(8)
    h = torch.randn(R, d_out, generator=g, device="cuda").to(dtype)
    gate, mask = torch.rand(R, generator=g, device="cuda"), (torch.rand(R, generator=g, device="cuda") < 0.7).float()
    b = torch.randn(d_out, generator=g, device="cuda")
    log_gain = torch.tensor([0.25], device="cuda")
    w8 = ops.weights_fp8(W)
    eps = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    d = 0.5 * torch.exp(log_gain.double()) * gate.double()[:, None] * (values(r) @ values(W).t() + b.double())
    delta, _, _ = ops.project_out(r, w8, h, b_out=b, scale=0.5, log_scale=log_gain, gate=gate)
    assert delta.dtype == dtype and rel(delta, d) < TOL + eps
    # the hook's epilogue: position mask, h + delta (rounded twice: delta, then the sum), the mag term
    h_new = torch.empty_like(h)
    _, h_new, mag = ops.project_out(r, w8, h, b_out=b, scale=0.5, log_scale=log_gain, gate=gate, pos_mask=mask,
                                    want_delta=False, h_out=h_new, want_rel=True)
    dm = d * mask.double()[:, None]
    assert float((h_new.double() - (h.double() + dm)).abs().max() / (h.double() + dm).abs().max()) < TOL + 2 * eps
    want = dm.norm(dim=-1) / (h.double().norm(dim=-1) + 1e-6)
    assert float((mag.double() - want).abs().max() / want.abs().max()) < TOL + eps
    # a LayerSelector's matched norm
    sel_w = torch.rand(R, generator=g, device="cuda")
    delta, _, _ = ops.project_out(r, w8, h, b_out=b, gate=gate, sel_w=sel_w, log_alpha=-0.5)
    e = gate.double()[:, None] * (values(r) @ values(W).t() + b.double())
    hd = h.double()
    matched = e / (e.norm(dim=-1, keepdim=True) / (hd.norm(dim=-1, keepdim=True) + 1e-6) + 1e-6)
    matched = matched * math.exp(-0.5) * sel_w.double()[:, None]
    assert rel(delta, matched) < TOL + eps


@pytest.mark.parametrize("R", [3, 8, 9, 20, 100, 129, 200])
def test_many_blocks_and_no_split(R):
    # 94 blocks in one split: several rounds of the ring's blocks, many words of scale factors
    n, k = 148 * 128 - 4, 12000
    h, w8 = rows(R, k, 40, dtype=torch.bfloat16), ops.weights_fp8(W := rows(n, k, 41) * k ** -0.5)
    assert rel(ops.project_in(h, w8, rms=False, l2=False)[0], values(h) @ values(W).t()) < TOL


@pytest.mark.parametrize("R", [1, 50, 2000])
def test_a_weight_is_read_after_it_is_written(R):
    # the products load weights before they wait for the launch before theirs: never before the weight is there
    h, Ws = rows(R, 2048, 42, dtype=torch.bfloat16), [rows(4096, 2048, s) for s in (43, 44)]
    want = [ops.project_in(h, ops.weights_fp8(W))[0] for W in Ws]
    w8 = ops.weights_fp8(Ws[0])
    torch.cuda.synchronize()
    for i in range(20):
        at = w8.w.data_ptr()
        del w8
        w8 = ops.weights_fp8(Ws[i & 1])  # the same memory as the weight before
        q = ops.project_in(h, w8)[0]
        assert w8.w.data_ptr() == at and torch.equal(q, want[i & 1])


def test_a_row_that_is_not_finite_is_alone():
    h, W = rows(70, 512, 9), rows(256, 512, 10)
    w8 = ops.weights_fp8(W)
    clean = ops.project_in(h, w8, rms=False, l2=False)[0]
    h2 = h.clone()
    h2[7, 100], h2[66, 3] = float("inf"), float("nan")
    out = ops.project_in(h2, w8, rms=False, l2=False)[0]
    bad = torch.zeros(70, dtype=torch.bool, device="cuda")
    bad[[7, 66]] = True
    assert bool(out[bad].isnan().all()) and torch.equal(out[~bad], clean[~bad])


def test_strided_rows_unaligned_rows_and_zeros():
    W = rows(64, 300, 11)
    w8 = ops.weights_fp8(W)
    big = rows(20, 700, 12)
    h = big[::2, 100:400]                      # neither dense nor contiguous
    assert rel(ops.project_in(h, w8, rms=False, l2=False)[0], values(h) @ values(W).t()) < TOL
    flat = torch.zeros(1 + 4 * 300, device="cuda")
    flat[1:] = rows(4, 300, 13).view(-1)
    h = flat[1:].view(4, 300)                  # 4-byte aligned only
    assert rel(ops.project_in(h, w8, rms=False, l2=False)[0], values(h) @ values(W).t()) < TOL
    z = torch.zeros(3, 300, device="cuda")
    assert not ops.project_in(z, w8)[0].any()


def test_e8m0_scales_and_a_batch_does_not_change_a_row():
    h, W = rows(300, 640, 14, dtype=torch.bfloat16), rows(384, 640, 15)
    w8 = ops.weights_fp8(W)
    want = ops.project_in(h, w8)[0]
    e8 = ops.Weights8(w=w8.w, scale=w8.scale.view(torch.float8_e8m0fnu), k=640)
    assert torch.equal(ops.project_in(h, e8)[0], want)
    assert torch.equal(ops.project_in(h, w8)[0], want)   # the same bits every time
    assert rel(ops.project_in(h[5:6], w8)[0], want[5:6].double()) < TOL


def test_captured_and_on_another_stream():
    h, W = rows(64, 1024, 16, dtype=torch.bfloat16), rows(512, 1024, 17)
    w8 = ops.weights_fp8(W)
    want = ops.project_in(h, w8)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.project_in(h, w8)[0]
    s.synchronize()
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    x = h.clone()
    with torch.cuda.graph(graph):
        q = ops.project_in(x, w8)[0]
    x.copy_(rows(64, 1024, 18, dtype=torch.bfloat16))
    graph.replay()
    assert torch.equal(q, ops.project_in(x, w8)[0])


def test_refusals():
    h, W = rows(4, 256, 19), rows(64, 256, 20)
    w8 = ops.weights_fp8(W)
    with pytest.raises(ValueError, match="columns"):
        ops.project_in(h[:, :128], w8)
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        ops.project_in(h, ops.Weights8(w=w8.w.view(torch.uint8), scale=w8.scale, k=256))
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        ops.project_in(h, ops.Weights8(w=w8.w[:, :128], scale=w8.scale, k=256))
    with pytest.raises(ValueError, match="scales"):
        ops.project_in(h, ops.Weights8(w=w8.w, scale=w8.scale[:, :1], k=256))
    with pytest.raises(ValueError, match="scales"):
        ops.project_in(h, ops.Weights8(w=w8.w, scale=w8.scale.float(), k=256))
    with pytest.raises(ValueError, match="w_prep"):
        ops.project_in(h, w8, w_prep=ops.weights_prep(W))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.project_in(h, ops.Weights8(w=w8.w.cpu(), scale=w8.scale, k=256))
    with pytest.raises(ValueError):
        ops.weights_fp8(torch.zeros(0, 4, device="cuda"))
    with pytest.raises(ValueError):
        ops.weights_fp8(torch.zeros(4, 4, device="cuda", dtype=torch.float64))
    a = ops.Adapters(torch.zeros(1, 2, 256, device="cuda"), torch.zeros(1, 64, 2, device="cuda"))
    with pytest.raises(NotImplementedError, match="adapters"):
        ops.project_in(h, w8, adapters=a, adapter_of=torch.zeros(4, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        ops.project_out(h, w8, torch.zeros(4, 60, device="cuda"))


@pytest.mark.parametrize("R,d_in,d_out", [(1, 300, 64), (9, 256, 512), (70, 512, 1024), (200, 640, 260), (1024, 1024, 2048),
                                          (6000, 384, 1284)])
@pytest.mark.parametrize("selector", [False, True])
def test_the_workspace_of_a_call_is_enough_and_no_less_is(R, d_in, d_out, selector):
    g, guard = gen(50), 4096
    h, W = rows(R, d_in, 51, dtype=torch.bfloat16), rows(d_out, d_in, 52) * d_in ** -0.5
    r, hm = rows(R, d_in, 53), torch.randn(R, d_out, generator=g, device="cuda").to(torch.bfloat16)
    sel_in, sel_row = torch.randn(3, d_in, generator=g, device="cuda") * 0.02, torch.rand(R, generator=g, device="cuda")
    w8 = ops.weights_fp8(W)
    want_q, _, _, want_z = ops.project_in(h, w8, sel_w=sel_in if selector else None)
    want = ops.project_out(r, w8, hm, sel_w=sel_row if selector else None, want_rel=True)
    q, z = torch.empty_like(want_q), torch.empty(R, 3, device="cuda")
    delta, rel = torch.empty_like(hm), torch.empty(R, device="cuda")
    at, stream = (lambda t: None if t is None else t.data_ptr()), torch.cuda.current_stream().cuda_stream
    calls = [("xencb_project_in8", N.lib().xencb_project_in8_workspace_for(R, d_in, d_out, selector),
              N.lib().xencb_project_in8_workspace(R, d_in, d_out), lambda ws, n: N.lib().xencb_project_in8(
                  at(h), N.BF16, R, d_in, at(w8.w), at(w8.scale), None, d_out, N.PIN_RMS | N.PIN_L2, None, 0.0, None,
                  at(sel_in) if selector else None, None, 3 if selector else 0, 1e-6, at(q), None, None,
                  at(z) if selector else None, ws, n, stream)),
             ("xencb_project_out8", N.lib().xencb_project_out8_workspace_for(R, d_in, d_out, selector),
              N.lib().xencb_project_out8_workspace(R, d_in, d_out), lambda ws, n: N.lib().xencb_project_out8(
                  at(r), R, d_in, at(w8.w), at(w8.scale), None, d_out, 1.0, None, None, at(sel_row) if selector else None,
                  0.0, None, None, at(hm), N.BF16, at(delta), None, at(rel), ws, n, stream))]
    for name, need, most, call in calls:
        assert 0 < need <= most, name
        ws = torch.full((need + guard,), 0x5A, dtype=torch.uint8, device="cuda")
        assert call(at(ws), need - 1) == N.EINVAL and call(at(ws), need) == N.OK, name
        assert bool((ws[need:] == 0x5A).all()), name
    assert torch.equal(q, want_q) and (not selector or torch.equal(z, want_z))
    assert torch.equal(delta, want[0]) and torch.equal(rel, want[2])


def test_many_rows_do_not_ask_for_partial_sums():
    # 8-bit rows, their factors, 1/rms and two sums for every 128 outputs of a row
    for query, d_in, d_out in (("in8", 5120, 2048), ("out8", 2048, 4096)):
        size = getattr(N.lib(), f"xencb_project_{query}_workspace_for")
        assert size(16384, d_in, d_out, 0) <= 16384 * (d_in + d_in // 128 + 4 + d_out // 128 * 8) + 1024
        assert size(16384, d_in, d_out, 1) > 16384 * d_out * 4


@pytest.mark.parametrize("R,k,n,selector,bound", [(2048, 5120, 2048, False, 6e-7), (2048, 4096, 2048, False, 6e-7),
                                                  (700, 2176, 2048, False, 6e-7), (2048, 5120, 2048, True, 1e-6),
                                                  (2048, 8192, 2048, False, 1e-6), (7, 12000, 18940, False, 1e-6),
                                                  (100, 12000, 18940, False, 1e-6), (64, 5120, 2048, False, 6e-7)])
def test_long_sums_keep_their_precision(R, k, n, selector, bound):
    """The accumulator drops about 3.5e-8 of the result, in norm, for every block of 128 columns that it runs over (4.4e-8 over
    many): 5.6e-7 over the 16 of calls of many rows, at most 8.8e-7 over the 20 of the others, and a float32 sum of a few runs
    adds 1e-7 that does not depend on it. Over 40, 64 and 94 blocks at once: 1.6e-6, 2.8e-6 and 4.1e-6."""
    loud = torch.exp(1.5 * torch.randn(k, generator=gen(60), device="cuda"))
    h = (torch.randn(R, k, generator=gen(61), device="cuda") * loud).to(torch.bfloat16)
    W = torch.randn(n, k, generator=gen(62), device="cuda") * k ** -0.5
    sel_w = torch.randn(2, k, generator=gen(63), device="cuda") if selector else None
    got = ops.project_in(h, ops.weights_fp8(W), rms=False, l2=False, sel_w=sel_w)[0].double()
    want = values(h) @ values(W).t()
    off = float((got - want).norm() / want.norm())
    assert off < bound, off


@pytest.mark.parametrize("R,k,n", [(5000, 5000, 1800), (9000, 2176, 1284), (20000, 2304, 516), (2600, 4224, 2052)])
def test_several_tiles_of_several_runs(R, k, n):
    """Calls of many rows whose CTAs take several tiles, the accumulator out two or three times in each (odd and even)."""
    h, W = rows(R, k, 64, dtype=torch.bfloat16), rows(n, k, 65) * k ** -0.5
    w8 = ops.weights_fp8(W)
    y = values(h) @ values(W).t()
    assert rel(ops.project_in(h, w8, rms=False, l2=False)[0], y) < TOL
    assert rel(ops.project_in(h, w8)[0], y / y.norm(dim=-1, keepdim=True)) < TOL
    r, x = h.float(), torch.randn(R, n, generator=gen(66), device="cuda").to(torch.bfloat16)
    _, got, mag = ops.project_out(r, w8, x, scale=0.5, want_delta=False, h_out=torch.empty_like(x), want_rel=True)
    want, half = x.double() + 0.5 * y, torch.finfo(torch.bfloat16).eps / 2
    assert float((got.double() - want).abs().max() / want.abs().max()) < TOL + 2 * half
    want = 0.5 * y.norm(dim=-1) / (x.double().norm(dim=-1) + 1e-6)
    assert float((mag.double() - want).abs().max() / want.max()) < TOL + half
