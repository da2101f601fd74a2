"""Refusals of the attention mass, eviction and the 8-bit projections that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from kv_skill_v2_b200 import _native as N
from kv_skill_v2_b200 import ops


def pages(d=64):
    return ops.Pages(slots=torch.zeros(2, 4, d, dtype=torch.float16), page_of=torch.zeros(1, 2, dtype=torch.int32),
                     n_valid=torch.ones(1, 2, dtype=torch.int32), S=torch.zeros(1, 2, d))


def test_cpu_tensors_are_refused():
    p = pages()
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.read_mass(torch.zeros(1, 64), p, torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, 1), rows_per_lib=1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.pages_evict([p.slots], p.page_of, p.n_valid, torch.zeros(2, 4), 2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.weights_fp8(torch.zeros(4, 64))
    w = ops.Weights8(torch.zeros(4, 128, dtype=torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.uint8), 64)
    assert w.shape == (4, 64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.project_in(torch.zeros(1, 64), w)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.project_out(torch.zeros(1, 64), w, torch.zeros(1, 4))
    with pytest.raises(ValueError, match="at least one pool"):
        ops.pages_evict([], p.page_of, p.n_valid, torch.zeros(2, 4), 2)


def test_read_mass_shapes():
    """The workspace query (host only) tells which shapes the kernel takes."""
    size = N.lib().xencb_read_mass_workspace
    for d in (8, 64, 200, 2048, 5120, 8192):
        for rows in (1, 96, 512, 700, 2048):
            assert size(4, 2, d, 10, rows, N.F16, N.F32) >= size(4, 2, d, 10, rows, N.F16, N.BF16) > 0
    for bad in ((4, 2, 60, 10, 512, N.F16, N.F32), (4, 2, 64, 10, 2049, N.F16, N.F32), (4, 2, 64, 10, 512, N.F32, N.F32),
                (4, 2, 64, 10, 512, N.F16, 7), (0, 2, 64, 10, 512, N.F16, N.F32), (4, 0, 64, 10, 512, N.F16, N.F32),
                (1 << 31, 64, 64, 10, 512, N.F16, N.F32), (4, 2, 64, 1 << 24, 512, N.F16, N.F32)):
        assert size(*bad) == 0


def call(fn, *args):
    return getattr(N.lib(), fn)(*args)


def test_evict_refuses_bad_arguments():
    one, buf, other = ctypes.c_void_p(256), (ctypes.c_void_p * 1)(256), (ctypes.c_void_p * 1)(512)
    row = (ctypes.c_int64 * 1)(16)

    def evict(pools=buf, out=other, rows=row, n=1, P=4, N_rows=8, new=4, table=one, C=2, n_lib=1, mass=one, floor=1, ws=one,
              ws_bytes=1 << 20):
        return call("xencb_pages_evict", pools, out, rows, n, P, N_rows, new, table, one, C, None, n_lib, mass, None, 3, 0,
                    floor, one, one, one, ws, ws_bytes, None)

    for bad in (dict(pools=None), dict(out=None), dict(rows=None), dict(n=0), dict(P=0), dict(table=None), dict(mass=None),
                dict(C=0), dict(n_lib=0), dict(new=0), dict(new=9), dict(floor=-1), dict(ws=None), dict(ws_bytes=8),
                dict(out=buf), dict(rows=(ctypes.c_int64 * 1)(3))):
        assert evict(**bad) == N.EINVAL, bad
    assert evict(N_rows=4097, new=4) == N.ENOTSUP and evict(n_lib=1 << 31) == N.ENOTSUP
    assert call("xencb_pages_evict_workspace", 4, 4097, 0) == 0 and call("xencb_pages_evict_workspace", 0, 8, 0) == 0
    assert call("xencb_pages_evict_workspace", 4, 8, 1) > call("xencb_pages_evict_workspace", 4, 8, 0) > 0


def test_evict_refuses_outputs_that_overlap():
    at = lambda *a: (ctypes.c_void_p * len(a))(*a)  # noqa: E731
    row, p = (ctypes.c_int64 * 2)(16, 16), ctypes.c_void_p(1 << 30)

    def evict(pools, out, new=4, mass=1 << 29):  # a workspace of 8 bytes ends the calls that get past the check
        return call("xencb_pages_evict", pools, out, row, 2, 4, 8, new, p, p, 2, None, 1, ctypes.c_void_p(mass), None, 3, 0, 1,
                    p, p, p, p, 8, None)

    for bad in ((at(4096, 8192), at(4096 + 496, 16384)), (at(4096, 8192), at(8192, 4096)), (at(4096, 8192), at(1 << 20, 1 << 20)),
                (at(4096, 8192), at(1 << 20, (1 << 20) + 240)), (at(4096, 8192), at(4096 - 240, 1 << 20))):
        assert evict(*bad) == N.EINVAL and b"overlaps" in N.lib().xencb_last_error(), bad
    for good in ((at(4096, 4096), at(4096 + 512, 4096 - 256)), (at(4096, 8192), at(1 << 20, (1 << 20) + 256))):
        assert evict(*good) == N.EINVAL and b"workspace" in N.lib().xencb_last_error()
    assert evict(at(4096, 4096), at(4096, 4096), new=8) == N.EINVAL and b"overlaps" in N.lib().xencb_last_error()
    assert evict(at(4096, 4608), at(4096, 4608), new=8) == N.EINVAL and b"workspace" in N.lib().xencb_last_error()
    assert evict(at(4096, 4608), at(4096, 4608), new=8, mass=1 << 30) == N.EINVAL and b"mass_out" in N.lib().xencb_last_error()


def test_mass_and_8_bit_calls_refuse_bad_arguments():
    p = ctypes.c_void_p(256)

    def mass(q=p, R=4, d=64, slots=p, dt=N.F16, P=4, stride=8 * 64, rows=8, rpl=4, n_lib=1, out=p, ws=p, ws_bytes=1 << 30):
        return call("xencb_read_mass", q, N.F32, R, d, slots, dt, P, stride, rows, p, p, 2, rpl, n_lib, p, p, 2, 12.0, None, 1.0,
                    out, ws, ws_bytes, None)

    for bad in (dict(q=None), dict(slots=None), dict(out=None), dict(R=0), dict(rpl=0), dict(R=9), dict(ws=None),
                dict(ws_bytes=8), dict(q=ctypes.c_void_p(258)), dict(slots=ctypes.c_void_p(264))):
        assert mass(**bad) == N.EINVAL, bad
    for bad in (dict(d=60, stride=480), dict(dt=N.F32), dict(stride=640), dict(rows=2049, stride=2049 * 64)):
        assert mass(**bad) == N.ENOTSUP, bad
    for bad in ((None, 0, 4, 64, p, p), (p, 0, 0, 64, p, p), (p, 0, 4, 0, p, p), (p, 9, 4, 64, p, p), (p, 0, 4, 64, None, p),
                (p, 0, 4, 64, p, None), (p, 0, 4, 64, ctypes.c_void_p(264), p)):
        assert call("xencb_quant8", *bad, None) == N.EINVAL, bad


def test_evict_refuses_pages_that_are_too_large_before_anything_moves():
    """The last of 33 pools, which the second launch would move: refused with the arguments (no device is needed to say so)."""
    p, big = ctypes.c_void_p(256), 1 << 40
    at = (ctypes.c_void_p * 33)(*[4096 * (i + 1) for i in range(33)])

    def evict(row, odd=0):
        rows = (ctypes.c_int64 * 33)(*[16] * 32, row)
        pools = (ctypes.c_void_p * 33)(*[at[i] for i in range(32)], big + odd)
        return call("xencb_pages_evict", pools, pools, rows, 33, 4, 8, 8, p, p, 2, None, 1, ctypes.c_void_p(1 << 20), None, 3, 0,
                    1, p, p, p, p, 8, None)

    for row, odd in ((1 << 33, 0), (1 << 45, 0), (1 << 30, 2), ((1 << 29) + 2, 0)):  # (in 16-byte units, or in 2-byte ones)
        assert evict(row, odd) == N.ENOTSUP and b"pool 32" in N.lib().xencb_last_error(), (row, odd)
    for row, odd in ((16, 0), (1 << 30, 0), ((1 << 28) - 2, 2)):  # a workspace of 8 bytes ends the calls that get past it
        assert evict(row, odd) == N.EINVAL and b"workspace" in N.lib().xencb_last_error(), (row, odd)
