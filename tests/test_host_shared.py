"""Refusals of the shared read, the page operators and the adapters that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from kv_skill_v2_b200 import _native as N
from kv_skill_v2_b200 import ops
from tests._fixtures import TinyReader


def _pages(d=64):
    return ops.Pages(slots=torch.zeros(2, 4, d, dtype=torch.float16), page_of=torch.zeros(1, 2, dtype=torch.int32),
                     n_valid=torch.ones(1, 2, dtype=torch.int32), S=torch.zeros(1, 2, d))


def test_cpu_tensors_are_refused():
    q, idx, wk = torch.zeros(1, 64), torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, 1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.read_shared(q, _pages(), idx, wk, rows_per_lib=1)
    p = _pages()
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.pages_fork([p.slots], p.page_of, p.n_valid, one, one)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.pages_compact([p.slots], p.page_of, p.n_valid)
    with pytest.raises(ValueError, match="at least one pool"):
        ops.pages_compact([], p.page_of, p.n_valid)
    ad = ops.Adapters(torch.zeros(1, 2, 64), torch.zeros(1, 64, 2))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.project_in(torch.zeros(1, 64), torch.zeros(64, 64), adapters=ad, adapter_of=one)


def test_read_shared_shapes():
    """The workspace query (host only) tells which shapes the kernel takes."""
    size = N.lib().xencb_read_shared_workspace
    for d in (8, 64, 200, 2048, 2560, 4096):
        assert size(4, 2, d, 10, 512, N.F16, N.F32) >= size(4, 2, d, 10, 512, N.F16, N.BF16) > 0
    for bad in ((4, 2, 60, 10, 512, N.F16, N.F32), (4, 2, 4104, 10, 512, N.F16, N.F32),
                (4, 2, 64, 10, 512, N.F32, N.F32), (4, 2, 64, 10, 512, N.F16, 7), (0, 2, 64, 10, 512, N.F16, N.F32),
                (4, 0, 64, 10, 512, N.F16, N.F32), (1 << 31, 64, 64, 10, 512, N.F16, N.F32),
                (4, 2, 64, 1 << 24, 512, N.F16, N.F32)):
        assert size(*bad) == 0
    assert ops.shared_supported(_pages()) and not ops.shared_supported(_pages(60))


def _call(fn, *args):
    return getattr(N.lib(), fn)(*args)


def test_page_operators_refuse_bad_arguments():
    one, buf = ctypes.c_void_p(256), (ctypes.c_void_p * 1)(256)
    row = (ctypes.c_int64 * 1)(16)

    def compact(pools=buf, rows=row, n=1, pages=4, page_rows=2, table=one, C=2, n_lib=1, ws=one, ws_bytes=1 << 20):
        return _call("xencb_pages_compact", pools, rows, n, pages, page_rows, table, one, C, None, n_lib, one, one, ws,
                     ws_bytes, None)

    def fork(m=1, parents=one, ws_bytes=1 << 20, C=2):
        return _call("xencb_pages_fork", buf, row, 1, 4, 2, one, one, C, None, 1, parents, one, m, one, one, one,
                     ws_bytes, None)

    assert compact(pools=None) == N.EINVAL and compact(n=0) == N.EINVAL and compact(pages=0) == N.EINVAL
    assert compact(rows=(ctypes.c_int64 * 1)(3)) == N.EINVAL and compact(table=None) == N.EINVAL
    assert compact(pages=(1 << 20) + 1) == N.ENOTSUP and compact(C=0) == N.EINVAL
    assert compact(C=1 << 20, n_lib=1 << 12) == N.ENOTSUP
    assert compact(ws=ctypes.c_void_p(264)) == N.EINVAL and compact(ws_bytes=8) == N.EINVAL
    assert fork(m=0) == N.EINVAL and fork(parents=None) == N.EINVAL and fork(ws_bytes=8) == N.EINVAL
    assert fork(m=1 << 20, C=1 << 12) == N.ENOTSUP
    assert N.lib().xencb_pages_fork_workspace(0, 4) == 0 and N.lib().xencb_pages_compact_workspace(0) == 0


class _OwnInterface:
    """An interface object of the caller's: query, gate, gain and write only."""

    d_s, inject_layers = 16, [0]

    def query(self, hn):
        return hn[..., :16]

    def gate(self, hn, li):
        return hn[..., :1]

    def gain(self, li):
        return 1.0

    def write(self, r):
        return r


@pytest.mark.parametrize("kind", ["XEncInjector", "LibraryInjector"])
def test_adapters_need_a_known_interface(kind):
    """An interface that the kernels do not see refuses adapters, rather than leaving them out."""
    import kv_skill_v2_b200 as pkg

    inj = getattr(pkg, kind)(TinyReader(32, 2), _OwnInterface())
    ad = pkg.ops.Adapters(a=torch.zeros(1, 2, 32), b=torch.zeros(1, 16, 2))
    with pytest.raises(NotImplementedError):
        inj.set_adapters(ad, None, torch.zeros(1, dtype=torch.int32))
    inj._adapters = (ad, None, torch.zeros(1, dtype=torch.int32))  # (an interface exchanged after set_adapters)
    with pytest.raises(NotImplementedError):
        inj._duck_finish(torch.zeros(1, 1, 32), torch.zeros(1, 32), torch.zeros(1, 16), 1.0, 0, False)
    inj.set_adapters()
    assert inj._adapters is None
    inj.detach()


def test_a_captured_step_is_keyed_by_the_adapters_layout():
    """Adapters of one address, shape and type but other strides are other adapters to a captured step."""
    from kv_skill_v2_b200 import LibraryInjector, make_interface

    inj = LibraryInjector(TinyReader(16, 2), make_interface(16, 16, [0]))
    a, of = torch.zeros(1, 16, 16), torch.zeros(1, dtype=torch.int32)
    keys = set()
    for x in (a, a.transpose(1, 2)):
        inj.set_adapters(ops.Adapters(a=x, b=a), None, of)
        keys.add(inj._adapter_key())
    assert len(keys) == 2
    inj.detach()


@pytest.mark.parametrize("entries,shape", [(4, (2, 2, 32)), (4, (8, 1, 32)), (4, (1, 64, 32)), (1, (3, 2, 32)),
                                           (0, (2, 1, 32)), (2, (4, 32)), (8, (2, 4, 32))])
@pytest.mark.parametrize("which", [0, 1])
def test_an_adapter_of_of_another_batch_is_refused(entries, shape, which):
    """Whatever divides the rows: the entries belong to batch rows."""
    from kv_skill_v2_b200 import LibraryInjector, PagedLibrary
    from kv_skill_v2_b200.interface import LinearInterface

    itf = LinearInterface(torch.zeros(32, 16), torch.zeros(16, 32), [0]).requires_grad_(False)
    ad = ops.Adapters(a=torch.zeros(1, 2, 32), b=torch.zeros(1, 16, 2))
    out = ops.Adapters(a=torch.zeros(1, 2, 16), b=torch.zeros(1, 32, 2))
    inj = LibraryInjector(TinyReader(32, 2), itf)
    inj.load_library(PagedLibrary({0: _pages(16)}))
    inj.set_adapters(ad if which == 0 else None, out if which else None, torch.zeros(entries, dtype=torch.int32))
    h = torch.zeros(shape)
    with torch.no_grad(), pytest.raises(ValueError, match="adapter_of"):
        if which == 0:
            inj._inject(h, 0)
        else:  # (the read before it needs a GPU)
            inj._finish(h, h.reshape(-1, 32), torch.zeros(h.numel() // 32, 16), None, 1.0, 0, True)
    inj.detach()


@pytest.mark.parametrize("entries,shape,each", [(2, (2, 2, 32), 2), (8, (8, 1, 32), 1), (1, (1, 64, 32), 64),
                                                (4, (4, 32), 1), (1, (5, 32), 5), (1, (32,), 1)])
def test_adapter_of_per_batch_row(entries, shape, each):
    from kv_skill_v2_b200 import LibraryInjector
    from kv_skill_v2_b200.interface import LinearInterface

    inj = LibraryInjector(TinyReader(32, 2), LinearInterface(torch.zeros(32, 16), torch.zeros(16, 32), [0]))
    inj.set_adapters(ops.Adapters(a=torch.zeros(1, 2, 32), b=torch.zeros(1, 16, 2)), None,
                     torch.zeros(entries, dtype=torch.int32))
    assert inj._adapter_args(0, torch.zeros(shape))["rows_per_adapter"] == each
    assert inj._adapter_args(1, torch.zeros(shape)) == {}
    inj.detach()


def test_read_shared_refuses_other_tables():
    """page_of and n_valid are read as dense int32 [n_lib, C]: any other layout would be misread, or read past its end."""
    q, idx, wk = torch.zeros(2, 64), torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, 1)
    t = torch.zeros(2, 3, dtype=torch.int32)
    for page_of, n_valid in ((t.long(), t), (t, t.long()), (t, t[:1]), (t, t[:, :2].contiguous()), (t.t().contiguous().t(), t),
                             (t, t.t().contiguous().t()), (t[0], t[0]), (t.expand(4, 2, 3)[0].repeat(1, 2)[:, ::2], t)):
        p = ops.Pages(slots=torch.zeros(2, 4, 64, dtype=torch.float16), page_of=page_of, n_valid=n_valid,
                      S=torch.zeros(2, 3, 64))
        with pytest.raises(ValueError, match="contiguous int32"):
            ops.read_shared(q, p, idx, wk, rows_per_lib=1)


def test_slices_of_a_shared_read():
    """Every row once and in order, no slice above the limit unless it is one row, and none that holds parts of two
    Libraries."""
    import random

    rng = random.Random(0)
    for _ in range(2000):
        rpl, n, per = rng.randint(1, 40), rng.randint(1, 200), rng.randint(1, 50)
        limit, most = rng.randint(1, 3000), rng.choice([10 ** 9, rng.randint(1, 50)])

        def size(rows):
            return 0 if rows > most else 7 + per * rows

        parts = ops.shared_slices(n, rpl, size, limit)
        assert [r for a, b in parts for r in range(a, b)] == list(range(n))
        for a, b in parts:
            assert 0 < size(b - a) <= limit or b - a == 1
            assert a // rpl == (b - 1) // rpl or a % rpl == 0
        if 0 < size(n) <= limit:
            assert parts == [(0, n)]


def test_a_dense_prompt_over_shared_pages_is_sliced():
    """4 x 2048 tokens on 64 chunks of 512 x 2048 would take 8.6 GB in one call."""
    p = ops.Pages(slots=torch.zeros(1, 1, 1).half().expand(64, 512, 2048), page_of=torch.zeros(4, 64, dtype=torch.int32),
                  n_valid=torch.ones(4, 64, dtype=torch.int32), S=torch.zeros(4, 64, 1))
    assert ops.shared_workspace(p, 4 * 2048, 64) > 8 << 30
    for rows, rpl in ((4 * 2048, 2048), (8 * 4096, 4096), (64, 1)):
        parts = ops.shared_slices(rows, rpl, lambda n: ops.shared_workspace(p, n, 64), ops.SHARED_WORKSPACE)
        assert max(ops.shared_workspace(p, b - a, 64) for a, b in parts) <= ops.SHARED_WORKSPACE
        assert len(parts) <= 1 + 2 * ops.shared_workspace(p, rows, 64) // ops.SHARED_WORKSPACE


@pytest.mark.parametrize("which", ["a", "b", "scale"])
@pytest.mark.parametrize("side", [0, 1])
def test_adapters_that_need_gradients_are_refused(which, side):
    """As an interface that needs them is: the kernels would leave the adapters out of the graph."""
    from kv_skill_v2_b200 import LibraryInjector, PagedLibrary
    from kv_skill_v2_b200.interface import LinearInterface

    itf = LinearInterface(torch.zeros(32, 16), torch.zeros(16, 32), [0]).requires_grad_(False)
    inj = LibraryInjector(TinyReader(32, 2), itf)
    inj.load_library(PagedLibrary({0: _pages(16)}))
    d_in, d_out = ((32, 16), (16, 32))[side]
    ad = ops.Adapters(a=torch.zeros(1, 2, d_in), b=torch.zeros(1, d_out, 2), scale=torch.ones(1))
    getattr(ad, which).requires_grad_()
    inj.set_adapters(*((ad, None), (None, ad))[side], torch.zeros(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="forward-only"):
        inj._inject(torch.zeros(1, 1, 32), 0)
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
        inj._inject(torch.zeros(1, 1, 32), 0)
    inj.detach()
