"""What a server does around a Library that shrinks: evictions that are refused leave it whole."""

from __future__ import annotations

import pytest
import torch

from kv_skill_v2_b200 import LibraryInjector, ops
from tests._fixtures import TinyReader
from tests.test_gpu_shrink import D_M, DEV, LAYERS, interface, library

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
