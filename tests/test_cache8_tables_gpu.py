"""The 8-bit cache over the page tables that the engine's packer makes for windowed groups."""

from __future__ import annotations

import pytest
import torch

from tests import cache8_util as cu
from tests import kernel_util as ku
from tests.test_cache8_gpu import _attend, _close

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _guarded(t: torch.Tensor, guard: torch.Tensor) -> torch.Tensor:
    """A tensor of t's size in the middle of ``guard``."""
    return guard[1024:1024 + t.numel()]


@pytest.mark.parametrize("nq,nkv,d,page", [(16, 8, 128, 16), (16, 2, 64, 16), (8, 1, 80, 8), (8, 1, 256, 32)])
@pytest.mark.parametrize("rows,window", [([(250, 300)], 40), ([(2900, 3000)], 512), ([(100, 200), (3, 140)], 5), ([(700, 300), (0, 500), (0, 33)], 200)])
def test_prompts_over_unpacked_pages_behind_a_window(nq, nkv, d, page, rows, window):
    """Pages that the window has passed are neither in the table nor unpacked; nothing beside the scratch is written."""
    pb = cu.Packed8(rows, page, nkv, d, window, seed=d)
    ctx = ku.make_context(pb)
    q, out = _attend(pb, nq, d, 0.1, window, ctx=ctx)
    held = ctx.scratch["cache8_pages"]
    _close(pb, q, out, 0.1, window)
    guards = [torch.full((t.numel() + 2048,), 77, dtype=t.dtype, device=DEV) for t in held[:3]]
    again = ku.make_context(pb)
    again.scratch = dict(ctx.scratch, cache8_pages=tuple(_guarded(t, g) for t, g in zip(held, guards)) + tuple(held[3:]))
    _, second = _attend(pb, nq, d, 0.1, window, ctx=again, q=q)
    assert torch.equal(out, second)
    for g in guards:
        assert bool((g[:1024] == 77).all()) and bool((g[-1024:] == 77).all())
