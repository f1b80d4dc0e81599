"""Adapted products while another device than the tensors' is the current one (which a single GPU shows by what they ask torch for)."""

from __future__ import annotations

import pytest
import torch

from . import adapters_util as au
from .test_adapters_gpu import EIGHT, LONG, run_linear

pytestmark = pytest.mark.gpu


@pytest.fixture
def elsewhere(monkeypatch):
    """A current device of 1 until torch.cuda.device(0) is entered; the devices that were entered."""
    entered, current = [], [1]

    class device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            entered.append(self.index)
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    return entered


@pytest.mark.parametrize("rows", [EIGHT, LONG])
def test_products_go_to_their_tensors_device(rows, elsewhere, monkeypatch):
    from miniserve_b200 import ops

    from .kernel_util import PagedBatch

    with monkeypatch.context() as here:
        here.setattr(torch.cuda, "current_device", lambda: 0)
        nq, nkv, d, page = 4, 2, 128, 16
        pb = PagedBatch([(0, n) for n, _ in rows], page, nkv, d, torch.bfloat16, seed=3)
        x, w, low, ar = au.made(rows, 512, (nq * d, nkv * d, nkv * d), 16, 4, torch.bfloat16)
        want = run_linear(x, w, low, ar)
        q = torch.full((x.shape[0], nq, d), float("nan"), dtype=torch.bfloat16, device="cuda")
        out = torch.empty_like(want)
        stream = torch.cuda.current_stream().cuda_stream
    elsewhere.clear()
    ops.linear(x, w, out=out, low_rank=low, adapter_rows=ar, stream=stream)
    assert elsewhere and set(elsewhere) == {0}
    elsewhere.clear()
    ops.qkv_norm_rope_kv(q, pb.k_pool, pb.v_pool, x, w, None, None, None, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, page, stream=stream,
                         low_rank=low, adapter_rows=ar)
    assert elsewhere and set(elsewhere) == {0}
    monkeypatch.undo()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    au.close(q.view(x.shape[0], -1), *(z[:, :nq * d] for z in au.formula(x, w, low, ar)))
