"""Numbers of an adapter that leave 32 bits give infinities of their sign in their own tokens' outputs, and in no others."""

from __future__ import annotations

import pytest
import torch

from . import adapters_util as au
from .test_adapters_gpu import DECODE64, EIGHT, LONG, run_linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("way,rows", [("stream", EIGHT), ("decode", EIGHT), ("decode", DECODE64), ("pair", LONG), ("apart", EIGHT), ("apart", LONG), ("float32 outputs", EIGHT)])
def test_infinities_keep_their_sign(way, rows, monkeypatch):
    """One number of slot 3's is infinite, and meets a column of B whose entries are of both signs."""
    from miniserve_b200 import ops

    monkeypatch.setattr(ops.adapters, "WAY", None if way == "float32 outputs" else way)
    x, w, low, ar = au.made(rows, 512, (264,), 16, 4, torch.bfloat16)
    x[:, 0] = 8.0
    low.a[3, 5] = 0.0
    low.a[3, 5, 0] = 3e38
    got = run_linear(x, w, low, ar, torch.float32 if way == "float32 outputs" else None)
    mine = ar.slot_of_row[ar.row_of_token.long()] == 3
    sign = torch.sign(low.b[3, :, 5].float())
    assert bool(mine.any()) and bool((sign != 0).all())
    want = (sign * float("inf")).expand(int(mine.sum()), -1)
    assert torch.equal(got[mine].float(), want)
    low.a[3, 5, 0] = 0.0
    y, tol = au.formula(x, w, low, ar)
    au.close(got[~mine], y[~mine], tol[~mine])
