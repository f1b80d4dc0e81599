"""Slots and rows that are written in place between calls: every way of an adapted product follows them."""

from __future__ import annotations

import pytest
import torch

from . import adapters_util as au
from .test_adapters_gpu import EIGHT, LONG, run_linear

pytestmark = pytest.mark.gpu

SHORT = [(3, i % 5 - 1) for i in range(10)]


@pytest.mark.parametrize("way,rows,rank", [("stream", EIGHT, 16), ("decode", EIGHT, 16), ("decode", SHORT, 16), ("pair", SHORT, 16), ("pair", LONG, 16), ("apart", SHORT, 16),
                                           ("apart", LONG[1:] + SHORT, 256), (None, LONG, 16), (None, SHORT, 16)])
@pytest.mark.parametrize("write", ["copy", "index", "rows", "uncounted"])
def test_products_follow_what_is_written(way, rows, rank, write, monkeypatch):
    """rank 256: v by a plan, in 32 bits, beside a product apart. uncounted: a write that torch does not count, and refresh behind it."""
    from miniserve_b200 import ops

    monkeypatch.setattr(ops.adapters, "WAY", way)
    x, w, low, ar = au.made(rows, 1024, (512, 264), rank, 4, torch.bfloat16, seed=rank)
    before = run_linear(x, w, low, ar)
    for turn in range(2):
        rolled = torch.roll(ar.slot_of_row, 1)
        if write == "copy":
            ar.slot_of_row.copy_(rolled)
        elif write == "index":
            ar.slot_of_row[0], ar.slot_of_row[-1] = (turn + 1) % 4, turn % 4
        elif write == "rows":
            gen = torch.Generator(device="cuda").manual_seed(turn)
            ar.row_of_token.copy_(torch.sort(torch.randint(0, ar.rows, (ar.tokens,), generator=gen, device="cuda")).values)
        else:
            ar.slot_of_row.data.copy_(rolled)
            ar.refresh()
        got = run_linear(x, w, low, ar)
        au.close(got, *au.formula(x, w, low, ar))
        assert not torch.equal(got, before)
        before = got


def test_rows_of_inference_mode_are_followed():
    x, w, low, _ = au.made(LONG, 1024, (2048,), 16, 4, torch.bfloat16)
    with torch.inference_mode():
        ar = au.rows_of(LONG)
        for slots in ((3, 1), (0, 2), (-1, 0)):
            ar.slot_of_row.copy_(torch.tensor(slots, dtype=torch.int32))
            got = run_linear(x, w, low, ar)
            au.close(got, *au.formula(x, w, low, ar))


def test_a_plan_is_kept_while_nothing_is_written():
    x, w, low, ar = au.made(LONG, 1024, (2048,), 16, 4, torch.bfloat16)
    stream = torch.cuda.current_stream().cuda_stream
    held = ar.plan(low.slots, stream)
    run_linear(x, w, low, ar)
    assert ar.plan(low.slots, stream) is held
    ar.slot_of_row.copy_(ar.slot_of_row.flip(0))
    assert ar.plan(low.slots, stream) is not held


def test_writes_between_two_products_of_one_capture():
    """The second product's plan is the graph's own, behind the write that the graph holds."""
    from miniserve_b200 import ops

    x, w, low, ar = au.made(LONG, 1024, (2048,), 16, 4, torch.bfloat16)
    run_linear(x, w, low, ar)
    given = [torch.tensor(s, dtype=torch.int32, device="cuda") for s in ((3, 1), (0, 2))]
    outs = [torch.empty((x.shape[0], 2048), dtype=torch.bfloat16, device="cuda") for _ in given]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for slots, out in zip(given, outs):
            ar.slot_of_row.copy_(slots)
            ops.linear(x, w, out=out, low_rank=low, adapter_rows=ar)
    for turn in range(2):
        given[turn].copy_(given[turn].flip(0))
        graph.replay()
        torch.cuda.synchronize()
        for slots, out in zip(given, outs):
            au.close(out, *au.formula(x, w, low, au.rows_of([(n, int(s)) for (n, _), s in zip(LONG, slots.tolist())])))
