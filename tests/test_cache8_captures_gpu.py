"""The 8-bit cache's attention of one context called eagerly, on another stream and captured, in turn."""

from __future__ import annotations

import pytest
import torch

from miniserve_b200 import ops
from tests import cache8_util as cu
from tests import kernel_util as ku
from tests.test_cache8_gpu import _attend, _close

pytestmark = pytest.mark.gpu
DEV = "cuda"
PROMPTS = [(16, 8, 128, [(30, 170), (0, 200)]), (16, 2, 64, [(30, 170), (0, 200)]), (16, 2, 128, [(900, 1), (37, 1)]), (8, 1, 64, [(700, 90)])]


@pytest.mark.parametrize("nq,nkv,d,rows", PROMPTS)
def test_a_context_captured_on_a_side_stream_after_an_eager_call(nq, nkv, d, rows):
    """All of the step's launches are in the graph, and its scratch stays when a longer prompt needs more."""
    pb, other = cu.Batch8(rows, 16, nkv, d, seed=8), cu.Batch8([(300, 2000)], 16, nkv, d, seed=9)
    ctx = ku.make_context(pb)
    q, want = _attend(pb, nq, d, 0.1, ctx=ctx)
    _close(pb, q, want, 0.1)
    out, graph, side = torch.full_like(q, float("nan")), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        ctx.stream = torch.cuda.current_stream().cuda_stream
        ops.attention(out, q, pb.k8, pb.v8, ctx, 0, 0.1, None)
    torch.cuda.synchronize()
    assert bool(out.isnan().all()), "something ran outside the graph"
    larger = ku.make_context(other)
    larger.scratch = ctx.scratch
    for _ in range(2):
        _close(other, *_attend(other, nq, d, 0.1, ctx=larger), 0.1)
        torch.full((1 << 24,), float("nan"), dtype=torch.bfloat16, device=DEV)  # (what has been given back is taken)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    ctx.stream = torch.cuda.current_stream().cuda_stream  # and eagerly again
    out.fill_(float("nan"))
    ops.attention(out, q, pb.k8, pb.v8, ctx, 0, 0.1, None)
    assert torch.equal(out, want)


@pytest.mark.parametrize("nq,nkv,d,rows", PROMPTS)
def test_two_graphs_of_one_context(nq, nkv, d, rows):
    """The second is replayed alone, before the first has ever run."""
    pb = cu.Batch8(rows, 16, nkv, d, seed=8)
    q, want = _attend(pb, nq, d, 0.1)
    ctx, outs, graphs = ku.make_context(pb), [torch.full_like(q, float("nan")) for _ in range(2)], [torch.cuda.CUDAGraph() for _ in range(2)]
    ops.attention(torch.empty_like(q), q, pb.k8, pb.v8, ku.make_context(pb), 0, 0.1, None)  # (what is loaded at a first call)
    torch.cuda.synchronize()
    for out, graph in zip(outs, graphs):
        torch.full((1 << 24,), float("nan"), dtype=torch.bfloat16, device=DEV)
        with torch.cuda.graph(graph):
            ctx.stream = torch.cuda.current_stream().cuda_stream
            ops.attention(out, q, pb.k8, pb.v8, ctx, 0, 0.1, None)
    for i in (1, 0, 1):
        outs[i].fill_(float("nan"))
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i], want)


@pytest.mark.parametrize("nq,nkv,d,rows", PROMPTS)
def test_a_context_s_stream_may_change(nq, nkv, d, rows):
    """Both of a prompt's kernels go where ``ctx.stream`` says at the call."""
    pb = cu.Batch8(rows, 16, nkv, d, seed=8)
    ctx = ku.make_context(pb)
    q, want = _attend(pb, nq, d, 0.1, ctx=ctx)
    side, out, new = torch.cuda.Stream(), torch.full_like(q, float("nan")), torch.randn_like(q)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # busy for some milliseconds: what goes elsewhere comes first
        q.copy_(new)
        ctx.stream = side.cuda_stream
        ops.attention(out, q, pb.k8, pb.v8, ctx, 0, 0.1, None)
    side.synchronize()
    _close(pb, new, out, 0.1)


def test_scratch_that_grows_gives_the_old_back_first():
    """A longer prompt's pages take the place of a shorter one's; a step whose groups' pages are of two sizes keeps the larger alone."""
    pb, longer = cu.Batch8([(3000, 3100)], 16, 8, 128, seed=8), cu.Batch8([(9000, 9100)], 16, 8, 128, seed=9)
    wide = cu.Batch8([(3000, 3100)], 16, 16, 128, seed=10)
    ctx = ku.make_context(pb)
    ctx.page_indptr.append(wide.page_indptr)
    ctx.page_indices.append(wide.page_indices)
    q, out = _attend(pb, 16, 128, 0.1, ctx=ctx)
    held = lambda c: sum(t.numel() * t.element_size() for t in c.scratch["cache8_pages"][:3])  # noqa: E731
    rest = lambda c: sum(t.numel() * t.element_size() for t in c.scratch.values() if isinstance(t, torch.Tensor)) + (1 << 20)  # noqa: E731  (the prompt kernel's own)
    first = held(ctx)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    ops.attention(out, q, wide.k8, wide.v8, ctx, 1, 0.1, None)
    again = torch.empty_like(q)
    ops.attention(again, q, pb.k8, pb.v8, ctx, 0, 0.1, None)
    assert held(ctx) >= 2 * first - 65536 and torch.cuda.max_memory_allocated() <= before - first + held(ctx) + again.numel() * 2 + rest(ctx)
    _close(pb, q, again, 0.1)
    larger = ku.make_context(longer)
    larger.scratch = ctx.scratch
    q, out = torch.randn((9100, 16, 128), device=DEV).bfloat16(), torch.empty((9100, 16, 128), dtype=torch.bfloat16, device=DEV)
    ctx.step_cache.clear()
    torch.cuda.synchronize()
    before, old = torch.cuda.memory_allocated(), held(ctx)
    torch.cuda.reset_peak_memory_stats()
    ops.attention(out, q, longer.k8, longer.v8, larger, 0, 0.1, None)
    assert held(larger) > old and torch.cuda.max_memory_allocated() <= before - old + held(larger) + rest(larger)


@pytest.mark.parametrize("nq,nkv,d", [(16, 8, 128), (16, 2, 64)])
@pytest.mark.parametrize("window", [None, 40])
def test_a_captured_prompt_s_beginning_that_changes_on_the_device(nq, nkv, d, window):
    """As many pages or fewer as the host counted: right. More: the status word, and nothing outside the scratch is looked at."""
    pb = cu.Batch8([(400, 500), (500, 400), (0, 150)], 16, nkv, d, seed=8)
    whole, ctx = list(pb.rows), ku.make_context(pb)
    first = [(200, 500), (100, 400), (0, 150)]
    ctx.host_q_start = [s for s, _ in first]
    ctx.q_start.copy_(torch.tensor(ctx.host_q_start, dtype=torch.int32))
    pb.rows = first
    q, out = _attend(pb, nq, d, 0.1, window, ctx=ctx)
    assert "cache8_pages" in ctx.scratch
    _close(pb, q, out, 0.1, window)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ctx.stream = torch.cuda.current_stream().cuda_stream
        ops.attention(out, q, pb.k8, pb.v8, ctx, 0, 0.1, window)
    fits = [[200, 100, 0], [0, 300, 0], [0, 0, 0], [100, 200, 0]]
    for starts in fits + ([] if window else [[s for s, _ in whole], [400, 100, 0], [0, 500, 0], [200, 101 + 16, 0]]) + [[0, 1, 0]]:
        ctx.q_start.copy_(torch.tensor(starts, dtype=torch.int32))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        pages = sum(-(-(s + n) // 16) - (max(0, s - (window or 0) + 1) // 16 if window else 0) for s, (_, n) in zip(starts, whole))
        counted = sum(-(-(s + n) // 16) - (max(0, s - (window or 0) + 1) // 16 if window else 0) for s, n in first)
        assert pb.status.item() == (2 if pages > counted else 0), starts
        pb.status.zero_()
        if pages <= counted:
            pb.rows = [(s, n) for s, (_, n) in zip(starts, whole)]
            _close(pb, q, out, 0.1, window)


@pytest.mark.parametrize("nq,nkv,d,rows", PROMPTS + [(16, 8, 128, [(9000, 300)])])
def test_a_stream_of_its_own_while_the_current_one_is_busy(nq, nkv, d, rows):
    """All that a first call makes, counters that a kernel finds zero among it, is made on the step's stream: what lies on the current one may come much later."""
    pb = cu.Batch8(rows, 16, nkv, d, seed=8)
    q, want = _attend(pb, nq, d, 0.1)
    side, out, ctx = torch.cuda.Stream(), torch.full_like(q, float("nan")), ku.make_context(pb)
    torch.cuda.synchronize()
    torch.cuda._sleep(50_000_000)
    ctx.stream = side.cuda_stream
    ops.attention(out, q, pb.k8, pb.v8, ctx, 0, 0.1, None)
    with torch.cuda.stream(side):
        assert torch.equal(out, want)
