"""Low-rank adapters of many requests beside a shared product, against the formula in 64 bits."""

from __future__ import annotations

import pytest
import torch

from . import adapters_util as au

pytestmark = pytest.mark.gpu

ONE = [(1, 2)]
EIGHT = [(1, 0), (1, 3), (1, 3), (1, 1), (1, -1), (1, 0), (1, 2), (1, 1)]
DECODE64 = [(1, (7 * i) % 5 - 1) for i in range(64)]
MIXED = [(1, i % 4) for i in range(20)] + [(0, 1), (157, 2), (1, -1), (33, 0)]
PROMPTS = [(300, 1), (7, -1), (255, 3), (1, 0), (513, 1)]
LONG = [(1531, 3), (517, 1)]


def run_linear(x, w, low, rows, out_dtype=None, stream=None):
    from miniserve_b200 import ops

    out = torch.full((x.shape[0], w.shape[0]), float("nan"), dtype=out_dtype or x.dtype, device=x.device)
    ops.linear(x, w, out=out, low_rank=low, adapter_rows=rows, stream=stream)
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,k,parts,rank", [
    (ONE, 1024, (256, 128, 128), 16), (ONE, 12288, (512,), 8), (ONE, 8, (3,), 8), (ONE, 2048, (1001,), 256),
    (EIGHT, 1024, (256, 128, 128), 16), (EIGHT, 4096, (1024,), 64), (EIGHT, 6144, (264, 8), 24), (EIGHT, 40, (37,), 8),
    (DECODE64[:16], 1000, (700, 40, 40), 16), (EIGHT, 2048, (72, 24, 8, 1), 32), (DECODE64[:9], 4096, (512,), 8), (DECODE64[:13], 2504, (96, 40), 24), (DECODE64, 512, (384, 64, 64), 32), (DECODE64[:17], 2048, (512,), 16), (DECODE64[:33], 4104, (200, 72, 24, 8), 40),
    (MIXED, 1024, (512, 256, 256), 16), (MIXED, 520, (100, 28), 136), (MIXED, 64, (77,), 8),
    (PROMPTS, 256, (256, 128, 128), 8), (PROMPTS, 1024, (640, 24), 72),
])
def test_linear(dtype, rows, k, parts, rank):
    x, w, low, ar = au.made(rows, k, parts, rank, 4, dtype, seed=len(rows) + k)
    want, tol = au.formula(x, w, low, ar)
    au.close(run_linear(x, w, low, ar), want, tol)
    if dtype is torch.bfloat16:
        au.close(run_linear(x, w, low, ar, torch.float32), want, tol)


@pytest.mark.parametrize("rows,k,parts,rank", [(LONG, 1024, (4096,), 16), (LONG, 1024, (2048, 1024, 1024), 16), (PROMPTS + LONG, 1024, (3000, 1000, 96), 24),
                                               (LONG + EIGHT, 512, (6144,), 136), (DECODE64 + LONG, 1024, (4096, 128), 8)])
def test_linear_of_whole_prompts(rows, k, parts, rank):
    x, w, low, ar = au.made(rows, k, parts, rank, 4, torch.bfloat16, seed=k)
    want, tol = au.formula(x, w, low, ar)
    au.close(run_linear(x, w, low, ar), want, tol)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,k,inter,rank,parts", [
    (DECODE64[:16], 1024, 1500, 16, 2), (EIGHT, 2048, 200, 32, 2), (DECODE64[:9], 72, 5, 24, 1), (DECODE64[:25], 256, 9728, 24, 2), (DECODE64[:60], 128, 9500, 8, 2),
    (ONE, 1024, 512, 16, 2), (EIGHT, 1024, 264, 16, 2), (EIGHT, 4096, 1024, 64, 2), (EIGHT, 2048, 96, 8, 1), (DECODE64[:17], 512, 1024, 16, 2), (DECODE64, 1024, 1000, 32, 2),
    (MIXED, 512, 136, 16, 2), (PROMPTS, 256, 1024, 24, 2)])
def test_silu_mul(dtype, rows, k, inter, rank, parts):
    from miniserve_b200 import ops

    x, w, low, ar = au.made(rows, k, (inter, inter) if parts == 2 else (2 * inter,), rank, 4, dtype, seed=inter)
    out = torch.full((x.shape[0], inter), float("nan"), dtype=dtype, device="cuda")
    ops.linear_silu_mul(x, w, out, low_rank=low, adapter_rows=ar)
    au.close(out, *au.gated(*au.formula(x, w, low, ar), dtype))


@pytest.mark.parametrize("rows,k,inter,rank,parts", [(LONG, 1024, 2048, 16, 2), (PROMPTS + LONG, 512, 2056, 72, 2), (LONG, 512, 4096, 8, 1)])
def test_silu_mul_of_whole_prompts(rows, k, inter, rank, parts):
    from miniserve_b200 import ops

    x, w, low, ar = au.made(rows, k, (inter, inter) if parts == 2 else (2 * inter,), rank, 4, torch.bfloat16, seed=inter)
    out = torch.full((x.shape[0], inter), float("nan"), dtype=torch.bfloat16, device="cuda")
    ops.linear_silu_mul(x, w, out, low_rank=low, adapter_rows=ar)
    au.close(out, *au.gated(*au.formula(x, w, low, ar), torch.bfloat16))


@pytest.mark.parametrize("rows,n", [(EIGHT, 512), (DECODE64, 512), (LONG, 4096)])
def test_a_token_that_is_not_a_number_spoils_its_own_row_alone(rows, n):
    x, w, low, ar = au.made(rows, 512, (n,), 16, 4, torch.bfloat16)
    clean = run_linear(x, w, low, ar)
    bad = x.shape[0] // 2
    x[bad, 3] = float("nan")
    x[bad + 1, 5] = float("inf")
    spoilt = run_linear(x, w, low, ar)
    keep = torch.ones(x.shape[0], dtype=torch.bool, device="cuda")
    keep[bad:bad + 2] = False
    assert torch.equal(spoilt[keep], clean[keep]) and bool(spoilt[bad].isnan().all()) and not bool(spoilt[bad + 1].isfinite().any())


def test_tokens_without_adapters_and_steps_without_tokens():
    from miniserve_b200 import ops

    x, w, low, ar = au.made([(5, -1), (1, -7)], 256, (128,), 8, 2, torch.bfloat16)
    au.close(run_linear(x, w, low, ar), *au.formula(x, w, low, ar))
    x, w, low, ar = au.made([(0, 1), (0, -1)], 256, (128,), 8, 2, torch.bfloat16)
    assert run_linear(x, w, low, ar).shape == (0, 128)
    out = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda")
    assert ops.linear_silu_mul(x, w, out, low_rank=low, adapter_rows=ar).shape == (0, 64)


@pytest.mark.parametrize("rows", [EIGHT, DECODE64, MIXED, LONG])
def test_a_slot_that_is_not_there_raises_the_status_word(rows):
    from miniserve_b200 import ops

    x, w, low, ar = au.made(rows, 256, (4096,), 8, 4, torch.bfloat16)
    status = ops.device_status("cuda")
    assert int(status) == 0
    ar.slot_of_row[-1] = 4
    ar = ops.AdapterRows(ar.slot_of_row, ar.row_of_token)
    try:
        got = run_linear(x, w, low, ar)
        assert int(status) == 6
    finally:
        status.zero_()
    au.close(got, *au.formula(x, w, low, ar))  # (the formula counts such a token as one without an adapter)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [EIGHT, DECODE64, MIXED, LONG])
def test_the_same_call_gives_the_same_bits(dtype, rows):
    x, w, low, ar = au.made(rows, 1024, (2048, 1024, 1024), 16, 4, dtype)
    assert torch.equal(run_linear(x, w, low, ar), run_linear(x, w, low, ar))


def test_32_bit_rows_do_not_depend_on_the_step_around_them():
    x, w, low, ar = au.made(PROMPTS, 1032, (300, 100), 24, 4, torch.float32)
    whole, at = run_linear(x, w, low, ar), 0
    for i, (n, slot) in enumerate(PROMPTS):
        for a, b in ((0, 1), (0, n)):
            part = run_linear(x[at + a:at + b].contiguous(), w, low, au.rows_of([(b - a, slot)]))
            assert torch.equal(part, whole[at + a:at + b]), (i, a, b)
        at += n


def test_another_stream_than_the_current_one():
    x, w, low, ar = au.made(MIXED, 1024, (512, 256), 16, 4, torch.bfloat16)
    want, tol = au.formula(x, w, low, ar)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [run_linear(x, w, low, ar, stream=side.cuda_stream) for _ in range(3)]
    noise = [torch.full((x.shape[0], 64), float("nan"), device="cuda") for _ in range(20)]  # memory that the current stream takes meanwhile
    side.synchronize()
    for out in outs:
        au.close(out, want, tol)
    assert len(noise) == 20


@pytest.mark.parametrize("rows", [EIGHT, DECODE64, LONG])
def test_a_captured_call_follows_its_inputs(rows):
    """Two graphs of one projection, replayed in turn, each with other tokens and other slots than it was captured with."""
    from miniserve_b200 import ops

    held = [au.made(rows, 1024, (2048, 1024, 1024), 16, 4, torch.bfloat16, seed=s) for s in (1, 2)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for x, w, low, ar in held:
        out = torch.empty((x.shape[0], 4096), dtype=torch.bfloat16, device="cuda")
        with torch.cuda.stream(side):
            ops.linear(x, w, out=out, low_rank=low, adapter_rows=ar)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            rows_in = ops.AdapterRows(ar.slot_of_row, ar.row_of_token)
            ops.linear(x, w, out=out, low_rank=low, adapter_rows=rows_in)
        graphs.append((graph, rows_in))
        outs.append(out)
    for turn in range(3):
        for (graph, _), out, (x, w, low, ar) in zip(graphs, outs, held):
            ar.slot_of_row.copy_(torch.roll(ar.slot_of_row, 1 + turn))
            x.copy_(torch.randn_like(x))
            out.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            au.close(out, *au.formula(x, w, low, ar))


# 8 and 16 tokens beside a weight of 128 MiB: the product's own warps make v (counters that a launch has to itself)
@pytest.mark.parametrize("tokens", [8, 16])
def test_own_terms_on_two_streams_at_once(tokens):
    """Calls of two streams with the same AdapterRows, more than a stretch of counters holds, against the same calls one after the other."""
    from miniserve_b200 import ops

    k, n = 4096, 16384
    assert ops.adapters.makes_its_own(8 * tokens, 2 * k * n >> 20)
    x, w, low, ar = au.made([(1, i % 3 - (i == 5)) for i in range(tokens)], k, (n,), 8, 3, torch.bfloat16)
    want, tol = au.formula(x, w, low, ar)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[torch.full((tokens, n), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(150)] for _ in streams]
    torch.cuda.synchronize()
    for i in range(150):
        for s, out in zip(streams, outs):
            ops.linear(x, w, out=out[i], low_rank=low, adapter_rows=ar, stream=s.cuda_stream)
    torch.cuda.synchronize()
    au.close(outs[0][0], want, tol)
    first = outs[0][0]
    assert all(torch.equal(o, first) for out in outs for o in out) and int(ops.device_status("cuda")) == 0


def test_own_terms_of_many_captured_calls():
    """More calls in one graph than a stretch of counters holds, replayed; another graph of the same AdapterRows in between."""
    from miniserve_b200 import ops

    x, w, low, ar = au.made(EIGHT, 4096, (16384,), 8, 4, torch.bfloat16)
    assert ops.adapters.makes_its_own(64, 128)
    side = torch.cuda.Stream()
    graphs = []
    with torch.cuda.stream(side):
        ops.linear(x, w, low_rank=low, adapter_rows=ar)
    side.synchronize()
    for calls in (ops.adapters.TICKETS + 20, 3):
        outs = [torch.empty((8, 16384), dtype=torch.bfloat16, device="cuda") for _ in range(calls)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            for out in outs:
                ops.linear(x, w, out=out, low_rank=low, adapter_rows=ar)
        graphs.append((graph, outs))
    for turn in range(4):
        x.copy_(torch.randn_like(x))
        graph, outs = graphs[turn % 2]
        for out in outs:
            out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        au.close(outs[0], *au.formula(x, w, low, ar))
        assert all(torch.equal(out, outs[0]) for out in outs)
    assert int(ops.device_status("cuda")) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_tokens_than_a_grid_has_rows(dtype):
    """70,000 tokens (beyond 65,535) of a few requests; the formula at some of them."""
    rows = [(1, 2), (65535, 1), (1, -1), (4000, 0), (463, 3)]
    x, w, low, ar = au.made(rows, 64, (128,), 8, 4, dtype)
    got = run_linear(x, w, low, ar)
    at = torch.tensor([0, 1, 2, 255, 256, 32767, 65535, 65536, 65537, 65538, 69536, 69537, 69999], device="cuda")
    from miniserve_b200 import ops

    want, tol = au.formula(x[at], w, low, ops.AdapterRows(ar.slot_of_row, ar.row_of_token[at].contiguous()))
    au.close(got[at], want, tol)
    plain = x.double() @ w.double().T
    none = torch.nonzero(ar.slot_of_row[ar.row_of_token.long()] < 0)[:, 0]
    assert none.tolist() == [65536] and bool(((got - plain).abs().amax(1) > 0.05).sum() > 69000)


@pytest.mark.parametrize("rows", [EIGHT, DECODE64, MIXED, LONG])
def test_a_row_that_is_not_there_raises_the_status_word(rows):
    from miniserve_b200 import ops

    x, w, low, ar = au.made(rows, 256, (4096,), 8, 4, torch.bfloat16)
    status, last = ops.device_status("cuda"), ar.rows
    of_token = ar.row_of_token.clone()
    of_token[0], of_token[-1] = -3, last
    try:
        got = run_linear(x, w, low, ops.AdapterRows(ar.slot_of_row, of_token))
        assert int(status) == 6
    finally:
        status.zero_()
    slots = torch.cat([ar.slot_of_row, torch.full((1,), -1, dtype=torch.int32, device="cuda")])
    of_token[0] = last
    au.close(got, *au.formula(x, w, low, ops.AdapterRows(slots, of_token)))


@pytest.mark.parametrize("way,rows", [("stream", EIGHT), ("decode", EIGHT), ("decode", DECODE64), ("pair", DECODE64[:5]), ("pair", PROMPTS), ("apart", ONE), ("apart", PROMPTS)])
@pytest.mark.parametrize("gated", [False, True])
def test_every_way_takes_sizes_that_the_rule_sends_elsewhere(way, rows, gated, monkeypatch):
    from miniserve_b200 import ops

    monkeypatch.setattr(ops.adapters, "WAY", way)
    k, parts = (4096, (520, 520)) if gated else (4096, (264, 96, 72))
    x, w, low, ar = au.made(rows, k, parts, 40, 4, torch.bfloat16, seed=3)
    want, tol = au.formula(x, w, low, ar)
    if gated:
        out = torch.full((x.shape[0], 520), float("nan"), dtype=torch.bfloat16, device="cuda")
        ops.linear_silu_mul(x, w, out, low_rank=low, adapter_rows=ar)
        au.close(out, *au.gated(want, tol, torch.bfloat16))
    else:
        au.close(run_linear(x, w, low, ar), want, tol)


def test_offsets_beyond_32_bits():
    """More than 2^31 numbers of B: the last slot's."""
    from miniserve_b200 import ops

    k, n, rank, slots = 64, 65536, 256, 136
    gen = torch.Generator(device="cuda").manual_seed(5)
    low = ops.LowRank(torch.zeros((slots, rank, k), dtype=torch.bfloat16, device="cuda"), torch.zeros((slots, n, rank), dtype=torch.bfloat16, device="cuda"),
                      torch.ones(slots, device="cuda"), (n,))
    assert low.b.numel() > 1 << 31
    low.a[-1] = torch.randn((rank, k), generator=gen, device="cuda").bfloat16()
    low.b[-1] = (torch.randn((n, rank), generator=gen, device="cuda") / 16).bfloat16()
    for tokens in (1, 300):
        x = torch.randn((tokens, k), generator=gen, device="cuda").bfloat16()
        w = torch.randn((n, k), generator=gen, device="cuda").bfloat16()
        ar = au.rows_of([(tokens, slots - 1)])
        got = run_linear(x, w, low, ar)
        want, tol = au.formula(x, w, low, ar)
        au.close(got, want, tol)


def test_refusals_on_the_device():
    from miniserve_b200 import ops

    x, w, low, ar = au.made(EIGHT, 256, (128,), 8, 4, torch.bfloat16)
    with pytest.raises(ValueError, match="contiguous"):
        ops.linear(x[:, ::2], w[:, ::2].contiguous(), low_rank=ops.LowRank(low.a[:, :, ::2].contiguous(), low.b, low.scale, low.ends), adapter_rows=ar)
    with pytest.raises(ValueError, match="out is"):
        ops.linear(x, w, out=torch.empty((8, 127), dtype=torch.bfloat16, device="cuda"), low_rank=low, adapter_rows=ar)
    with pytest.raises(ValueError, match="one device"):
        ops.linear(x, w, low_rank=low, adapter_rows=au.rows_of(EIGHT, "cpu"))
    with pytest.raises(ValueError, match="16 bytes"):
        shifted = torch.empty(8 * 256 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(8, 256)
        ops.linear(shifted, w, low_rank=low, adapter_rows=ar)
    with pytest.raises(ValueError, match="weight on 16 bytes"):
        ops.linear(x, torch.empty(128 * 256 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(128, 256), low_rank=low, adapter_rows=ar)
    with pytest.raises(ValueError, match="on 16 bytes"):
        ops.linear(x, w, out=torch.empty(8 * 128 + 1, dtype=torch.float32, device="cuda")[1:].view(8, 128), low_rank=low, adapter_rows=ar)


@pytest.mark.parametrize("rows,rank,full", [(LONG[:1], 16, False), (LONG, 16, True), (PROMPTS, 72, True), (DECODE64 + PROMPTS, 8, True), ([(40, 1)], 24, False)])
def test_qkv_with_norm_rotation_and_cache_write_behind(rows, rank, full):
    """The q|k|v product's epilogue works on the adapted product: against the formula in 64 bits, carried through norm and rotation. The tolerance follows
    the product's through them: a norm's factor moves with the mean of squares, a rotated number with both of its pair (first order, 5 % for the rest)."""
    from miniserve_b200 import ops

    from .kernel_util import PagedBatch

    nq, nkv, d, page, hidden, eps = 4, 2, 128, 16, 1024, 1e-6
    pb = PagedBatch([(3 * i, n) for i, (n, _) in enumerate(rows)], page, nkv, d, torch.bfloat16, seed=3)
    x, w, low, ar = au.made(rows, hidden, (nq * d, nkv * d, nkv * d), rank, 4, torch.bfloat16, seed=rank)
    t = x.shape[0]
    gen = torch.Generator(device="cuda").manual_seed(1)
    qw, kw = ((1 + 0.1 * torch.randn((d,), generator=gen, device="cuda")).bfloat16() for _ in range(2)) if full else (None, None)
    inv_freq = (1.0 / (1e6 ** (torch.arange(0, d, 2, dtype=torch.float64) / d))).float().cuda()
    table = ops.rope_table(pb.positions, inv_freq, t, d) if full else None
    q = torch.full((t, nq, d), float("nan"), dtype=torch.bfloat16, device="cuda")
    ops.qkv_norm_rope_kv(q, pb.k_pool, pb.v_pool, x, w, qw, kw, ops.rope_table_tiled(table) if full else None, eps, pb.positions, pb.row_of_token, pb.page_indptr,
                         pb.page_indices, page, low_rank=low, adapter_rows=ar)
    y, tol = (z.view(t, nq + 2 * nkv, d) for z in au.formula(x, w, low, ar))
    want, off = [y[:, :nq], y[:, nq:nq + nkv], y[:, nq + nkv:]], [tol[:, :nq], tol[:, nq:nq + nkv], tol[:, nq + nkv:]]
    if full:
        cos, sin = table[:, None, :d // 2].double(), table[:, None, d // 2:].double()
        for i, weight in enumerate((qw, kw)):
            v, dv, g = want[i], off[i], weight.double()
            inv = (v * v).mean(-1, keepdim=True).add(eps).rsqrt()
            v, dv = v * inv * g, 1.05 * g.abs() * (inv * dv + v.abs() * inv ** 3 * (v.abs() * dv).mean(-1, keepdim=True))
            (lo, hi), (dlo, dhi) = v.chunk(2, -1), dv.chunk(2, -1)
            want[i] = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
            off[i] = torch.cat([dlo * cos.abs() + dhi * sin.abs(), dhi * cos.abs() + dlo * sin.abs()], -1) + (2.0 ** -8 + 2.0 ** -18) * v.abs().amax(-1, keepdim=True) * 1.42
    au.close(q, want[0], off[0])
    at = 0
    for r, (start, n) in enumerate(pb.rows):
        for pool, i in ((pb.k_pool, 1), (pb.v_pool, 2)):
            got = pb.read(r, pool, start + n)[start:]
            au.close(got, want[i][at:at + n], off[i][at:at + n])
        at += n
    assert int(ops.device_status("cuda")) == 0
