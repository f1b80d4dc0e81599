"""Sampling with temperature, top-k, top-p and min-p from given random numbers, token for token against lists in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def plain(logits, t, u, k=0, p=1.0, m=0.0):
    """The token of one row by the definition, on the host in 64 bits."""
    z = logits.double().cpu()
    z = torch.where(z.isnan(), -math.inf, z)
    top = float(z.max())
    if top == -math.inf:
        return 0
    if not t > 0:
        return int((z == top).nonzero()[0, 0])
    w = torch.where(z == top, 1.0, torch.exp((z - top) / t)) if math.isfinite(top) else (z == top).double()
    w = torch.where(z == -math.inf, 0.0, w)
    order = torch.argsort(z, descending=True, stable=True)
    if 0 < k < z.numel():
        order = order[:k]
    if p < 1:
        sums = torch.cumsum(w[order], 0)
        keep = sums - w[order] < p * float(sums[-1])
        keep[0] = True
        order = order[keep]
    kept = torch.sort(order[w[order] >= min(m, 1.0)]).values
    sums = torch.cumsum(w[kept], 0)
    return int(kept[min(int((sums <= u * float(sums[-1])).sum()), kept.numel() - 1)])


def draw(logits, t, u, k=None, p=None, m=None, dtype=torch.float64, before=-5):
    """Tokens of rows with settings given as numbers or lists."""
    from miniserve_b200 import ops

    rows = logits.shape[0]

    def row(x, dt):
        return None if x is None else torch.tensor([x] * rows if not isinstance(x, (list, tuple)) else list(x), dtype=dt, device="cuda")

    tokens = torch.full((rows,), before, dtype=torch.int32, device="cuda")
    ops.sample_filtered(tokens, logits, row(t, torch.float32), row(u, dtype), top_k=row(k, torch.int32), top_p=row(p, torch.float32), min_p=row(m, torch.float32))
    return tokens.tolist()


def f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def peaked(rows, vocab, seed, std=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn((rows, vocab), generator=gen, device="cuda") * std
    at = torch.randint(0, vocab, (rows, min(vocab, 16)), generator=gen, device="cuda")
    return logits.scatter_add_(1, at, 10 * torch.rand(at.shape, generator=gen, device="cuda")), gen


SETTINGS = [dict(), dict(k=1), dict(k=3), dict(k=40), dict(k=100000), dict(p=0.9), dict(p=0.3), dict(p=0.999), dict(m=0.1), dict(m=0.9), dict(k=20, p=0.8),
            dict(k=50, p=0.9, m=0.05), dict(p=0.95, m=0.02), dict(k=5, m=0.2)]


@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 4097, 50000, 151936, 400003, 1 << 20])
@pytest.mark.parametrize("t", [0.7, 1.0, 3.0])
def test_tokens(vocab, t):
    rows = len(SETTINGS)
    logits, gen = peaked(rows, vocab, vocab)
    u = torch.rand((rows,), generator=gen, device="cuda", dtype=torch.float64).tolist()
    ks, ps, ms = ([s.get(n, d) for s in SETTINGS] for n, d in (("k", 0), ("p", 1.0), ("m", 0.0)))
    got = draw(logits, t, u, ks, ps, ms)
    assert got == [plain(logits[i], f32(t), u[i], ks[i], f32(ps[i]), f32(ms[i])) for i in range(rows)]


@pytest.mark.parametrize("vocab,rows", [(1000, 300), (32001, 70), (151936, 64)])
def test_many_rows_of_settings_of_their_own(vocab, rows):
    logits, gen = peaked(rows, vocab, rows)
    r = torch.rand((5, rows), generator=gen, device="cuda", dtype=torch.float64).cpu()
    t = [0.0 if x < 0.1 else f32(0.2 + 1.5 * x) for x in r[0].tolist()]
    k = [0 if x < 0.4 else int(1 + 200 * x ** 3) for x in r[1].tolist()]
    p = [1.0 if x < 0.4 else f32(x) for x in r[2].tolist()]
    m = [0.0 if x < 0.5 else f32(0.3 * x) for x in r[3].tolist()]
    u = r[4].tolist()
    assert draw(logits, t, u, k, p, m) == [plain(logits[i], t[i], u[i], k[i], p[i], m[i]) for i in range(rows)]


def test_one_filter_at_a_time_is_an_argument_left_out():
    logits, gen = peaked(6, 5000, 3)
    u = torch.rand((6,), generator=gen, device="cuda", dtype=torch.float64).tolist()
    for kw in (dict(), dict(k=7), dict(p=0.8), dict(m=0.1)):
        full = {n: f32(v) if n != "k" else v for n, v in kw.items()}
        assert draw(logits, 0.9, u, **kw) == [plain(logits[i], f32(0.9), u[i], **full) for i in range(6)]


@pytest.mark.parametrize("digits", [torch.bfloat16, "whole", "same"])
@pytest.mark.parametrize("vocab", [100, 20000, 151936])
def test_ties_go_by_the_vocabulary(digits, vocab):
    """Logits of few different values: cuts fall inside a run of equals."""
    logits, gen = peaked(len(SETTINGS), vocab, 11)
    logits = logits.to(digits).float() if isinstance(digits, torch.dtype) else torch.round(logits) if digits == "whole" else torch.full_like(logits, 1.25)
    u = torch.rand((len(SETTINGS),), generator=gen, device="cuda", dtype=torch.float64).tolist()
    ks, ps, ms = ([s.get(n, d) for s in SETTINGS] for n, d in (("k", 0), ("p", 1.0), ("m", 0.0)))
    assert draw(logits, 1.0, u, ks, ps, ms) == [plain(logits[i], 1.0, u[i], ks[i], f32(ps[i]), f32(ms[i])) for i in range(len(SETTINGS))]


def test_half_of_equal_tokens():
    logits = torch.zeros((8, 64), device="cuda")
    u = [i / 8 for i in range(8)]
    assert draw(logits, 1.0, u, p=0.5) == [4 * i for i in range(8)]  # tokens 0 .. 31
    assert draw(logits, 1.0, u, k=16) == [2 * i for i in range(8)]
    assert draw(logits, 1.0, u, k=16, p=0.5) == list(range(8))


def test_the_ends_of_the_random_numbers():
    logits, _ = peaked(1, 3000, 5)
    one = 1 - 2.0 ** -53
    for kw in (dict(), dict(k=10), dict(p=0.7), dict(m=0.3)):
        full = {n: f32(v) if n != "k" else v for n, v in kw.items()}
        assert draw(logits, 1.0, [0.0], **kw) == [plain(logits[0], 1.0, 0.0, **full)]
        assert draw(logits, 1.0, [one], **kw) == [plain(logits[0], 1.0, one, **full)]
    gen = torch.Generator().manual_seed(1)
    u = torch.rand((64,), generator=gen)
    logits, _ = peaked(64, 3000, 6)
    assert draw(logits, 1.0, u.tolist(), p=0.9, dtype=torch.float32) == [plain(logits[i], 1.0, float(u[i]), p=f32(0.9)) for i in range(64)]


def test_rows_without_a_random_number_keep_their_token():
    logits, _ = peaked(6, 500, 7)
    u = [0.5, -1.0, math.nan, 1.0, math.inf, -math.inf]
    got = draw(logits, [1.0] * 6, u, k=5, before=77)
    assert got[1:] == [77] * 5 and got[0] == plain(logits[0], 1.0, 0.5, k=5)
    assert draw(logits, 0.0, u, before=77)[1:] == [77] * 5


def test_settings_outside_their_ranges():
    """What the documentation says of them: nothing is left out by k <= 0 or beyond the vocabulary, top_p >= 1 or NaN, min_p <= 0 or NaN; one token at least stays."""
    logits, _ = peaked(1, 700, 8)
    row = lambda **kw: draw(logits, 1.0, [0.73], **kw)  # noqa: E731
    free = [plain(logits[0], 1.0, 0.73)]
    for kw in (dict(k=-3), dict(k=0), dict(k=700), dict(k=2 ** 31 - 1), dict(p=1.0), dict(p=7.0), dict(p=math.nan), dict(p=math.inf), dict(m=0.0), dict(m=-1.0), dict(m=math.nan)):
        assert row(**kw) == free, kw
    best = [int(logits[0].argmax())]
    for kw in (dict(k=1), dict(p=0.0), dict(p=-1.0), dict(p=-math.inf), dict(p=1e-30), dict(m=1.0), dict(m=50.0), dict(m=math.inf)):
        assert row(**kw) == best, kw
    for t in (0.0, -1.0, math.nan):
        assert draw(logits, t, [0.73]) == best
    assert draw(logits, 1e-38, [0.73], p=0.9) == best and draw(logits, 1e-45, [0.73], k=9) == best
    assert draw(logits, math.inf, [0.73]) == [plain(logits[0], math.inf, 0.73)]


@pytest.mark.parametrize("vocab", [40, 30000])
def test_rows_of_numbers_that_are_not_finite(vocab):
    inf, nan, low = math.inf, math.nan, torch.finfo(torch.float32).min
    base, _ = peaked(1, vocab, 9)
    base = base[0]

    def with_(*pairs, fill=None):
        x = base.clone() if fill is None else torch.full_like(base, fill)
        for i, v in pairs:
            x[i] = v
        return x

    logits = torch.stack([
        with_(fill=-inf), with_(fill=nan), with_((3, 1.0), fill=-inf), with_((5, 2.0), (17, 2.0), fill=nan), with_((4, inf)), with_((4, inf), (9, inf), (30, nan)),
        with_((0, nan), (1, -inf), (2, low)), with_((7, -3.0), (8, -3.5), fill=low), with_(fill=low), with_((6, -0.0), (7, 0.0), fill=-inf), with_((2, 3e38), (3, -3e38)),
    ])
    n = logits.shape[0]
    for t in (0.0, 0.8, 1.0):
        for u in (0.0, 0.4, 0.9):
            for kw in (dict(), dict(k=1), dict(k=2), dict(k=12), dict(p=0.6), dict(k=9, p=0.6, m=0.1)):
                full = {a: f32(v) if a != "k" else v for a, v in kw.items()}
                assert draw(logits, t, [u] * n, **kw) == [plain(logits[i], f32(t), u, **full) for i in range(n)], (t, u, kw)


def test_a_captured_call_follows_its_inputs_and_another_stream():
    from miniserve_b200 import ops

    logits, gen = peaked(9, 30000, 12)
    new = lambda x, dt: torch.full((9,), x, dtype=dt, device="cuda")  # noqa: E731
    t, u, k, p, m = new(1.0, torch.float32), new(0.5, torch.float64), new(5, torch.int32), new(0.9, torch.float32), new(0.0, torch.float32)
    tokens = new(-1, torch.int32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ops.sample_filtered(tokens, logits, t, u, k, p, m, stream=side.cuda_stream)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.sample_filtered(tokens, logits, t, u, k, p, m)
    for seed in (1, 2, 3):
        other, gen = peaked(9, 30000, seed)
        logits.copy_(other)
        u.copy_(torch.rand((9,), generator=gen, device="cuda", dtype=torch.float64))
        k.copy_(torch.randint(0, 60, (9,), generator=gen, device="cuda"))
        p.copy_(torch.rand((9,), generator=gen, device="cuda") * 0.6 + 0.5)
        t.copy_(torch.rand((9,), generator=gen, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert tokens.tolist() == [plain(logits[i], float(t[i]), float(u[i]), int(k[i]), float(p[i])) for i in range(9)]


def test_refusals():
    from miniserve_b200 import ops

    logits, f, i = torch.zeros((2, 8), device="cuda"), torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    bad = [dict(logits=logits.bfloat16()), dict(logits=logits[:, ::2]), dict(tokens=i.long()), dict(tokens=i[:1]), dict(temperature=f.double()), dict(uniform=i), dict(uniform=f[:1]),
           dict(top_k=f), dict(top_p=i), dict(min_p=f.cpu()), dict(top_p=torch.zeros(4, device="cuda")[::2]), dict(logits=torch.zeros((2, 0), device="cuda"))]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.sample_filtered(**{**dict(tokens=i, logits=logits, temperature=f, uniform=f), **kw})
    ops.sample_filtered(i[:0], logits[:0], f[:0], f[:0])
