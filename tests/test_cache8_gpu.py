"""The 8-bit paged cache: its kernels alone against 64-bit arithmetic, refusals, and the operators one behind the other."""

from __future__ import annotations

import math

import pytest
import torch

from miniserve_b200 import ops
from tests import cache8_util as cu
from tests import kernel_util as ku

pytestmark = pytest.mark.gpu
DEV = "cuda"


# ------------------------------------------------------------------ write
def _projection(tokens, nq, nkv, d, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn((tokens, (nq + 2 * nkv) * d), generator=gen, device=DEV).mul_(1.5).bfloat16(), gen


def _turn64(x, w, eps, cos, sin, rot):
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    if rot:
        half = rot // 2
        lo, hi = x[..., :half], x[..., half:rot]
        c, s = cos[:, None].double(), sin[:, None].double()
        x = torch.cat([lo * c - hi * s, hi * c + lo * s, x[..., rot:]], -1)
    return x


@pytest.mark.parametrize("nq,nkv,d,page,norm,rot,rows", [
    (16, 8, 128, 16, True, 128, [(0, 5), (1030, 1), (77, 33)]),
    (4, 2, 64, 16, True, 64, [(0, 1)]),
    (4, 1, 64, 8, False, 64, [(3, 40), (0, 7)]),
    (6, 3, 48, 32, True, 24, [(9, 12)]),
    (5, 5, 80, 16, True, 80, [(0, 17), (500, 1)]),
    (8, 2, 256, 16, True, 256, [(15, 18)]),
    (2, 2, 16, 64, False, 0, [(0, 100)]),
    (32, 8, 128, 16, False, 128, [(31, 130)]),
    (7, 1, 128, 16, True, 128, [(0, 3), (16, 16), (8, 1)]),
])
@pytest.mark.parametrize("table", [True, False])
def test_write(nq, nkv, d, page, norm, rot, rows, table):
    pb = ku.PagedBatch(rows, page, nkv, d, torch.bfloat16, seed=d)
    t = pb.num_tokens
    qkv, gen = _projection(t, nq, nkv, d, seed=d + nq)
    wq, wk = ((1 + 0.3 * torch.randn((2, d), generator=gen, device=DEV)).bfloat16().unbind() if norm else (None, None))
    wq, wk = (None if w is None else w.clone() for w in (wq, wk))
    inv = (1e4 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / max(rot, 1))).float() if rot else None
    cos = sin = cs = None
    if rot:
        angle = (pb.positions.float()[:, None] * inv).double()  # the contract: the angle is a float32 product
        cos, sin = angle.cos(), angle.sin()
        cs = torch.cat([cos, sin], -1).float().contiguous() if table else None
    k8, v8 = ops.Pool8.empty(pb.num_pages, nkv, page, d), ops.Pool8.empty(pb.num_pages, nkv, page, d)
    for pool in (k8, v8):
        pool.codes.fill_(0xA5)
        pool.exponents.fill_(0xA5)
    q = torch.empty((t, nq, d), dtype=torch.bfloat16, device=DEV)
    ops.qk_norm_rope_kv(q, k8, v8, qkv, wq, wk, inv, rot, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, page, pb.status, cos_sin=cs)
    assert pb.status.item() == 0
    x = qkv.double().view(t, nq + 2 * nkv, d)
    q64 = _turn64(x[:, :nq], wq, 1e-6, cos, sin, rot)
    # float32 arithmetic: a norm (a sum of d squares, a root, two products) and a rotation, some 20 roundings; CUDA's sine and cosine of the angle 2 ulp
    slack = 32 * 2.0 ** -24
    assert bool(((q.double() - q64).abs() <= 2.0 ** -8 * q64.abs() + slack * q64.abs().amax(-1, keepdim=True)).all())
    at = 0
    written = torch.zeros((pb.num_pages, page), dtype=torch.bool, device=DEV)
    for r, (s, n) in enumerate(rows):
        pos = torch.arange(s, s + n)
        pages, slots = torch.tensor([pb.tables[r][p // page] for p in pos.tolist()], device=DEV), (pos % page).to(DEV)
        written[pages, slots] = True
        for pool, y in ((k8, _turn64(x[at:at + n, nq:nq + nkv], wk, 1e-6, None if cos is None else cos[at:at + n], None if sin is None else sin[at:at + n], rot)),
                        (v8, x[at:at + n, nq + nkv:])):
            cu.check_held(pool.codes[pages, :, slots], pool.exponents[pages, :, slots], y, slack)
        at += n
    for pool in (k8, v8):  # every other slot is as it was
        assert bool((pool.codes.permute(0, 2, 1, 3)[~written] == 0xA5).all()) and bool((pool.exponents.transpose(1, 2)[~written] == 0xA5).all())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("which", ["q", "k"])
def test_write_with_one_norm(d, which):
    rows, nq, nkv, page = [(5, 20)], 4, 2, 16
    pb = ku.PagedBatch(rows, page, nkv, d, torch.bfloat16)
    qkv, gen = _projection(20, nq, nkv, d, 4)
    w = (1 + 0.3 * torch.randn(d, generator=gen, device=DEV)).bfloat16()
    k8, v8 = ops.Pool8.empty(pb.num_pages, nkv, page, d), ops.Pool8.empty(pb.num_pages, nkv, page, d)
    q = torch.empty((20, nq, d), dtype=torch.bfloat16, device=DEV)
    wq, wk = (w, None) if which == "q" else (None, w)
    ops.qk_norm_rope_kv(q, k8, v8, qkv, wq, wk, None, 0, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, page, pb.status)
    x, slack = qkv.double().view(20, nq + 2 * nkv, d), 32 * 2.0 ** -24  # (as in test_write)
    q64 = _turn64(x[:, :nq], wq, 1e-6, None, None, 0)
    assert bool(((q.double() - q64).abs() <= 2.0 ** -8 * q64.abs() + slack * q64.abs().amax(-1, keepdim=True)).all())
    pos = torch.arange(5, 25)
    pages, slots = torch.tensor([pb.tables[0][p // page] for p in pos.tolist()], device=DEV), (pos % page).to(DEV)
    cu.check_held(k8.codes[pages, :, slots], k8.exponents[pages, :, slots], _turn64(x[:, nq:nq + nkv], wk, 1e-6, None, None, 0), slack)
    cu.check_held(v8.codes[pages, :, slots], v8.exponents[pages, :, slots], x[:, nq + nkv:], slack)


def test_write_of_values_at_the_format_s_borders():
    """Values (neither normed nor rotated) where rounding, the exponent's choice and its limits show: all bits are known."""
    d, page = 64, 16
    rows = torch.zeros((16, d), dtype=torch.float64)
    rows[0] = 0.0
    rows[1, :3] = torch.tensor([448.0, -448.0, 1.0])  # the largest at exponent 0
    rows[2, :2] = torch.tensor([450.0, 1.0])  # one step of bfloat16 more: exponent 1
    rows[3, 0] = 2.0 ** -100  # below everything: zero
    rows[4, :3] = torch.tensor([1e30, -1e30, 3.0])  # beyond the largest: saturates
    rows[5, 0] = math.inf
    rows[6, 5] = math.nan
    rows[7] = torch.linspace(-3, 3, d, dtype=torch.float64)
    rows[8, :4] = torch.tensor([256.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10])  # codes of the smallest size, ties to even
    rows[9, :3] = torch.tensor([256.0, 17.0, 19.0])  # ties between 16 and 18, 18 and 20
    rows[10, 0] = 57344.0
    rows[11, 0] = -57600.0
    rows[12, 0] = 448 * 2.0 ** -60
    rows[13, 0] = 448 * 2.0 ** -61
    rows[14, :2] = torch.tensor([-math.inf, math.nan])
    rows[15] = -0.0
    v = rows.bfloat16()
    qkv = torch.cat([torch.zeros((16, 2 * d)), v.float()], -1).bfloat16().to(DEV)
    pb = ku.PagedBatch([(0, 16)], page, 1, d, torch.bfloat16)
    k8, v8 = ops.Pool8.empty(pb.num_pages, 1, page, d), ops.Pool8.empty(pb.num_pages, 1, page, d)
    q = torch.empty((16, 1, d), dtype=torch.bfloat16, device=DEV)
    ops.qk_norm_rope_kv(q, k8, v8, qkv, None, None, None, 0, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, page, pb.status)
    codes, exps = v8.codes[pb.tables[0][0], 0].cpu(), v8.exponents[pb.tables[0][0], 0].cpu()
    e = exps.long() - 127
    assert e.tolist()[:7] == [-60, 0, 1, -60, 7, 128, 128] and e[14] == 128 and e[15] == -60 and e[8] == 0 and e[9] == 0
    assert e[10] == 7 and e[11] == 7 and e[12] == -60 and e[13] == -60
    got = cu.values64(codes, exps)
    assert bool((got[0] == 0).all()) and bool((got[3] == 0).all()) and bool((got[15] == 0).all())
    assert got[1, :3].tolist() == [448, -448, 1] and got[4, :3].tolist() == [57344, -57344, 0 + got[4, 2].item()] and got[2, 0].item() == 448
    assert got[8, :4].tolist() == [256, 2.0 ** -9, 0, 2.0 ** -8] and got[9, :3].tolist() == [256, 16, 20]
    assert got[10, 0] == 57344 and got[11, 0] == -57344 and got[12, 0] == 448 * 2.0 ** -60 and got[13, 0] == 224 * 2.0 ** -60
    for r in (5, 6, 14):
        assert bool(got[r].isnan().all()) and bool((codes[r] == 0).all()), "a vector that is not finite reads as NaN and has no code that is one"
    out = torch.empty((16, 1, d), dtype=torch.bfloat16, device=DEV)
    ops.read_cache(torch.empty_like(out), out, k8, v8, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, pb.status)
    assert torch.equal(out[:, 0].cpu().double().nan_to_num(7), got.nan_to_num(7))


# ------------------------------------------------------------------ read
@pytest.mark.parametrize("nkv,d,page,rows", [(8, 128, 16, [(0, 1), (0, 333), (40, 7)]), (1, 16, 8, [(5, 20)]), (3, 80, 32, [(0, 65)]), (2, 256, 64, [(0, 130)]), (4, 64, 16, [(100, 1)])])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_read(nkv, d, page, rows, dtype):
    pb = cu.Batch8(rows, page, nkv, d, seed=d)
    k, v = (torch.empty((pb.num_tokens, nkv, d), dtype=dtype, device=DEV) for _ in range(2))
    ops.read_cache(k, v, pb.k8, pb.v8, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, pb.status)
    at = 0
    for r, (s, n) in enumerate(rows):
        k64, v64 = pb.dense64(r)
        assert torch.equal(k[at:at + n].double(), k64[s:]) and torch.equal(v[at:at + n].double(), v64[s:])  # both types hold every number exactly
        at += n
    assert pb.status.item() == 0


def test_pages_that_are_not_there():
    """A table that is too short, a page given back, a page beyond the pool: the status word, and nothing touched."""
    nkv, d, page = 2, 64, 16
    for bad in ("short", "gone", "beyond"):
        pb = cu.Batch8([(0, 20)], page, nkv, d, seed=3)
        if bad == "short":
            pb.page_indptr = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
        else:
            pb.page_indices[1] = -1 if bad == "gone" else pb.num_pages
        k, v = (torch.full((20, nkv, d), 3.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        ops.read_cache(k, v, pb.k8, pb.v8, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, pb.status)
        assert pb.status.item() == 2 and bool((k[16:] == 3).all()) and bool((v[16:] == 3).all()), bad
        assert torch.equal(k[:16].double(), pb.dense64(0)[0][:16])
        pb.status.zero_()
        before = pb.k8.codes.clone()
        qkv, _ = _projection(20, 2, nkv, d, 1)
        q = torch.empty((20, 2, d), dtype=torch.bfloat16, device=DEV)
        ops.qk_norm_rope_kv(q, pb.k8, pb.v8, qkv, None, None, None, 0, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, page, pb.status)
        changed = (pb.k8.codes != before).any(-1).any(1).any(-1)
        assert pb.status.item() == 2 and changed.nonzero().flatten().tolist() in ([pb.tables[0][0]], []), bad
        pb.status.zero_()
        ctx = ku.make_context(pb)
        out = torch.empty((20, 2, d), dtype=torch.bfloat16, device=DEV)
        ops.attention(out, q, pb.k8, pb.v8, ctx, 0, 0.1, None)
        assert pb.status.item() == 2, bad
        for heads in (8, 16):  # as many query rows as go over unpacked pages
            pb.status.zero_()
            q = torch.zeros((20, heads, d), dtype=torch.bfloat16, device=DEV)
            ops.attention(torch.empty_like(q), q, pb.k8, pb.v8, ku.make_context(pb), 0, 0.1, None)
            assert pb.status.item() == 2, (bad, heads)


# ------------------------------------------------------------------ attention
def _attend(pb, nq, d, scale, window=None, sink=False, seed=0, ctx=None, q=None):
    gen = torch.Generator(device=DEV).manual_seed(seed + 77)
    if q is None:
        q = torch.randn((pb.num_tokens, nq, d), generator=gen, device=DEV).bfloat16()
    out = torch.full_like(q, float("nan"))
    ops.attention(out, q, pb.k8, pb.v8, ctx or ku.make_context(pb), 0, scale, window, sink)
    return q, out


def _close(pb, q, out, scale, window=None, sink=False):
    """Against 64 bits: the output's rounding (2^-8 of it) and the weights' (2^-8 of what they carry, where they are bfloat16; 2^-11 in
    float16), and scores to float32: 2^-20 of a weight for each unit of sum |q k| scale log2(e), which stays below 64 here."""
    at = 0
    for r, (s, n) in enumerate(pb.rows):
        if n:
            k, v = pb.dense64(r)
            want, mass = cu.attention64(q[at:at + n], k, v, list(range(s, s + n)), scale, window, sink)
            off = (out[at:at + n].double() - want).abs() - (2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -14) * mass + 1e-30)
            assert bool((off <= 0).all()), (r, s, n, off.max().item())
        at += n
    assert pb.status.item() == 0


SHAPES = [(16, 8, 128, 16), (8, 1, 128, 16), (32, 4, 64, 16), (5, 1, 80, 16), (4, 4, 256, 32), (3, 3, 16, 8), (20, 1, 64, 8), (6, 2, 48, 64), (40, 1, 128, 16)]


@pytest.mark.parametrize("nq,nkv,d,page", SHAPES)
@pytest.mark.parametrize("rows", [[(0, 1)], [(299, 1)], [(15, 1), (16, 1), (0, 1), (1000, 1)], [(2000 + 37 * i, 1) for i in range(9)]])
def test_single_tokens(nq, nkv, d, page, rows):
    pb = cu.Batch8(rows, page, nkv, d, seed=nq + len(rows))
    q, out = _attend(pb, nq, d, d ** -0.5)
    _close(pb, q, out, d ** -0.5)


@pytest.mark.parametrize("nq,nkv,d,page", SHAPES)
@pytest.mark.parametrize("rows", [[(0, 2)], [(0, 129)], [(100, 5), (731, 5), (0, 5)], [(1500, 70), (0, 1), (3, 257)], [(64, 1), (900, 1), (128, 128)]])
def test_chunks(nq, nkv, d, page, rows):
    pb = cu.Batch8(rows, page, nkv, d, seed=nq + len(rows))
    q, out = _attend(pb, nq, d, d ** -0.5)
    _close(pb, q, out, d ** -0.5)


@pytest.mark.parametrize("nq,nkv,d,page", [(16, 8, 128, 16), (8, 2, 64, 8), (4, 1, 256, 16)])
@pytest.mark.parametrize("window,sink", [(1, False), (5, True), (16, False), (100, True), (4000, True)])
def test_windows_and_sinks(nq, nkv, d, page, window, sink):
    """With a window, pages that it has passed are not in the table any more."""
    rows = [(700, 1), (33, 1), (0, 1), (260, 40), (0, 150)]
    pb = cu.Batch8(rows, page, nkv, d, seed=window)
    for r, (s, n) in enumerate(rows):
        passed = max(0, s - window + 1) // page
        pb.page_indices[int(pb.page_indptr[r]):int(pb.page_indptr[r]) + passed] = -1
    q, out = _attend(pb, nq, d, 0.1, window, sink)
    _close(pb, q, out, 0.1, window, sink)


@pytest.mark.parametrize("d", [64, 128])
def test_a_long_context_of_one_token(d):
    pb = cu.Batch8([(40000, 1)], 16, 2, d, seed=5)
    q, out = _attend(pb, 4, d, d ** -0.5)
    _close(pb, q, out, d ** -0.5)


@pytest.mark.parametrize("rows", [[(400, 1)], [(400, 9)]])
@pytest.mark.parametrize("d", [64, 128])
def test_values_and_keys_of_every_size(rows, d):
    """Vectors from the smallest to the largest exponents side by side, zero vectors, and queries from tiny to huge."""
    pb = cu.Batch8(rows, 16, 2, d, seed=9, spread=0.0)
    n = sum(rows[0])
    gen = torch.Generator(device=DEV).manual_seed(1)
    pb.v8.exponents[pb.v8.exponents != 255] = 127
    spread = torch.randint(67, 135, pb.v8.exponents.shape, generator=gen, device=DEV, dtype=torch.uint8)
    pb.v8.exponents.copy_(torch.where(pb.v8.exponents == 255, pb.v8.exponents, spread))
    pb.k8.codes[pb.tables[0][2]] = 0
    pb.v8.codes[pb.tables[0][3]] = 0
    pb.v8.exponents[pb.tables[0][3]] = 67
    q = torch.randn((rows[0][1], 4, d), generator=gen, device=DEV)
    q[:, 1] *= 2.0 ** -100
    q[:, 2] = 0
    q[:, 3] *= 2.0 ** 60  # (one key takes it all)
    q = q.bfloat16()
    q, out = _attend(pb, 4, d, d ** -0.5, q=q)
    _close(pb, q, out, d ** -0.5)
    assert n <= 409


def test_what_is_not_finite_reaches_only_who_sees_it():
    d = 128
    for rows in ([(100, 1), (50, 1)], [(100, 4), (50, 4)]):
        pb = cu.Batch8(rows, 16, 2, d, seed=2)
        page, slot = pb.tables[0][20 // 16], 20 % 16
        pb.v8.codes[page, 1, slot] = 0
        pb.v8.exponents[page, 1, slot] = 255  # value 20 of row 0, kv head 1
        q, out = _attend(pb, 4, d, 0.1)
        n = rows[0][1]
        assert bool(out[:n, 2:].isnan().all()) and bool(out[:n, :2].isfinite().all()) and bool(out[n:].isfinite().all())
        q, out = _attend(pb, 4, d, 0.1, window=30)  # position 100 does not see 20
        assert bool(out.isfinite().all())
        pb.v8.exponents[page, 1, slot] = 127
        pb.k8.exponents[page, 0, slot] = 255
        pb.k8.codes[page, 0, slot] = 0
        q, out = _attend(pb, 4, d, 0.1)
        assert bool(out[:n, :2].isnan().all()) and bool(out[:n, 2:].isfinite().all()) and bool(out[n:].isfinite().all())
        if n > 1:  # a later token's key and value: the tokens before it do not see them
            pb.k8.exponents[page, 0, slot] = 127
            page, slot = pb.tables[0][102 // 16], 102 % 16
            pb.v8.codes[page, 0, slot] = 0
            pb.v8.exponents[page, 0, slot] = 255
            pb.k8.exponents[page, 1, slot] = 255
            pb.k8.codes[page, 1, slot] = 0
            q, out = _attend(pb, 4, d, 0.1)
            assert bool(out[2:n].isnan().all()) and bool(out[:2].isfinite().all()) and bool(out[n:].isfinite().all())


@pytest.mark.parametrize("rows", [[(0, 0)], [(40, 0), (7, 0)]])
def test_a_step_without_tokens(rows):
    pb = cu.Batch8(rows, 16, 2, 64, seed=4)
    q, out = _attend(pb, 8, 64, 0.1)
    assert out.shape[0] == 0 and pb.status.item() == 0


def test_rows_without_keys_are_zero():
    """A row that brings a token but whose table says no key (start -1): nothing is seen, the output is zero."""
    d = 64
    pb = cu.Batch8([(10, 1), (20, 1)], 16, 2, d, seed=4)
    ctx = ku.make_context(pb)
    ctx.q_start.copy_(torch.tensor([-1, 20], dtype=torch.int32))
    q, out = _attend(pb, 4, d, 0.1, ctx=ctx)
    assert bool((out[0] == 0).all())
    k, v = pb.dense64(1)
    want, mass = cu.attention64(q[1:], k, v, [20], 0.1)
    assert bool(((out[1:].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -8 * mass).all())


def test_the_same_call_gives_the_same_bits_and_leaves_its_workspace():
    pb = cu.Batch8([(5000, 1), (3, 1), (700, 12)], 16, 2, 128, seed=6)
    ctx = ku.make_context(pb)
    q, first = _attend(pb, 8, 128, 0.1, ctx=ctx)
    for _ in range(5):
        _, again = _attend(pb, 8, 128, 0.1, ctx=ctx, q=q)
        assert torch.equal(first, again)


def test_on_another_stream_and_replayed():
    """Captured on a side stream, replayed with other lengths, queries and cache contents in the same places."""
    pb = cu.Batch8([(900, 1), (37, 1)], 16, 2, 128, seed=8)
    ctx = ku.make_context(pb)
    q = torch.randn((2, 8, 128), device=DEV).bfloat16()
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ctx.stream = side.cuda_stream
        ops.attention(out, q, pb.k8, pb.v8, ctx, 0, 0.1, None)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        ctx.step_cache.clear()
        with torch.cuda.graph(graph, stream=side):
            ctx.stream = torch.cuda.current_stream().cuda_stream
            ops.attention(out, q, pb.k8, pb.v8, ctx, 0, 0.1, None)
    torch.cuda.synchronize()
    for start in ((900, 37), (200, 12), (899, 0)):
        pb.rows = [(s, 1) for s in start]
        ctx.q_start.copy_(torch.tensor(start, dtype=torch.int32))
        q.copy_(torch.randn((2, 8, 128), device=DEV).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        _close(pb, q, out, 0.1)


def _spare_entries(pb, spare):
    """Each row's table goes on behind the pages that it needs; those entries name no page."""
    tables = [t + [-1] * n for t, n in zip(pb.tables, spare)]
    indptr = [0]
    for t in tables:
        indptr.append(indptr[-1] + len(t))
    i32 = dict(dtype=torch.int32, device=DEV)
    pb.page_indptr, pb.page_indices = torch.tensor(indptr, **i32), torch.tensor([p for t in tables for p in t], **i32)


@pytest.mark.parametrize("nq,nkv,d,page", [(16, 8, 128, 16), (8, 2, 64, 8), (16, 2, 80, 32), (2, 1, 128, 256), (2, 2, 128, 128)])
@pytest.mark.parametrize("window", [None, 40])
def test_tables_that_list_more_than_a_row_needs(nq, nkv, d, page, window):
    rows = [(700, 1), (33, 1), (260, 140), (0, 70), (1, 2), (515, 99)]
    pb = cu.Batch8(rows, page, nkv, d, seed=d)
    _spare_entries(pb, [3, 0, 5, 1, 0, 2])
    q, out = _attend(pb, nq, d, 0.1, window)
    _close(pb, q, out, 0.1, window)


@pytest.mark.parametrize("nq,nkv,d", [(16, 2, 128), (16, 2, 64)])
def test_prompts_behind_a_window_over_scratch_that_held_something_else(nq, nkv, d):
    """Pages that a window has passed are not unpacked; what lies in their place is weighed by zero at most."""
    for _ in range(3):
        torch.full((1 << 24,), float("nan"), dtype=torch.bfloat16, device=DEV)  # (given back at once: the next allocations get it)
    scratch = {}
    for seed, rows in enumerate(([(700, 1), (333, 90), (1200, 70)], [(64, 40), (1501, 64)], [(4000, 300)], [(10, 64), (90, 33)])):
        pb = cu.Batch8(rows, 16, nkv, d, seed=seed)
        for r, (s, n) in enumerate(rows):
            passed = max(0, s - 50 + 1) // 16
            pb.page_indices[int(pb.page_indptr[r]):int(pb.page_indptr[r]) + passed] = -1
        ctx = ku.make_context(pb)
        ctx.scratch = scratch
        q, out = _attend(pb, nq, d, 0.1, 50, seed=seed, ctx=ctx)
        _close(pb, q, out, 0.1, 50)


def test_more_requests_than_a_launch_takes():
    rows = [(3 + 7 * i % 190, 1) for i in range(300)]
    pb = cu.Batch8(rows, 16, 1, 64, seed=2)
    q, out = _attend(pb, 4, 64, 0.1)
    _close(pb, q, out, 0.1)
    rows = [(3 + 7 * i % 190, 5) for i in range(150)]
    pb = cu.Batch8(rows, 16, 1, 64, seed=2)
    q, out = _attend(pb, 8, 64, 0.1)  # 40 query rows a request: two tiles each
    _close(pb, q, out, 0.1)


@pytest.mark.parametrize("nq,nkv,d,page", [(8, 1, 64, 16), (4, 2, 80, 16), (2, 1, 256, 16), (2, 1, 128, 256)])
def test_prompts_behind_long_contexts_of_shapes_that_share_out_keys(nq, nkv, d, page, window=None):
    """Prompts of very different lengths, one of more tiles than a launch takes, behind more keys than they bring."""
    rows = [(50, 1), (2500, 701), (9000, 3), (3000, 1), (40, 17), (2000, 1200), (0, 0), (7, 30)]
    pb = cu.Batch8(rows, page, nkv, d, seed=d)
    ctx = ku.make_context(pb)
    q, out = _attend(pb, nq, d, 0.1, ctx=ctx)
    assert "cache8_pages" not in ctx.scratch
    _close(pb, q, out, 0.1)


@pytest.mark.parametrize("nq,nkv,d,page", [(16, 8, 128, 16), (8, 2, 64, 8), (4, 1, 256, 16)])
@pytest.mark.parametrize("rows", [[(0, 1)], [(2047 + 3 * i, 1) for i in range(8)], [(100, 5), (731, 5), (0, 5)], [(31, 1), (32, 1), (33, 1), (5000, 1)]])
@pytest.mark.parametrize("window", [None, 40])
def test_tables_and_older_tokens_ahead_of_the_kernels_before(nq, nkv, d, page, rows, window):
    """A context that says so (everything is in place: the device has been waited for) gets the same bits, behind a write of the step's own tokens too."""
    pb = cu.Batch8(rows, page, nkv, d, seed=len(rows))
    qkv, _ = _projection(pb.num_tokens, nq, nkv, d, 3)
    outs = []
    for ahead in (False, True):
        k8, v8 = (ops.Pool8(p.codes.clone(), p.exponents.clone()) for p in (pb.k8, pb.v8))
        ctx = ku.make_context(pb)
        ctx.tables_ahead = ahead
        q, out = (torch.full((pb.num_tokens, nq, d), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
        torch.cuda.synchronize()
        for _ in range(3):
            ops.qk_norm_rope_kv(q, k8, v8, qkv, None, None, None, 0, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, page, pb.status)
            ops.attention(out, q, k8, v8, ctx, 0, 0.1, window)
        outs.append(out)
    assert torch.equal(*outs) and bool(outs[0].isfinite().all()) and pb.status.item() == 0


@pytest.mark.parametrize("rows", [[(5000, 1), (3, 1), (700, 1)], [(900, 90), (0, 33)]])
def test_two_contexts_on_two_streams(rows):
    """At once, each with scratch of its own: the bits of a call alone."""
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    batches = [cu.Batch8(rows, 16, 2, 128, seed=11 + i) for i in range(2)]
    alone = [_attend(pb, 16, 128, 0.1, seed=i) for i, pb in enumerate(batches)]
    outs = [torch.full_like(q, float("nan")) for q, _ in alone]
    contexts = [ku.make_context(pb) for pb in batches]
    torch.cuda.synchronize()
    for _ in range(5):
        for pb, side, ctx, (q, _), out in zip(batches, sides, contexts, alone, outs):
            with torch.cuda.stream(side):
                ctx.stream = side.cuda_stream
                ops.attention(out, q, pb.k8, pb.v8, ctx, 0, 0.1, None)
    torch.cuda.synchronize()
    for out, (_, want) in zip(outs, alone):
        assert torch.equal(out, want)


@pytest.mark.parametrize("captured", [False, True])
def test_lengths_that_change_on_the_device_alone(captured):
    """Single tokens go by the lengths on the device: a call (or a graph of one) whose context was first used for short rows serves long ones, and the other way round."""
    pb = cu.Batch8([(1900, 1), (1500, 1)], 16, 2, 128, seed=8)
    for first in ((60, 30), (1900, 1500)):
        ctx = ku.make_context(pb)
        ctx.host_q_start, ctx.max_kv_len = list(first), max(first) + 1
        ctx.q_start.copy_(torch.tensor(first, dtype=torch.int32))
        pb.rows = [(s, 1) for s in first]
        q, out = _attend(pb, 8, 128, 0.1, ctx=ctx)
        _close(pb, q, out, 0.1)
        graph = torch.cuda.CUDAGraph()
        if captured:
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                ctx.stream = torch.cuda.current_stream().cuda_stream
                ops.attention(out, q, pb.k8, pb.v8, ctx, 0, 0.1, None)
        for now in ((1900, 1500), (12, 1499), (0, 3)):
            ctx.q_start.copy_(torch.tensor(now, dtype=torch.int32))
            pb.rows = [(s, 1) for s in now]
            out.fill_(float("nan"))
            if captured:
                graph.replay()
            else:
                ops.attention(out, q, pb.k8, pb.v8, ctx, 0, 0.1, None)
            torch.cuda.synchronize()
            _close(pb, q, out, 0.1)


@pytest.mark.parametrize("rows", [[(900, 1), (37, 1)], [(300, 70), (15, 40)]])
def test_a_step_s_stream_that_is_not_the_current_one(rows):
    """``ctx.stream`` says where the kernels go; what they need is made there too."""
    pb = cu.Batch8(rows, 16, 2, 128, seed=8)
    q, want = _attend(pb, 16, 128, 0.1)
    side, out, ctx = torch.cuda.Stream(), torch.full_like(q, float("nan")), ku.make_context(pb)
    torch.cuda.synchronize()
    ctx.stream = side.cuda_stream
    ops.attention(out, q, pb.k8, pb.v8, ctx, 0, 0.1, None)
    side.synchronize()
    assert torch.equal(out, want)


def test_a_captured_prompt_outlives_larger_ones():
    """A graph of a prompt over unpacked pages, replayed after a longer prompt of the same scratch."""
    pb, other = cu.Batch8([(300, 70)], 16, 2, 64, seed=8), cu.Batch8([(3000, 200)], 16, 2, 64, seed=9)
    ctx = ku.make_context(pb)
    q, want = _attend(pb, 16, 64, 0.1, ctx=ctx)
    out, graph = torch.full_like(q, float("nan")), torch.cuda.CUDAGraph()
    ctx.step_cache.clear()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ctx.stream = torch.cuda.current_stream().cuda_stream
        ops.attention(out, q, pb.k8, pb.v8, ctx, 0, 0.1, None)
    larger = ku.make_context(other)
    larger.scratch = ctx.scratch
    for _ in range(2):
        _close(other, *_attend(other, 16, 64, 0.1, ctx=larger), 0.1)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("nq,nkv,d,page", [(8, 1, 64, 16), (4, 2, 80, 8), (4, 1, 256, 32), (8, 4, 128, 16), (2, 1, 128, 256)])
@pytest.mark.parametrize("window,sink", [(None, False), (50, True)])
def test_prompts_over_unpacked_pages(nq, nkv, d, page, window, sink):
    """Prompts that bring more than lies behind them, the unpacked pages beginning as NaN where they are not written; again with other prompts in the same scratch."""
    for _ in range(3):
        torch.full((1 << 24,), float("nan"), dtype=torch.bfloat16, device=DEV)  # (given back at once: the next allocations get it)
    scratch = {}
    for seed, rows in enumerate(([(9, 1), (100, 200), (0, 33), (60, 129), (5, 64)], [(0, 128), (1, 100), (130, 300), (0, 0), (2, 97)])):
        pb = cu.Batch8(rows, page, nkv, d, seed=seed)
        if window:
            for r, (s, n) in enumerate(rows):
                passed = max(0, s - window + 1) // page
                pb.page_indices[int(pb.page_indptr[r]):int(pb.page_indptr[r]) + passed] = -1
        ctx = ku.make_context(pb)
        ctx.scratch = scratch
        q, out = _attend(pb, nq, d, 0.1, window, sink, ctx=ctx)
        assert "cache8_pages" in scratch
        _close(pb, q, out, 0.1, window, sink)


def test_a_captured_prompt_over_unpacked_pages_outlives_larger_ones():
    pb, other = cu.Batch8([(30, 170), (0, 200)], 16, 2, 64, seed=8), cu.Batch8([(300, 2000)], 16, 2, 64, seed=9)
    ctx = ku.make_context(pb)
    q, want = _attend(pb, 16, 64, 0.1, ctx=ctx)
    out, graph = torch.full_like(q, float("nan")), torch.cuda.CUDAGraph()
    ctx.step_cache.clear()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ctx.stream = torch.cuda.current_stream().cuda_stream
        ops.attention(out, q, pb.k8, pb.v8, ctx, 0, 0.1, None)
    larger = ku.make_context(other)
    larger.scratch = ctx.scratch
    for _ in range(2):
        _close(other, *_attend(other, 16, 64, 0.1, ctx=larger), 0.1)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and "cache8_pages" in ctx.scratch


def test_pages_beyond_4_gb():
    """Codes whose offset passes 32 bits: written, read, attended over by single tokens and by a prompt."""
    nkv, d, page = 8, 256, 16
    rows = [(300, 1), (77, 1), (100, 40)]
    pb = cu.Batch8(rows, page, nkv, d, seed=5)
    pages = 2 ** 32 // (nkv * page * d) + pb.num_pages + 5
    far = pages - pb.num_pages
    k8, v8 = (ops.Pool8.empty(pages, nkv, page, d) for _ in range(2))
    for big, small in ((k8, pb.k8), (v8, pb.v8)):
        big.codes[far:], big.exponents[far:] = small.codes, small.exponents
    pb.k8, pb.v8 = k8, v8
    pb.tables = [[p + far for p in t] for t in pb.tables]
    pb.page_indices += far
    pb.num_pages = pages
    q, out = _attend(pb, 16, d, 0.06)
    _close(pb, q, out, 0.06)
    qkv, _ = _projection(pb.num_tokens, 16, nkv, d, 3)
    ops.qk_norm_rope_kv(q, k8, v8, qkv, None, None, None, 0, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, page, pb.status)
    k, v = (torch.empty((pb.num_tokens, nkv, d), dtype=torch.float32, device=DEV) for _ in range(2))
    ops.read_cache(k, v, k8, v8, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, pb.status)
    x = qkv.double().view(pb.num_tokens, 16 + 2 * nkv, d)
    # half a step: 2^-4 of the number, or half of the smallest code of the vector's scale (2^-10 of 2^e, 448 * 2^e below twice the largest number)
    for got, want in ((k, x[:, 16:16 + nkv]), (v, x[:, 16 + nkv:])):
        assert bool(((got.double() - want).abs() <= torch.maximum(want.abs() * 2.0 ** -4, want.abs().amax(-1, keepdim=True) * 2.0 ** -9 / 448)).all())
    assert pb.status.item() == 0 and bool((k8.codes[:far] == 0).all())


# ------------------------------------------------------------------ one behind the other
@pytest.mark.parametrize("nq,nkv,d", [(4, 2, 128), (8, 2, 64)])
def test_write_attend_read_a_request_in_portions(nq, nkv, d):
    """A prompt in two portions and then token by token: what attention sees is what the pages hold, whatever wrote it."""
    page, steps = 16, [(0, 70), (70, 45), (115, 1), (116, 1), (117, 3)]
    total = sum(n for _, n in steps)
    whole = ku.PagedBatch([(0, total)], page, nkv, d, torch.bfloat16, seed=1)
    k8, v8 = (ops.Pool8.empty(whole.num_pages, nkv, page, d) for _ in range(2))
    qkv, gen = _projection(total, nq, nkv, d, 3)
    inv = (1e4 ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)).float()
    for s, n in steps:
        pb = ku.PagedBatch([(s, n)], page, nkv, d, torch.bfloat16, share=whole)
        pb.k8, pb.v8 = k8, v8
        pb.dense64 = lambda r, pb=pb: cu.Batch8.dense64(pb, r)
        q = torch.empty((n, nq, d), dtype=torch.bfloat16, device=DEV)
        ops.qk_norm_rope_kv(q, k8, v8, qkv[s:s + n].contiguous(), None, None, inv, d, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, page, pb.status)
        out = torch.empty_like(q)
        ops.attention(out, q, k8, v8, ku.make_context(pb), 0, d ** -0.5, None)
        _close(pb, q, out, d ** -0.5)
    k, v = (torch.empty((total, nkv, d), dtype=torch.float32, device=DEV) for _ in range(2))
    ops.read_cache(k, v, k8, v8, whole.positions, whole.row_of_token, whole.page_indptr, whole.page_indices, whole.status)
    whole.k8, whole.v8 = k8, v8
    k64, v64 = cu.Batch8.dense64(whole, 0)
    assert torch.equal(k.double(), k64) and torch.equal(v.double(), v64) and whole.status.item() == 0


# ------------------------------------------------------------------ refusals
def test_refusals():
    pb = cu.Batch8([(10, 1)], 16, 2, 64, seed=4)
    ctx = ku.make_context(pb)
    q = torch.zeros((1, 4, 64), dtype=torch.bfloat16, device=DEV)
    good = torch.empty_like(q)
    with pytest.raises(ValueError, match="bfloat16"):
        ops.attention(good.float(), q.float(), pb.k8, pb.v8, ctx, 0, 0.1, None)
    with pytest.raises(ValueError, match="query heads"):
        ops.attention(good[:, :3].contiguous(), q[:, :3].contiguous(), pb.k8, pb.v8, ctx, 0, 0.1, None)
    with pytest.raises(ValueError, match="contiguous"):
        ops.attention(good, torch.zeros((1, 64, 4), dtype=torch.bfloat16, device=DEV).transpose(1, 2), pb.k8, pb.v8, ctx, 0, 0.1, None)
    with pytest.raises(TypeError, match="both"):
        ops.attention(good, q, pb.k8, pb.v_pool, ku.make_context(pb), 0, 0.1, None)
    with pytest.raises(ValueError, match="no learned sinks"):
        ops.attention(good, q, pb.k8, pb.v8, ctx, 0, 0.1, None, extras=ops.AttentionExtras(softcap=3.0))
    rows = torch.empty((1, 2, 64), dtype=torch.float16, device=DEV)
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        ops.read_cache(rows, rows, pb.k8, pb.v8, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, pb.status)
    with pytest.raises(ValueError, match="int32"):
        ops.read_cache(rows.float(), rows.float(), pb.k8, pb.v8, pb.positions.long(), pb.row_of_token, pb.page_indptr, pb.page_indices, pb.status)
    qkv, _ = _projection(1, 4, 2, 64, 0)
    with pytest.raises(ValueError, match="page size"):
        ops.qk_norm_rope_kv(q, pb.k8, pb.v8, qkv, None, None, None, 0, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, 32, pb.status)
    with pytest.raises(ValueError, match="bfloat16"):
        ops.qk_norm_rope_kv(q, pb.k8, pb.v8, qkv.float(), None, None, None, 0, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, 16, pb.status)
