"""The 8-bit cache's numbers: exponents that the writer never makes, the norm's rounding, weights of 11 bits, places that other tests do not look at."""

from __future__ import annotations

import pytest
import torch

from miniserve_b200 import ops
from tests import cache8_util as cu
from tests import kernel_util as ku
from tests.test_cache8_gpu import _attend, _close, _projection

pytestmark = pytest.mark.gpu
DEV = "cuda"

# ways through attention: one token (a CTA an item, and cut), drafted tokens, prompts that share out keys, prompts over unpacked pages
WAYS = [(4, 2, 128, [(100, 1), (33, 1)]), (4, 2, 64, [(5000, 1)]), (8, 2, 64, [(60, 5), (700, 4)]), (8, 1, 64, [(700, 90)]), (16, 2, 128, [(20, 200)]), (8, 1, 80, [(20, 200)])]


# ------------------------------------------------------------------ exponents below the writer's
@pytest.mark.parametrize("nq,nkv,d,rows", WAYS)
@pytest.mark.parametrize("sink", [False, True])
def test_a_pool_of_zeros_gives_zeros(nq, nkv, d, rows, sink):
    pb = cu.Batch8(rows, 16, nkv, d, seed=3)
    pb.k8, pb.v8 = (ops.Pool8.empty(pb.num_pages, nkv, 16, d) for _ in range(2))
    q, out = _attend(pb, nq, d, 0.1, sink=sink)
    assert pb.status.item() == 0 and bool((out == 0).all())
    k, v = (torch.full((pb.num_tokens, nkv, d), 3.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    ops.read_cache(k, v, pb.k8, pb.v8, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, pb.status)
    assert bool((k == 0).all()) and bool((v == 0).all())


@pytest.mark.parametrize("nq,nkv,d,rows", WAYS)
def test_zero_vectors_of_exponent_zero_among_others(nq, nkv, d, rows):
    """The first pages of every row as an empty pool has them, the others as the writer makes them."""
    pb = cu.Batch8(rows, 16, nkv, d, seed=3)
    for t in pb.tables:
        for pool in (pb.k8, pb.v8):
            pool.codes[t[:2]] = 0
            pool.exponents[t[:2]] = 0
    q, out = _attend(pb, nq, d, 0.1)
    _close(pb, q, out, 0.1)


@pytest.mark.parametrize("nq,nkv,d,rows", WAYS)
@pytest.mark.parametrize("least,most", [(0, 1), (0, 67), (1, 40), (30, 135)])
def test_exponents_below_the_writer_s(nq, nkv, d, rows, least, most):
    """Values of any exponent: finite, and where they are smaller than what the writer makes within 2^-82 a key of the formula: a weight's half step at the end of float16 is 2^-25, a code
    below 2^9, and the weights' sum, in units of the least exponent's 2^-60 and the 2^6 that weights are kept below, 2^66 or more."""
    pb = cu.Batch8(rows, 16, nkv, d, seed=3)
    gen = torch.Generator(device=DEV).manual_seed(1)
    e = torch.randint(least, most, pb.v8.exponents.shape, generator=gen, device=DEV, dtype=torch.uint8)
    pb.v8.exponents.copy_(torch.where(pb.v8.exponents == 255, pb.v8.exponents, e))
    q, out = _attend(pb, nq, d, 0.1)
    at = 0
    for r, (s, n) in enumerate(rows):
        k, v = pb.dense64(r)
        want, mass = cu.attention64(q[at:at + n], k, v, list(range(s, s + n)), 0.1)
        off = (out[at:at + n].double() - want).abs() - (2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -14) * mass + (s + n) * 2.0 ** -82)
        assert bool(out[at:at + n].isfinite().all()) and bool((off <= 0).all())
        at += n
    assert pb.status.item() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_every_exponent_is_read_by_the_formula(dtype):
    """code * 2^(b - 127) for every byte b but 255, where the type holds it (2^-133 and 2^-149 are the smallest numbers)."""
    d, page = 16, 256
    pool = ops.Pool8.empty(1, 1, page, d)
    pool.exponents[0, 0] = torch.arange(256, device=DEV, dtype=torch.uint8)
    pool.codes[0, 0] = torch.tensor([0x38, 0xB8, 0x7E, 0x08] * 4, device=DEV, dtype=torch.uint8)  # 1, -1, 448, 2^-6
    pb = ku.PagedBatch([(0, 256)], page, 1, d, torch.bfloat16)
    pb.page_indices.zero_()
    k, v = (torch.empty((256, 1, d), dtype=dtype, device=DEV) for _ in range(2))
    ops.read_cache(k, v, pool, pool, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, pb.status)
    want = torch.tensor([1.0, -1.0, 448.0, 2.0 ** -6] * 4, dtype=torch.float64, device=DEV) * torch.exp2(torch.arange(255, device=DEV).double() - 127)[:, None]
    want = torch.where(want.abs() < 2.0 ** 128, want, want.sign() * float("inf"))
    assert torch.equal(k[:255, 0].double(), want) and torch.equal(v[:255, 0].double(), want) and bool(k[255].isnan().all())


# ------------------------------------------------------------------ the norm
@pytest.mark.parametrize("nq,nkv,d", [(16, 8, 128), (8, 2, 64), (8, 4, 256), (6, 3, 48)])
def test_the_norm_is_rounded_as_a_root_and_a_division(nq, nkv, d):
    """1 / sqrt(mean + eps) in float32, each operation to the nearest, as the package's other norms have it: of whole numbers up to 15 the sum of squares is exact in any order, so
    that every bit of the queries (and of keys, to the code) is known."""
    tokens, page = 4096, 16
    pb = ku.PagedBatch([(0, tokens)], page, nkv, d, torch.bfloat16)
    gen = torch.Generator(device=DEV).manual_seed(d)
    x = torch.randint(-15, 16, (tokens, nq + 2 * nkv, d), generator=gen, device=DEV).bfloat16()
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=gen, device=DEV)).bfloat16() for _ in range(2))
    k8, v8 = (ops.Pool8.empty(pb.num_pages, nkv, page, d) for _ in range(2))
    q = torch.empty((tokens, nq, d), dtype=torch.bfloat16, device=DEV)
    ops.qk_norm_rope_kv(q, k8, v8, x.view(tokens, -1), wq, wk, None, 0, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, page, pb.status)
    f = x.float().cpu()
    mean = f.square().sum(-1, keepdim=True) / d
    inv = 1.0 / (mean + torch.tensor(1e-6, dtype=torch.float32)).sqrt()
    want = f * inv * torch.cat([wq.float().cpu().expand(nq, d), wk.float().cpu().expand(nkv, d), torch.ones(nkv, d)])
    assert torch.equal(q.cpu(), want[:, :nq].bfloat16())
    pages = torch.tensor(pb.tables[0], device=DEV)[torch.arange(tokens, device=DEV) // page]
    held = cu.values64(k8.codes[pages, :, pb.positions.long() % page], k8.exponents[pages, :, pb.positions.long() % page]).cpu()
    key = want[:, nq:nq + nkv].double()
    e = cu.exponent64(key)[..., None]
    y = key * torch.exp2(-e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -40))).clamp_min(-6) - 3)
    assert torch.equal(held, torch.round(y / step) * step * torch.exp2(e))


# ------------------------------------------------------------------ weights of 11 bits
def _close11(pb, q, out, scale, window=None, sink=False):
    """The kernel that shares out keys against 64 bits: the output's rounding (2^-8 of it), the weights' in float16 (2^-11 of what they carry), and 2^-14 of that for scores to float32
    (2^-20 of a weight for each unit of sum |q k| scale log2(e), which stays below 64 here), sums of a few thousand terms and weights below float16's normal range (2^-31 of the largest)."""
    at = 0
    for r, (s, n) in enumerate(pb.rows):
        if n:
            k, v = pb.dense64(r)
            want, mass = cu.attention64(q[at:at + n], k, v, list(range(s, s + n)), scale, window, sink)
            off = (out[at:at + n].double() - want).abs() - (2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -14) * mass + 1e-30)
            assert bool((off <= 0).all()), (r, s, n, off.max().item())
        at += n
    assert pb.status.item() == 0


@pytest.mark.parametrize("nq,nkv,d,page", [(16, 8, 128, 16), (32, 4, 64, 16), (5, 1, 80, 16), (4, 4, 256, 32), (3, 3, 16, 8), (6, 2, 48, 64)])
@pytest.mark.parametrize("rows", [[(299, 1)], [(15, 1), (1000, 1), (0, 1), (64, 1)], [(2000 + 37 * i, 1) for i in range(9)], [(100, 5), (731, 5), (0, 5)], [(20000, 1)]])
@pytest.mark.parametrize("window,sink", [(None, False), (100, True)])
def test_single_and_drafted_tokens_keep_11_bits_of_a_weight(nq, nkv, d, page, rows, window, sink):
    pb = cu.Batch8(rows, page, nkv, d, seed=nq + len(rows))
    q, out = _attend(pb, nq, d, 0.5 * d ** -0.5, window, sink)
    _close11(pb, q, out, 0.5 * d ** -0.5, window, sink)


@pytest.mark.parametrize("nq,d,rows", [(4, 64, [(131071, 1)]), (4, 128, [(147000, 1)]), (8, 64, [(140000, 2)]), (1, 128, [(150000, 1)])])
def test_one_kv_head_and_a_context_cut_into_more_than_128_pieces(nq, d, rows):
    pb = cu.Batch8(rows, 16, 1, d, seed=5)
    q, out = _attend(pb, nq, d, d ** -0.5)
    _close11(pb, q, out, d ** -0.5)


# ------------------------------------------------------------------ places that other tests do not look at
def test_a_number_beside_ones_that_saturate():
    d, page = 64, 16
    v = torch.zeros((1, d))
    v[0, :3] = torch.tensor([1e30, -1e30, 3.0])  # exponent 7: 3 is 1.5 * 2^-6 of 2^7, a code
    qkv = torch.cat([torch.zeros((1, 2 * d)), v], -1).bfloat16().to(DEV)
    pb = ku.PagedBatch([(0, 1)], page, 1, d, torch.bfloat16)
    k8, v8 = ops.Pool8.empty(pb.num_pages, 1, page, d), ops.Pool8.empty(pb.num_pages, 1, page, d)
    q = torch.empty((1, 1, d), dtype=torch.bfloat16, device=DEV)
    ops.qk_norm_rope_kv(q, k8, v8, qkv, None, None, None, 0, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, page, pb.status)
    assert cu.values64(v8.codes, v8.exponents)[pb.tables[0][0], 0, 0, :4].tolist() == [57344, -57344, 3, 0]


@pytest.mark.parametrize("nq,nkv,d", [(16, 8, 128), (16, 2, 64)])
@pytest.mark.parametrize("window", [None, 50])
def test_prompts_unpacked_in_several_parts(nq, nkv, d, window, monkeypatch):
    """As many rows at a time as have room, here for some 20 pages: the bits of all at once."""
    from miniserve_b200.ops import cache8

    rows = [(9, 1), (100, 200), (0, 333), (60, 129), (5, 64), (0, 0), (2, 97)]
    pb = cu.Batch8(rows, 16, nkv, d, seed=2)
    q, want = _attend(pb, nq, d, 0.1, window)
    _close(pb, q, want, 0.1, window)
    monkeypatch.setattr(cache8, "UNPACKED_BYTES", 20 * 4 * nkv * 16 * d)
    ctx = ku.make_context(pb)
    _, out = _attend(pb, nq, d, 0.1, window, ctx=ctx, q=q)
    assert ctx.scratch["cache8_pages"][0].numel() <= 32 * nkv * 16 * d  # (the longest row has 21 pages)
    _close(pb, q, out, 0.1, window)


# ------------------------------------------------------------------ tables read ahead
@pytest.mark.parametrize("nq,nkv,d,page", [(16, 8, 128, 16), (8, 2, 64, 8), (4, 1, 256, 16), (4, 1, 64, 8), (2, 1, 128, 64)])
@pytest.mark.parametrize("rows", [[(0, 1)], [(2047 + 3 * i, 1) for i in range(8)], [(100, 5), (731, 5), (0, 5)], [(31, 1), (32, 1), (33, 1), (5000, 1)], [(6 + i, 1) for i in range(40)]])
@pytest.mark.parametrize("window", [None, 40])
def test_what_is_read_ahead_is_never_a_step_s_own(nq, nkv, d, page, rows, window):
    """Every pass writes other tokens into slots that held poison or the pass before's, and attends at once: a slot read before its own write would show in the pass that it belongs to."""
    pb = cu.Batch8(rows, page, nkv, d, seed=len(rows))
    pos = pb.positions.long()
    pages = torch.tensor([pb.tables[r][p // page] for r, p in zip(pb.row_of_token.tolist(), pos.tolist())], device=DEV)
    for pool in (pb.k8, pb.v8):  # the step's own slots: nothing has been written there yet
        pool.codes[pages, :, pos % page] = 0x7F
        pool.exponents[pages, :, pos % page] = 255
    projections = [_projection(pb.num_tokens, nq, nkv, d, 3 + i)[0] for i in range(4)]
    got = []
    for ahead in (False, True):
        k8, v8 = (ops.Pool8(p.codes.clone(), p.exponents.clone()) for p in (pb.k8, pb.v8))
        ctx = ku.make_context(pb)
        ctx.tables_ahead = ahead
        outs = [torch.full((pb.num_tokens, nq, d), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in projections]
        q = torch.full_like(outs[0], float("nan"))
        warm = ops.Pool8(k8.codes.clone(), k8.exponents.clone())
        ops.attention(torch.empty_like(q), torch.zeros_like(q), warm, warm, ctx, 0, 0.1, window)  # (the plan is made)
        torch.cuda.synchronize()
        for qkv, out in zip(projections, outs):
            ops.qk_norm_rope_kv(q, k8, v8, qkv, None, None, None, 0, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, page, pb.status)
            ops.attention(out, q, k8, v8, ctx, 0, 0.1, window)
        got.append(outs)
        pb.k8, held = k8, pb.k8
        pb.v8, held_v = v8, pb.v8
        _close(pb, q, outs[-1], 0.1, window)
        pb.k8, pb.v8 = held, held_v
    for plain, early in zip(*got):
        assert bool(plain.isfinite().all()) and torch.equal(plain, early)
    assert pb.status.item() == 0


def _close_wide(pb, q, out, scale):
    """``_close`` for scores of any size. Scores to float32: 2^-20 of a weight for each unit of sum |q k| scale log2(e), here up to some thousands (queries and keys are scaled by 8 each: 128
    channels of 12 x 12 make 2,600), where that text takes 64. And one key may take nearly all: a weight with its value's scale is kept to 2^-25 (half of float16's smallest step), the
    row's largest is 2^6 or more, so that a key's part is off by 2^-31 of a largest code (448) at most, in the scale of the largest's value, whatever it carries itself."""
    at = 0
    for r, (s, n) in enumerate(pb.rows):
        k, v = pb.dense64(r)
        mine = q[at:at + n]
        want, mass = cu.attention64(mine, k, v, list(range(s, s + n)), scale)
        group = mine.shape[1] // k.shape[1]
        size = torch.stack([(mine[:, h].double().abs() @ k[:, h // group].abs().T).amax(1) for h in range(mine.shape[1])], 1) * scale * 1.4427
        e = pb.v8.exponents[torch.tensor(pb.tables[r], device=DEV)].permute(0, 2, 1).reshape(-1, k.shape[1])[:s + n].amax(0).double() - 127
        lost = ((s + n) * 448 * 2.0 ** -31 * torch.exp2(e)).repeat_interleave(group)[None, :, None]
        off = (out[at:at + n].double() - want).abs() - (2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -20 * size.clamp_min(64)[..., None]) * mass + lost)
        assert bool((off <= 0).all()), (r, s, n, off.max().item())
        at += n
    assert pb.status.item() == 0


def _pages_in_order(pb, first):
    """The same batch with its rows' pages one behind the other from page ``first`` on, as an allocator that begins there gives them."""
    order = [p for t in pb.tables for p in t]
    rest = [p for p in range(pb.num_pages) if p not in set(order)]
    place = rest[:first] + order + rest[first:]
    at = torch.tensor(place, device=DEV)
    pb.k8, pb.v8 = (ops.Pool8(x.codes[at].contiguous(), x.exponents[at].contiguous()) for x in (pb.k8, pb.v8))
    new = {p: i for i, p in enumerate(place)}
    pb.tables = [[new[p] for p in t] for t in pb.tables]
    pb.page_indices = torch.tensor([p for t in pb.tables for p in t], dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("nq,nkv,d,page", [(4, 1, 64, 8), (4, 1, 64, 16), (8, 1, 128, 16), (4, 2, 64, 8), (16, 8, 128, 16)])
@pytest.mark.parametrize("first", [0, 1, 2, 3])
@pytest.mark.parametrize("rows", [[(36, 1)], [(32 + 5 * i, 1) for i in range(12)], [(33, 5), (64, 3), (1000, 1)], [(2000 + i, 1) for i in range(40)]])
def test_a_step_s_own_slots_beside_ones_that_were_read_ahead(nq, nkv, d, page, first, rows):
    """The kernels wait behind one that takes long, with what they read ahead long there: exponents of neighbouring slots, pages and heads share 32 bytes of memory, and the write in between
    changes some of them."""
    pb = cu.Batch8(rows, page, nkv, d, seed=len(rows))
    _pages_in_order(pb, first)
    slow = ku.PagedBatch([(2500, 1)], 16, 1, 64, torch.float32)
    slow.k_pool.zero_(), slow.v_pool.zero_()
    busy = torch.zeros((1, 1, 64), device=DEV)
    ctx = ku.make_context(pb)
    ctx.tables_ahead = True
    q, out = (torch.full((pb.num_tokens, nq, d), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    ops.attention(torch.empty_like(q), torch.zeros_like(q), pb.k8, pb.v8, ctx, 0, 0.1, None)  # (the plan is made)
    for i in range(3):
        qkv = _projection(pb.num_tokens, nq, nkv, d, 3 + i)[0]
        qkv *= (1.0, 8.0, 0.125)[i]  # (other exponents)
        torch.cuda.synchronize()
        ops.attention_rowwise(busy, busy, slow.k_pool, slow.v_pool, slow.positions, slow.row_of_token, slow.page_indptr, slow.page_indices, 0.1, None, slow.status)
        ops.qk_norm_rope_kv(q, pb.k8, pb.v8, qkv, None, None, None, 0, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, page, pb.status)
        ops.attention(out, q, pb.k8, pb.v8, ctx, 0, 0.1, None)
        torch.cuda.synchronize()
        _close_wide(pb, q, out, 0.1)
