"""The 8-bit cache over the page tables that the engine's packer makes for windowed groups."""

from __future__ import annotations

import pytest
import torch

from miniserve_b200 import ops
from tests import cache8_util as cu
from tests import kernel_util as ku
from tests.test_cache8_gpu import _attend, _close, _projection

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


# ------------------------------------------------------------------ several rows behind their windows
PACKED = [(16, 8, 128, 16), (8, 2, 64, 8), (4, 1, 80, 16), (8, 1, 256, 32)]
SINGLE = [(40, 1), (60, 1)]


def _whole(pb, r):
    """Row r's pages on the device, from position 0 on."""
    return torch.tensor(pb.tables[r], device=DEV)


@pytest.mark.parametrize("nq,nkv,d,page", PACKED + [(4, 2, 48, 8)])
@pytest.mark.parametrize("rows,window", [(SINGLE, 16), ([(3000, 1), (5000, 1), (7, 1), (600, 1)], 512), ([(1000, 40), (2000, 3), (0, 9), (70, 1)], 33)])
def test_write_and_read_behind_windows(nq, nkv, d, page, rows, window):
    """Every token goes to its own place, and nothing else changes; what is read back is what the pages hold."""
    pb = cu.Packed8(rows, page, nkv, d, window, seed=d)
    before = [(p.codes.clone(), p.exponents.clone()) for p in (pb.k8, pb.v8)]
    qkv, _ = _projection(pb.num_tokens, nq, nkv, d, 5)
    q = torch.empty((pb.num_tokens, nq, d), dtype=torch.bfloat16, device=DEV)
    ops.qk_norm_rope_kv(q, pb.k8, pb.v8, qkv, None, None, None, 0, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, page, pb.status)
    k, v = (torch.empty((pb.num_tokens, nkv, d), dtype=torch.float32, device=DEV) for _ in range(2))
    ops.read_cache(k, v, pb.k8, pb.v8, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, pb.status)
    assert pb.status.item() == 0
    x = qkv.double().view(pb.num_tokens, nq + 2 * nkv, d)
    pages = torch.cat([_whole(pb, r)[torch.arange(s, s + n, device=DEV) // page] for r, (s, n) in enumerate(rows)])
    slots = pb.positions.long() % page
    for pool, (codes, exps), want, read in ((pb.k8, before[0], x[:, nq:nq + nkv], k), (pb.v8, before[1], x[:, nq + nkv:], v)):
        cu.check_held(pool.codes[pages, :, slots], pool.exponents[pages, :, slots], want, 0.0)  # (neither normed nor rotated: one rounding)
        assert torch.equal(read.double(), cu.values64(pool.codes[pages, :, slots], pool.exponents[pages, :, slots]))
        pool.codes[pages, :, slots], pool.exponents[pages, :, slots] = codes[pages, :, slots], exps[pages, :, slots]
        assert torch.equal(pool.codes, codes) and torch.equal(pool.exponents, exps)


@pytest.mark.parametrize("nq,nkv,d,page", PACKED)
@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("rows,window", [
    (SINGLE, 16), ([(3000, 1), (5000, 1), (7, 1), (600, 1)], 512), ([(100 + 77 * i, 1) for i in range(40)], 100),  # single tokens
    ([(700, 5), (1000, 5), (3, 5), (2000, 4)], 64),  # drafted ones
    ([(900, 1), (3000, 90), (4000, 200), (2500, 33)], 200),  # prompts behind more than they bring
    ([(300, 1), (250, 300), (500, 700), (0, 200), (90, 260)], 40),  # prompts over unpacked pages
])
def test_attention_of_rows_behind_their_windows(nq, nkv, d, page, rows, window, sink):
    pb = cu.Packed8(rows, page, nkv, d, window, seed=d)
    q, out = _attend(pb, nq, d, 0.1, window, sink)
    _close(pb, q, out, 0.1, window, sink)


@pytest.mark.parametrize("rows", [[(40, 1), (60, 1)], [(40, 5), (60, 5)], [(40, 70), (60, 100)]])
@pytest.mark.parametrize("d", [64, 128])
def test_a_short_table_ahead_of_another_row_s(rows, d):
    """Without a window every row's table is whole and ends where the next one begins: a row whose own is too short does not go on in the next one's."""
    pb = cu.Batch8(rows, 16, 2, d, seed=3)
    short = len(pb.tables[0]) - 1
    pb.page_indices = torch.tensor(pb.tables[0][:short] + pb.tables[1], dtype=torch.int32, device=DEV)
    pb.page_indptr = torch.tensor([0, short, short + len(pb.tables[1])], dtype=torch.int32, device=DEV)
    q, out = _attend(pb, 16, d, 0.1)
    assert pb.status.item() == 2


def test_rows_and_places_outside_the_tables():
    """A position, a row or a beginning that leads out of the tables raises the status word; nothing is written or read."""
    nkv, d, page = 2, 64, 16
    for what in ("ahead", "behind", "row", "position"):
        pb = cu.Batch8([(0, 20), (40, 1)], page, nkv, d, seed=3)
        if what == "ahead":
            pb.page_indptr = torch.tensor([-2, 2, 5], dtype=torch.int32, device=DEV)
        elif what == "behind":
            pb.page_indptr = torch.tensor([4, 2, 5], dtype=torch.int32, device=DEV)
            pb.page_indices = pb.page_indices[:5].contiguous()
        elif what == "row":
            pb.row_of_token[:20] = torch.tensor([2, -1] * 10, dtype=torch.int32, device=DEV)
        else:
            pb.positions[:20] = -1 - torch.arange(20, dtype=torch.int32, device=DEV)
        there = 1 if what == "behind" else 0  # (row 0's first page is then the last of the table)
        k, v = (torch.full((21, nkv, d), 3.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        ops.read_cache(k, v, pb.k8, pb.v8, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, pb.status)
        assert pb.status.item() == 2 and bool((k[16 * there:20] == 3).all()) and bool((v[16 * there:20] == 3).all()), what
        pb.status.zero_()
        before = pb.k8.codes.clone()
        qkv, _ = _projection(21, 2, nkv, d, 1)
        q = torch.empty((21, 2, d), dtype=torch.bfloat16, device=DEV)
        ops.qk_norm_rope_kv(q, pb.k8, pb.v8, qkv, None, None, None, 0, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, page, pb.status)
        changed = (pb.k8.codes != before).any(-1).any(1).any(-1).nonzero().flatten().tolist()
        assert pb.status.item() == 2 and changed == [pb.tables[1][2]], what


def test_exactly_the_pages_that_are_there_are_written():
    """Of a row whose second page is missing the first is written, whichever way it is missing."""
    nkv, d, page = 2, 64, 16
    for bad in ("short", "gone", "beyond"):
        pb = cu.Batch8([(0, 20)], page, nkv, d, seed=3)
        if bad == "short":
            pb.page_indptr = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
        else:
            pb.page_indices[1] = -1 if bad == "gone" else pb.num_pages
        before = pb.k8.codes.clone()
        qkv, _ = _projection(20, 2, nkv, d, 1)
        q = torch.empty((20, 2, d), dtype=torch.bfloat16, device=DEV)
        ops.qk_norm_rope_kv(q, pb.k8, pb.v8, qkv, None, None, None, 0, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, page, pb.status)
        changed = (pb.k8.codes != before).any(-1).any(1).any(-1)
        assert pb.status.item() == 2 and changed.nonzero().flatten().tolist() == [pb.tables[0][0]], bad


@pytest.mark.parametrize("tail", [0, -7, 1 << 30])
def test_tables_with_room_for_more_rows(tail):
    """Whole tables in a ``page_indptr`` of more places than the step has rows, whatever stands in the places behind."""
    rows, nkv, d, page = [(0, 20), (40, 1), (7, 30)], 2, 64, 16
    pb = cu.Batch8(rows, page, nkv, d, seed=3)
    pb.page_indptr = torch.cat([pb.page_indptr, torch.full((5,), tail, dtype=torch.int32, device=DEV)])
    k, v = (torch.empty((pb.num_tokens, nkv, d), dtype=torch.float32, device=DEV) for _ in range(2))
    ops.read_cache(k, v, pb.k8, pb.v8, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, pb.status)
    at = 0
    for r, (s, n) in enumerate(rows):
        k64, v64 = pb.dense64(r)
        assert torch.equal(k[at:at + n].double(), k64[s:]) and torch.equal(v[at:at + n].double(), v64[s:])
        at += n
    qkv, _ = _projection(pb.num_tokens, 4, nkv, d, 1)
    q = torch.empty((pb.num_tokens, 4, d), dtype=torch.bfloat16, device=DEV)
    ops.qk_norm_rope_kv(q, pb.k8, pb.v8, qkv, None, None, None, 0, 1e-6, pb.positions, pb.row_of_token, pb.page_indptr, pb.page_indices, page, pb.status)
    out = torch.empty_like(q)
    ops.attention(out, q, pb.k8, pb.v8, ku.make_context(pb), 0, 0.1, None)
    _close(pb, q, out, 0.1)
    ops.attention(out, q, pb.k8, pb.v8, ku.make_context(pb), 0, 0.1, 10)
    _close(pb, q, out, 0.1, 10)
