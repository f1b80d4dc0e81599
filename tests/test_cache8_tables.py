"""The page tables that the engine's packer makes for a windowed cache group, and what the 8-bit cache's host side makes of them; without a GPU."""

from __future__ import annotations

from types import SimpleNamespace

import pytest

from miniserve_b200.ops import cache8
from tests import cache8_util as cu


def _tables(rows, page):
    out, at = [], 100
    for s, n in rows:
        count = -(-(s + n) // page)
        out.append(list(range(at, at + count)))
        at += count
    return out


def test_tables_of_a_window_begin_ahead_of_their_entries():
    """What makes these tables different: rows begin at negative places and inside other rows' entries, and a difference of neighbours is not a row's length."""
    indptr, indices = cu.packed_tables([(40, 1), (60, 1)], 8, 16, _tables([(40, 1), (60, 1)], 8))
    assert indptr == [-2, 0, 8] and len(indices) == 8
    assert indices[indptr[0] + 5] == 105 and indices[indptr[1] + 7] == 106 + 7


@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("window", [0, 1, 16, 100, 512])
def test_the_pages_that_are_unpacked_are_those_that_a_row_looks_at(page, window):
    """Counted through the rows, the pages from the first that a row's window reaches to its last: all of them lie in the row's table, and none ahead of them is asked for."""
    rows = [(3000, 300), (0, 40), (5, 1), (777, 64), (2048, 2)]
    indptr, indices = cu.packed_tables(rows, page, window, _tables(rows, page))
    ctx = SimpleNamespace(num_rows=len(rows), host_q_start=[s for s, _ in rows], host_q_len=[n for _, n in rows])
    parts = cache8._parts(ctx, 0, window, page, 1)
    looked_at = []
    for r, (s, n) in enumerate(rows):
        seen = sorted({p // page for q in range(s, s + n) for p in range(max(0, q - window + 1) if window else 0, q + 1)})
        assert all(0 <= indptr[r] + e < len(indices) and indices[indptr[r] + e] >= 100 for e in seen)
        looked_at.append(len(seen))
    assert parts == [(0, len(rows), sum(looked_at))]


def test_parts_of_rows_without_tokens_have_no_pages():
    ctx = SimpleNamespace(num_rows=4, host_q_start=[0, 50, 7, 9], host_q_len=[0, 0, 3, 0])
    assert cache8._parts(ctx, 0, 0, 16, 1) == [(0, 4, 1)]
    assert cache8._parts(ctx, 3, 0, 16, 1) == []


def test_parts_are_cut_by_the_bytes_of_their_pages(monkeypatch):
    monkeypatch.setattr(cache8, "UNPACKED_BYTES", 1000)
    ctx = SimpleNamespace(num_rows=4, host_q_start=[0, 160, 1600, 0], host_q_len=[16, 16, 32, 5])
    assert cache8._parts(ctx, 0, 0, 16, 100) == [(0, 1, 1), (1, 2, 11), (2, 3, 102), (3, 4, 1)]
    assert cache8._parts(ctx, 0, 40, 16, 100) == [(0, 3, 1 + 4 + 5), (3, 4, 1)]


def test_an_engine_with_a_cache_of_its_caller_s_checks_the_model_too():
    """The error is the one of an engine that makes its own cache, before any step."""
    import torch

    from miniserve_b200.cache import CacheManager
    from miniserve_b200.config import preset, resolve
    from miniserve_b200.engine.engine import Engine
    from miniserve_b200.parts.decoder import DecoderModel

    model = DecoderModel(resolve(preset("fekulix-tiny"))[2], torch.bfloat16, "cpu")
    cache = CacheManager(model.entry_caches, 8, 16, 2, device=None, kv_dtype="fp8")
    for dtype in ("auto", "fp8"):
        with pytest.raises(ValueError, match="run entry"):
            Engine(model, cache=cache, kv_cache_dtype=dtype)


@pytest.mark.parametrize("free_gb", [4, 20, 170])
def test_the_pool_leaves_room_for_a_request_as_long_as_it(free_gb, monkeypatch):
    """What a step needs beside the pool fits at the start: a gigabyte of unpacked pages, or the longest request's if that is more."""
    import torch

    from miniserve_b200.engine.engine import Engine
    from miniserve_b200.parts.base import PagedKV
    from miniserve_b200.parts.decoder import EntryCache

    free = free_gb << 30
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (free, free))
    for layers, heads, dim in ((2, 8, 128), (28, 8, 128), (4, 2, 64)):
        model = SimpleNamespace(dtype=torch.bfloat16, device="cuda", entry_caches=[EntryCache(i, PagedKV(heads, dim)) for i in range(layers)],
                                spec=SimpleNamespace(hidden_size=1024, vocab_size=50000))
        reserve = 2048 * 8192 * 16 + 8 * 50000 * 12 + (1 << 30)
        pages, = Engine._pool_pages(model, None, 16, 0.9, 2048, 8, True)
        pool, unpacked = pages * 16 * layers * heads * 2 * (dim + 1), pages * 16 * heads * dim * 4
        room = 0.9 * (free - reserve - (1 << 30))
        assert pool + max(0, unpacked - (1 << 30)) <= room
        assert pool + max(0, unpacked - (1 << 30)) >= room - 16 * layers * heads * 4 * (dim + 1) - 16 * heads * dim * 4 - 1, "all but a page of the room is used"
        plain, = Engine._pool_pages(model, None, 16, 0.9, 2048, 8)
        assert plain == int(0.9 * (free - reserve)) // (2 * layers * heads * dim * 2 * 16)
