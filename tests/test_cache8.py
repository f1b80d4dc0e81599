"""The 8-bit cache's pools and arguments, without a GPU."""

from __future__ import annotations

import pytest
import torch

from miniserve_b200 import ops
from miniserve_b200.ops import cache8


def test_a_pool_says_what_it_is():
    p = ops.Pool8.empty(3, 2, 16, 64, device="cpu")
    assert p.shape == (3, 2, 16, 64) and p.exponents.shape == (3, 2, 16) and p.codes.dtype == torch.uint8


@pytest.mark.parametrize("shape,what", [((3, 2, 16, 40), "multiples of 16"), ((3, 2, 16, 272), "multiples of 16"), ((3, 2, 4, 64), "at least 8"), ((3, 2, 24, 64), "power of two")])
def test_pools_that_no_kernel_takes_are_refused(shape, what):
    with pytest.raises(ValueError, match=what):
        ops.Pool8.empty(*shape, device="cpu")
    assert not cache8.takes(shape[3], shape[2])


def test_pools_of_other_types_and_layouts_are_refused():
    codes, exps = torch.zeros((3, 2, 16, 64), dtype=torch.uint8), torch.zeros((3, 2, 16), dtype=torch.uint8)
    for bad in ((codes.to(torch.int8), exps), (codes, exps.int()), (codes, exps[:2]), (codes[..., 0], exps)):
        with pytest.raises(ValueError):
            ops.Pool8(*bad)
    with pytest.raises(ValueError, match="contiguous"):
        ops.Pool8(codes.transpose(0, 1).contiguous().transpose(0, 1), exps)


def test_pools_on_the_host_are_refused_by_the_kernels():
    p = ops.Pool8.empty(3, 2, 16, 64, device="cpu")
    rows = torch.empty((1, 2, 64))
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.read_cache(rows, rows, p, p, i, i, i, i, i)
    with pytest.raises(TypeError, match="both"):
        ops.read_cache(rows, rows, p, p.codes, i, i, i, i, i)


def test_prompts_are_shared_out_in_ranges_that_a_launch_takes():
    from types import SimpleNamespace

    lib = SimpleNamespace(most_rows=16, max_units=256)
    for lens in ([1, 700, 3, 1, 17, 1200, 30], [5] * 300, [0, 0, 9], [5000], [0], []):
        ctx = SimpleNamespace(num_rows=len(lens) + 2, host_q_len=[1, 1] + lens)
        ranges = cache8._of_one_size(ctx, 2, 4, lib)
        seen = [r for first, rows, _ in ranges for r in range(first, first + rows)]
        assert len(seen) == len(set(seen)) and all(n == 0 or r + 2 in seen for r, n in enumerate(lens))
        for first, rows, most in ranges:
            assert most == max(ctx.host_q_len[first:first + rows]) > 0
            assert rows == 1 or rows * -(-most * 4 // 16) <= 256


# ------------------------------------------------------------------ the cache manager
def _entries(head_dim=64, values=True):
    from miniserve_b200.parts.base import PagedKV
    from miniserve_b200.parts.decoder import EntryCache

    return [EntryCache(0, PagedKV(2, head_dim, values=values)), EntryCache(1, PagedKV(2, head_dim, values=values))]


def test_the_manager_counts_a_byte_a_number_and_one_a_vector():
    from miniserve_b200.cache import CacheManager

    cm = CacheManager(_entries(), 6, 16, 2, device="cpu", kv_dtype="fp8")
    assert cm.bytes_per_token() == 2 * 2 * 2 * 65 and cm.pool_bytes() == 2 * 2 * 7 * 2 * 16 * 65
    view = cm.entry_views[1]
    assert isinstance(view.k, ops.Pool8) and view.k.shape == (7, 2, 16, 64) and view.k.codes.data_ptr() != cm.entry_views[0].k.codes.data_ptr()
    plain = CacheManager(_entries(), 6, 16, 2, device="cpu")
    assert plain.bytes_per_token() == 2 * 2 * 2 * 128


def test_freed_pages_are_poisoned():
    from miniserve_b200.cache import CacheManager

    cm = CacheManager(_entries(), 3, 16, 2, device="cpu", kv_dtype="fp8", poison_on_free=True)
    rc = cm.new_request()
    cm.reserve([(rc, 20)])
    pages = list(rc.tables[0].blocks)
    cm.release(rc)
    for e in (0, 1):
        k = cm.entry_views[e].k
        assert bool((k.exponents[pages] == 255).all()) and bool((k.codes[pages] == 0x7F).all())
        assert not bool((k.exponents == 255).all())


@pytest.mark.parametrize("kwargs,what", [(dict(page=4), "at least 8"), (dict(head_dim=40), "multiples of 16"), (dict(values=False), "latent"),
                                         (dict(dtype=torch.float32), "bfloat16 model"), (dict(kv_dtype="int4"), "kv_dtype")])
def test_what_an_8_bit_cache_does_not_go_with(kwargs, what):
    from miniserve_b200.cache import CacheManager

    kwargs = dict(kwargs)
    page, entries = kwargs.pop("page", 16), _entries(kwargs.pop("head_dim", 64), kwargs.pop("values", True))
    with pytest.raises(ValueError, match=what):
        CacheManager(entries, 3, page, 2, device=None, **{"kv_dtype": "fp8", **kwargs})


def test_models_with_other_mixers_are_refused():
    from miniserve_b200.config import preset, resolve
    from miniserve_b200.parts.decoder import DecoderModel

    def build(name, dtype):
        return DecoderModel(resolve(preset(name))[2], dtype, "cpu")

    build("tiny-b", torch.bfloat16).check_cache8(16)
    for name, dtype, what in (("tiny-b", torch.float32, "bfloat16 model"), ("fekulix-tiny", torch.bfloat16, "run entry"), ("mugipel-tiny", torch.bfloat16, "run entry|latent")):
        with pytest.raises(ValueError, match=what):
            build(name, dtype).check_cache8(16)


def test_an_engine_s_cache_is_of_the_type_asked_for():
    from miniserve_b200.cache import CacheManager
    from miniserve_b200.engine.engine import Engine

    plain = CacheManager(_entries(), 6, 16, 2, device=None)
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        Engine(None, cache=plain, kv_cache_dtype="fp8")


def test_a_cache_on_the_host_s_books_alone_has_nothing_to_read():
    from miniserve_b200.cache import CacheManager

    cm = CacheManager(_entries(), 6, 16, 2, device=None, kv_dtype="fp8")
    rc = cm.new_request()
    cm.reserve([(rc, 20)])
    with pytest.raises(ValueError, match="no pools"):
        cm.read(rc, 0)


def test_the_command_line_has_the_option():
    import argparse

    from miniserve_b200.engine.cli import add_engine_args, engine_kwargs

    ap = argparse.ArgumentParser()
    add_engine_args(ap)
    assert engine_kwargs(ap.parse_args(["--kv-cache-dtype", "fp8"]))["kv_cache_dtype"] == "fp8"
    assert engine_kwargs(ap.parse_args([]))["kv_cache_dtype"] == "auto"


def test_items_that_get_a_cta_each_are_those_that_the_kernel_finds():
    """The host's rule, against its words: as many slices of 32 keys as an item's rows see and 2 for going on to it, shared by 8 warps; a third and one more than in equal runs, at most 3."""
    from types import SimpleNamespace

    lib = SimpleNamespace(slice=32, alone_most=lambda each: each + min(3, 1 + each // 3), switch=2, warps=lambda tile_rows: 8)

    def alone(rows, nkv=8, heads=2, window=0, tiles=1, tile_rows=8, **more):
        ctx = SimpleNamespace(**{**dict(sm_count=148, host_q_start=[s for s, _ in rows], host_q_len=[n for _, n in rows]), **more})
        return cache8._alone(ctx, lib, range(len(rows)), range(tiles), tile_rows, heads, nkv, window)

    assert alone([(299, 1)]) and alone([(16 * 32 - 1, 1)]) and not alone([(16 * 32, 1)])  # 16 slices are 2 a warp, equal runs 1
    assert alone([(2047, 1)] * 16) and not alone([(2047, 1)] * 8)  # 64 slices are 8 a warp; equal runs 8 and 4
    assert not alone([(100000, 1)], window=512) and alone([(100000, 1)], window=480)  # 17 slices and 16, where they begin inside one
    assert not alone([(299, 1)], host_q_len=[])
    assert alone([(10, 0), (20, 9)], tiles=3, tile_rows=8)  # rows without tokens have no item
