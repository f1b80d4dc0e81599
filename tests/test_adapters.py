"""Adapters' shapes and arguments, without a GPU."""

from __future__ import annotations

import pytest
import torch

from miniserve_b200 import ops


def _low(slots=3, parts=2, rank=8, k=16, n=20, ends=(12, 20), dtype=torch.bfloat16, **other):
    t = dict(a=torch.zeros((slots, parts * rank, k), dtype=dtype), b=torch.zeros((slots, n, rank), dtype=dtype), scale=torch.ones(slots))
    t.update(other)
    return ops.LowRank(t["a"], t["b"], t["scale"], ends)


def test_adapters_say_what_they_are():
    low = _low()
    assert (low.slots, low.rank, low.parts, low.inputs, low.outputs, low.ends) == (3, 8, 2, 16, 20, (12, 20))
    zeros = ops.LowRank.zeros(2, 24, (5,), 16, torch.float32, device="cpu")
    assert zeros.a.shape == (2, 16, 24) and zeros.b.shape == (2, 5, 16) and zeros.parts == 1 and not bool(zeros.scale.any())


@pytest.mark.parametrize("kwargs,error,what", [
    (dict(rank=12), ValueError, "multiple of 8"), (dict(rank=264), ValueError, "multiple of 8"), (dict(k=12), ValueError, "multiple of 8"),
    (dict(parts=3), ValueError, "parts"), (dict(ends=(12, 19)), ValueError, "end at"), (dict(ends=(0, 20)), ValueError, "end at"),
    (dict(ends=(20, 12)), ValueError, "end at"), (dict(ends=()), ValueError, "parts"), (dict(parts=5, ends=(1, 2, 3, 4, 20)), ValueError, "up to 4 parts"),
    (dict(dtype=torch.float16), TypeError, "bfloat16 or float32"), (dict(b=torch.zeros((3, 20, 8))), TypeError, "one type"),
    (dict(scale=torch.ones(3, dtype=torch.float64)), TypeError, "float32"), (dict(scale=torch.ones(2)), ValueError, "scale"),
    (dict(b=torch.zeros((2, 20, 8), dtype=torch.bfloat16)), ValueError, "slots"), (dict(slots=0), ValueError, "multiple of 8"),
    (dict(a=torch.zeros((16, 3, 16), dtype=torch.bfloat16).transpose(0, 1)), ValueError, "contiguous"),
])
def test_adapters_that_no_kernel_takes_are_refused(kwargs, error, what):
    with pytest.raises(error, match=what):
        _low(**kwargs)


def test_rows_are_int32_lists():
    i = torch.zeros(3, dtype=torch.int32)
    rows = ops.AdapterRows(i[:2].clone(), i)
    assert rows.rows == 2 and rows.tokens == 3
    for bad in ((i.long(), i), (i, i.long()), (i[None], i), (torch.zeros(6, dtype=torch.int32)[::2], i)):
        with pytest.raises(ValueError, match="int32"):
            ops.AdapterRows(*bad)


def test_products_on_the_host_or_of_other_shapes_are_refused():
    low, i = _low(), torch.zeros(4, dtype=torch.int32)
    x, w = torch.zeros((4, 16), dtype=torch.bfloat16), torch.zeros((20, 16), dtype=torch.bfloat16)
    rows = ops.AdapterRows(i, i)
    for call in (lambda **kw: ops.linear(x, w, stream=0, **kw), lambda **kw: ops.linear_silu_mul(x, w, torch.zeros((4, 10), dtype=torch.bfloat16), stream=0, **kw)):
        with pytest.raises(ValueError, match="CUDA"):
            call(low_rank=low, adapter_rows=rows)
        with pytest.raises(TypeError, match="both"):
            call(low_rank=low)
        with pytest.raises(TypeError, match="both"):
            call(adapter_rows=rows)
        with pytest.raises(ValueError, match="tokens"):
            call(low_rank=low, adapter_rows=ops.AdapterRows(i, i[:3].clone()))
    with pytest.raises(ValueError, match="adapters take"):
        ops.linear(x, w[:19].contiguous(), stream=0, low_rank=low, adapter_rows=rows)
    with pytest.raises(TypeError, match="one type"):
        ops.linear(x.float(), w.float(), stream=0, low_rank=low, adapter_rows=rows)


def test_which_way_a_product_goes():
    """The rule's borders: decode steps, narrow products of some hundred tokens beside wide and long ones."""
    way = lambda t, n, k, rank=16, gated=False: ops.adapters.way_of(t, n, k, rank, gated, 148)  # noqa: E731
    assert all(way(t, 4096, 1024) == "stream" for t in (1, 16)) and way(8, 4096, 1024, 32) == way(16, 2048, 1024, gated=True) == "stream"
    assert all(w == "decode" for w in (way(17, 4096, 1024), way(32, 4096, 1024), way(9, 4096, 1024, 32), way(8, 4104, 2048), way(8, 64, 2056)))
    assert way(64, 6144, 4096, 32) == way(64, 6144, 4096, 64) == way(64, 6144, 2048, 32, True) == "decode" and way(65, 6144, 4096, 32) == "apart" and way(512, 6144, 4096, 32) == "pair"
    assert way(32, 12288, 4096, 64, True) == "decode" and "decode" not in (way(65, 12288, 4096, gated=True), way(33, 12288, 4096, 64, True), way(33, 4096, 1024, 64))
    for n, k, gated in ((4096, 4096, False), (4096, 12288, False), (1024, 1024, False), (12288, 4096, True), (8, 8, False)):
        ways = [way(t, n, k, gated=gated) for t in (100, 400, 1600, 6400, 100000)]
        assert ways == sorted(ways) and set(ways) <= {"apart", "pair"}, ways  # from some number of tokens on, the 2-CTA kernel


def test_whose_work_the_numbers_are():
    own = ops.adapters.makes_its_own
    assert own(16, 48) and not own(19, 48) and own(256, 192) and not own(512, 192) and not own(8, 47) and not own(128, 96)


def test_sampling_on_the_host_or_of_other_types_is_refused():
    logits, f, i = torch.zeros((2, 8)), torch.zeros(2), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.sample_filtered(i, logits, f, f)
