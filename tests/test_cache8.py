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
