"""Adapters of bfloat16 beside a product whose output is asked for in 32 bits: nothing on the way to it is rounded to fewer."""

from __future__ import annotations

import pytest
import torch

from . import adapters_util as au
from .test_adapters_gpu import DECODE64, EIGHT, LONG, MIXED, run_linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,k,parts,rank", [(EIGHT[:1], 64, (200,), 8), (EIGHT, 64, (264, 96, 72), 40), (DECODE64, 128, (1000, 24), 16), (MIXED, 72, (512, 256, 256), 136), (LONG, 64, (77, 400), 72),
                                               (LONG, 4096, (128,), 8)])
def test_terms_keep_32_bits(rows, k, parts, rank):
    """The weight is zero, so the output is the adapters' terms. x, A and B are given exactly, so what is off are sums of k and rank products in 32 bits, the scale, and what the kernels split v into
    for the tensor cores. v: each of k additions and the scale are off by 2^-23 of a partial sum at most (an addition may truncate), no larger than the products' magnitudes. The split into three
    numbers of 8 bits: 2^-22 counts more than the 2^-24 that it leaves out. The sum over the rank: 2^-23 of the terms' magnitudes an addition, three for each product."""
    x, w, low, ar = au.made(rows, k, parts, rank, 4, torch.bfloat16, seed=rank)
    w.zero_()
    got = run_linear(x, w, low, ar, torch.float32)
    slot, x64 = ar.slot_of_row[ar.row_of_token.long()], x.double()
    want, tol = torch.zeros(got.shape, dtype=torch.float64, device="cuda"), torch.zeros(got.shape, dtype=torch.float64, device="cuda")
    for s in range(low.slots):
        mine, at = (slot == s).nonzero()[:, 0], 0
        for p, end in enumerate(low.ends):
            a, b, c = low.a[s, p * rank:(p + 1) * rank].double(), low.b[s, at:end].double(), float(low.scale[s])
            v, mags = c * (x64[mine] @ a.T), c * (x64[mine].abs() @ a.abs().T)
            want[mine, at:end] = v @ b.T
            tol[mine, at:end] = 2.0 ** -23 * (k + 2) * (mags @ b.abs().T) + (2.0 ** -22 + 2.0 ** -23 * (3 * rank + 4)) * (v.abs() @ b.abs().T)
            at = end
    au.close(got, want, tol)
