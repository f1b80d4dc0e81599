"""Rows of the fewest tokens that a cluster of CTAs has, launched in great number behind one another."""

from __future__ import annotations

import math

import pytest
import torch

from .test_sample_filtered_gpu import f32, peaked, plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [16384, 16385, 17000])
@pytest.mark.parametrize("rows", [1, 9, 40])  # (16 CTAs a row, 16, 8)
def test_filtered_rows_of_few_tokens_a_cta(vocab, rows):
    """Every fourth row has no random number (its CTAs leave at once); short kernels run between the calls."""
    from miniserve_b200 import ops

    logits, gen = peaked(rows, vocab, rows)
    u = torch.rand((rows,), generator=gen, device="cuda", dtype=torch.float64)
    u[3::4] = math.nan
    t, p = (torch.full((rows,), x, device="cuda") for x in (0.9, 0.7))
    k = torch.tensor([5 if i % 2 else 0 for i in range(rows)], dtype=torch.int32, device="cuda")
    tokens = [torch.full((rows,), -7, dtype=torch.int32, device="cuda") for _ in range(100)]
    wide, narrow = torch.empty(256, device="cuda"), torch.ones(256, dtype=torch.bfloat16, device="cuda")
    for i, out in enumerate(tokens):
        if i % 3 == 0:
            ops.to_float(wide, narrow)
        ops.sample_filtered(out, logits, t, u, top_k=k, top_p=p)
    want = [-7 if i % 4 == 3 else plain(logits[i], f32(0.9), float(u[i]), int(k[i]), f32(0.7)) for i in range(rows)]
    assert all(out.tolist() == want for out in tokens)


@pytest.mark.parametrize("rows", [1, 9])
def test_nucleus_rows_of_few_tokens_a_cta(rows):
    """Rows by top_p, by temperature alone and greedy ones, a cluster each: the same tokens in every launch, and of the greedy rows the first of the likeliest."""
    from miniserve_b200 import ops

    logits, _ = peaked(rows, 16385, 2)
    scratch = torch.empty(rows * ops.nucleus_bytes(), dtype=torch.uint8, device="cuda")
    kinds = [(0.9, 0.7), (1.1, 1.0), (0.0, 1.0)]
    t, p = (torch.tensor([kinds[i % 3][q] for i in range(rows)], device="cuda") for q in range(2))
    seed, counter = torch.arange(rows, device="cuda"), torch.arange(rows, device="cuda") + 5
    tokens = [torch.full((rows,), -7, dtype=torch.int32, device="cuda") for _ in range(200)]
    for out in tokens:
        ops.sample(out, logits, temperature=t, top_p=p, seed=seed, counter=counter, scratch=scratch)
    first = tokens[0].tolist()
    assert all(out.tolist() == first for out in tokens)
    assert all(first[i] == int(logits[i].argmax()) for i in range(2, rows, 3)) and all(0 <= x < 16385 for x in first)
