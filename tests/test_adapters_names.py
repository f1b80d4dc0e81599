"""Adapters of models whose tensors' names do not end in ``.weight``, without a GPU."""

from __future__ import annotations

import pytest
import torch

from miniserve_b200.engine.adapters import AdapterStore

from .test_adapters_engine import model


def pairs(m, rank, seed=0):
    """Random pairs for every matrix that takes one, by its name without ``.weight``."""
    gen, out = torch.Generator().manual_seed(seed), {}
    for matrix in AdapterStore(m, 1, 8).places:
        n, k = m.weight_decls()[matrix].shape
        stem = matrix.removesuffix(".weight")
        out[stem + ".lora_A.weight"], out[stem + ".lora_B.weight"] = torch.randn((rank, k), generator=gen), torch.randn((n, rank), generator=gen)
    return out


@pytest.mark.parametrize("name", ["vumedra-tiny", "kovusun-tiny", "tiny-b"])
def test_every_place_can_be_named(name):
    m = model(name)
    store, given = AdapterStore(m, 1, 8), pairs(m, 3)
    assert len(given) == 2 * len(store.places) > 0
    store.load("x", given)
    for matrix, (low, part, first, behind) in store.places.items():
        stem = matrix.removesuffix(".weight")
        assert torch.equal(low.a[0, 8 * part:8 * part + 3], given[stem + ".lora_A.weight"]) and torch.equal(low.b[0, first:behind, :3], given[stem + ".lora_B.weight"])
    with pytest.raises(ValueError, match="no projection"):
        AdapterStore(m, 1, 8).load("x", {"nothing.lora_A.weight": torch.zeros((3, 8)), "nothing.lora_B.weight": torch.zeros((8, 3))})
