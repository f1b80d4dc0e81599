"""Adapters whose files leave more than one reading are refused, without a GPU."""

from __future__ import annotations

import json

import pytest
import torch
from safetensors.torch import save_file

from miniserve_b200.engine.adapters import AdapterStore

from .test_adapters_engine import model, tensors

PREFIX = "base_model.model."


def written(path, parts, **config):
    path.mkdir(exist_ok=True)
    (path / "adapter_config.json").write_text(json.dumps({**dict(r=4, lora_alpha=8), **config}))
    for name, part in parts.items():
        save_file(part, str(path / name))
    return path


def test_a_matrix_that_is_named_in_both_ways():
    m = model()
    store, given = AdapterStore(m, 1, 8), tensors(m, 4, only="q_proj")
    key = next(k for k in given if k.endswith("lora_B.weight"))
    with pytest.raises(ValueError, match="given twice"):
        store.load("x", {**given, key[len(PREFIX):]: given[key] + 1})
    assert not store.names
    store.load("x", {k[len(PREFIX):] if i % 2 else k: t for i, (k, t) in enumerate(given.items())})


def test_a_tensor_that_two_files_hold(tmp_path):
    m = model()
    given = tensors(m, 4, only="q_proj")
    keys = sorted(given)
    halves = {"a.safetensors": {k: given[k] for k in keys[:3]}, "b.safetensors": {k: given[k] for k in keys[3:]}}
    store = AdapterStore(m, 2, 8)
    store.load("x", written(tmp_path / "good", halves))
    halves["b.safetensors"][keys[0]] = torch.zeros_like(given[keys[0]])
    with pytest.raises(ValueError, match="holds too"):
        store.load("y", written(tmp_path / "bad", halves))
    assert list(store.names) == ["x"]


def test_a_rank_that_is_not_the_tensors(tmp_path):
    """The factor is lora_alpha over the rank, so the two have to agree."""
    m = model()
    store = AdapterStore(m, 1, 8)
    with pytest.raises(ValueError, match="says 8"):
        store.load("x", written(tmp_path / "bad", {"a.safetensors": tensors(m, 4, only="q_proj")}, r=8))
    assert not store.names
    store.load("x", written(tmp_path / "bad", {}, r=4))


def test_kinds_of_adapters_that_there_is_nothing_for(tmp_path):
    """Adapters that count behind certain tokens alone, and methods of other names."""
    m = model()
    given = {"a.safetensors": tensors(m, 4, only="q_proj")}
    for i, extra in enumerate((dict(alora_invocation_tokens=[5, 7]), dict(peft_type="ADALORA"))):
        with pytest.raises(ValueError, match="nothing for here"):
            AdapterStore(m, 1, 8).load("x", written(tmp_path / str(i), given, **extra))
    for i, extra in enumerate((dict(alora_invocation_tokens=None, peft_type="LORA"), dict(peft_type=None))):
        AdapterStore(m, 1, 8).load("x", written(tmp_path / f"good{i}", given, **extra))


def test_a_factor_that_32_bits_do_not_hold(tmp_path):
    m = model()
    store, given = AdapterStore(m, 1, 8), tensors(m, 4, only="q_proj")
    with pytest.raises(ValueError, match="32 bits"):
        store.load("x", given, alpha=1e39 * 4)
    with pytest.raises(ValueError, match="32 bits"):
        store.load("x", written(tmp_path / "bad", {"a.safetensors": given}, lora_alpha=-1e40))
    assert not store.names and not any(bool(low.scale.any()) for low in store.products.values())
    store.load("x", given, alpha=4e38)
    assert all(bool(torch.isfinite(low.scale).all()) for low in store.products.values())


def test_a_rank_of_nothing(tmp_path):
    m = model()
    for r in (0, -4):
        with pytest.raises(ValueError, match="says a rank"):
            AdapterStore(m, 1, 8).load("x", written(tmp_path / "bad", {"a.safetensors": tensors(m, 4, only="q_proj")}, r=r))


def test_a_place_keeps_nothing_beside_the_matrices_that_the_next_adapter_does_not_have():
    """A factor of 0 is not enough: numbers of an earlier adapter may give an infinity, which times 0 is no number."""
    m = model()
    store = AdapterStore(m, 1, 8)
    store.load("wide", {k: 1e38 * t.sign() for k, t in tensors(m, 8).items()})
    store.unload("wide")
    store.load("narrow", tensors(m, 2, 1, only="k_proj"))
    for (_, product), low in store.products.items():
        assert bool(low.a[0].any()) == bool(low.b[0].any()) == bool(low.scale[0]) == (product == "qkv")
