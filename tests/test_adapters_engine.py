"""Adapters, top_k and min_p around the engine, without a GPU: what is taken in, what is refused, the random numbers."""

from __future__ import annotations

import json

import numpy as np
import pytest
import torch

from miniserve_b200.config import preset, resolve
from miniserve_b200.engine import SamplingParams
from miniserve_b200.engine.adapters import AdapterStore
from miniserve_b200.parts.decoder import DecoderModel
from miniserve_b200.sampling import sampler


def model(name="tiny-b", dtype=torch.float32):
    return DecoderModel(resolve(preset(name))[2], dtype, "cpu")


def tensors(m, rank, seed=0, only=None):
    """Random pairs for every matrix (or those whose name holds ``only``), by the names that adapters' files have."""
    gen, out = torch.Generator().manual_seed(seed), {}
    for matrix in AdapterStore(m, 1, 8).places:
        if only is None or only in matrix:
            n, k = m.weight_decls()[matrix].shape
            stem = "base_model.model." + matrix[:-len(".weight")]
            out[stem + ".lora_A.weight"], out[stem + ".lora_B.weight"] = torch.randn((rank, k), generator=gen), torch.randn((n, rank), generator=gen)
    return out


def test_every_projection_of_a_dense_layer_takes_adapters():
    m = model()
    store = AdapterStore(m, 3, 5)
    names = {n.split(".", 3)[3] for n in store.places}
    assert names == {f"self_attn.{x}_proj.weight" for x in "qkvo"} | {f"mlp.{x}_proj.weight" for x in ("gate", "up", "down")}
    qkv = store.products[m.layers[0].mixer, "qkv"]
    assert qkv.parts == 3 and qkv.rank == 8 and store.products[m.layers[0].feed_forward, "gate_up"].parts == 2
    assert store.bytes() == sum(t.numel() * t.element_size() for low in store.products.values() for t in (low.a, low.b, low.scale))


def test_an_adapter_lies_where_its_matrix_is_stacked():
    m = model()
    store = AdapterStore(m, 2, 8)
    given = tensors(m, 3)
    assert store.load("first", given, alpha=6) == 0 and store.load("second", tensors(m, 8, 1, only="v_proj")) == 1
    low, stem = store.products[m.layers[0].mixer, "qkv"], "base_model.model.model.layers.0.self_attn."
    assert float(low.scale[0]) == 2.0 and float(low.scale[1]) == 1.0
    for p, x in enumerate("qkv"):
        first = low.ends[p - 1] if p else 0
        assert torch.equal(low.a[0, 8 * p:8 * p + 3], given[stem + f"{x}_proj.lora_A.weight"]) and not bool(low.a[0, 8 * p + 3:8 * p + 8].any())
        assert torch.equal(low.b[0, first:low.ends[p], :3], given[stem + f"{x}_proj.lora_B.weight"]) and not bool(low.b[0, first:low.ends[p], 3:].any())
    assert not bool(low.a[1, :16].any()) and bool(low.a[1, 16:].any())
    assert float(store.products[m.layers[0].mixer, "o"].scale[1]) == 0.0


def test_two_stores_of_one_model_are_apart():
    m = model()
    first, second = AdapterStore(m, 1, 8), AdapterStore(m, 2, 16)
    first.load("a", tensors(m, 4))
    assert all(bool(low.a.any()) for low in first.products.values()) and not any(bool(low.a.any()) for low in second.products.values())


def test_a_freed_place_keeps_nothing_of_the_adapter_before():
    m = model()
    store = AdapterStore(m, 1, 8)
    store.load("wide", tensors(m, 8))
    store.unload("wide")
    store.load("narrow", tensors(m, 2, 1, only="k_proj"))
    for part in (m.layers[0].mixer, m.layers[0].feed_forward):
        for (owner, name), low in store.products.items():
            assert owner is not part or (float(low.scale[0]) == 0.0) == (name != "qkv")
    low = store.products[m.layers[0].mixer, "qkv"]
    assert not bool(low.a[0, :8].any()) and not bool(low.a[0, 16:].any()) and not bool(low.b[0, :low.ends[0]].any()) and not bool(low.b[0, :, 2:].any())


def test_all_that_does_not_fit_is_one_error_and_changes_nothing():
    m = model()
    store = AdapterStore(m, 1, 8)
    good = tensors(m, 4, only="q_proj")
    stem = "base_model.model.model.layers.0.self_attn."
    bad = dict(good)
    bad["base_model.model.lm_head.lora_A.weight"] = torch.zeros((4, 8))
    bad[stem + "k_proj.lora_A.weight"] = torch.zeros((4, m.spec.hidden_size))
    bad[stem + "v_proj.lora_A.weight"], bad[stem + "v_proj.lora_B.weight"] = torch.zeros((4, 7)), torch.zeros((3, 4))
    bad[stem + "o_proj.weight"] = torch.zeros((2, 2))
    with pytest.raises(ValueError) as e:
        store.load("bad", bad)
    for what in ("lm_head", "lora_B is missing", "v_proj.weight: A (4, 7)", "o_proj.weight: no projection"):
        assert what in str(e.value)
    assert not store.names and not any(bool(low.a.any()) for low in store.products.values())
    with pytest.raises(ValueError, match="rank 9"):
        store.load("wide", tensors(m, 9))
    with pytest.raises(ValueError, match="all of an adapter's are one"):
        store.load("two", {**tensors(m, 4, only="q_proj"), **tensors(m, 2, only="o_proj")})
    with pytest.raises(ValueError, match="no tensors"):
        store.load("empty", {})
    store.load("good", good)
    with pytest.raises(ValueError, match="already"):
        store.load("good", good)
    with pytest.raises(ValueError, match="places are taken"):
        store.load("another", good)
    with pytest.raises(ValueError, match="no adapter named"):
        store.unload("another")


def test_numbers_that_are_not_finite_are_refused():
    m = model(dtype=torch.bfloat16)
    store = AdapterStore(m, 1, 8)
    for value in (float("nan"), float("inf"), 3.4e38):  # (the last is finite in 32 bits alone)
        given = tensors(m, 4)
        next(iter(given.values()))[1, 2] = value
        with pytest.raises(ValueError, match="not finite"):
            store.load("bad", given)
    with pytest.raises(ValueError, match="factor"):
        store.load("bad", tensors(m, 4), alpha=float("inf"))
    assert not store.names and not any(bool(low.a.any()) for low in store.products.values())


def test_a_folder_says_rank_and_factor(tmp_path):
    from safetensors.torch import save_file

    m = model()
    with pytest.raises(FileNotFoundError):
        AdapterStore(m, 1, 8).load("x", tmp_path)
    config = dict(r=4, lora_alpha=8, target_modules=["q_proj"])
    (tmp_path / "adapter_config.json").write_text(json.dumps(config))
    with pytest.raises(FileNotFoundError, match="safetensors"):
        AdapterStore(m, 1, 8).load("x", tmp_path)
    save_file(tensors(m, 4, only="q_proj"), str(tmp_path / "adapter_model.safetensors"))
    for extra, factor in ((dict(), 2.0), (dict(use_rslora=True), 4.0), (dict(bias="none"), 2.0)):
        (tmp_path / "adapter_config.json").write_text(json.dumps({**config, **extra}))
        store = AdapterStore(m, 1, 8)
        store.load("x", tmp_path)
        assert float(store.products[m.layers[0].mixer, "qkv"].scale[0]) == factor
        with pytest.raises(ValueError, match="alpha"):
            AdapterStore(m, 1, 8).load("x", tmp_path, alpha=3)
    for extra in (dict(use_dora=True), dict(bias="all"), dict(rank_pattern={"q_proj": 2}), dict(modules_to_save=["lm_head"])):
        (tmp_path / "adapter_config.json").write_text(json.dumps({**config, **extra}))
        with pytest.raises(ValueError, match="nothing for here"):
            AdapterStore(m, 1, 8).load("x", tmp_path)


def test_models_and_sizes_that_take_no_adapters():
    for name in ("fekulix-tiny", "mugipel-tiny"):
        m = model(name)
        kinds = {n.rsplit(".", 2)[1] for n in (AdapterStore(m, 1, 8).places if any(p.adapted_products() for layer in m.layers for p in layer.sub_parts().values()) else ())}
        assert not kinds & {"q_proj", "k_proj", "v_proj"}  # (their attention is not the plain one)
    for slots, rank in ((0, 8), (1, 0), (1, 257)):
        with pytest.raises(ValueError, match="max_adapter"):
            AdapterStore(model(), slots, rank)


def test_engines_without_room_say_so():
    from miniserve_b200.cache import CacheManager
    from miniserve_b200.engine.engine import Engine
    from miniserve_b200.parts.base import PagedKV
    from miniserve_b200.parts.decoder import EntryCache

    class Toy:
        device = dtype = None

        class spec:
            vocab_size = 7

    cache = CacheManager([EntryCache(0, PagedKV(1, 16))], 8, 4, 2, device=None)
    engine = Engine(Toy(), cache=cache, step_fn=object(), sampler=object(), max_running=2)
    for call in (lambda: engine.load_adapter("a", {}), lambda: engine.unload_adapter("a"), lambda: engine.add_request([1], SamplingParams(1), adapter="a"),
                 lambda: engine.generate([[1]], SamplingParams(1), adapters="a")):
        with pytest.raises(ValueError, match="max_adapters"):
            call()
    with pytest.raises(ValueError, match="1 prompts but 2 adapters"):
        engine.generate([[1]], SamplingParams(1), adapters=[None, None])
    assert not engine.has_unfinished


def test_parameters_of_filters():
    for bad in (dict(top_k=-1), dict(top_k=1.5), dict(top_k=1 << 31), dict(min_p=-0.1), dict(min_p=1.1), dict(min_p=float("nan"))):
        with pytest.raises(ValueError, match="top_k|min_p"):
            SamplingParams(4, temperature=1.0, **bad)
    assert not SamplingParams(4, top_k=5).is_filtered and not SamplingParams(4, temperature=1.0, top_p=0.5).is_filtered
    assert SamplingParams(4, temperature=1.0, top_k=5).is_filtered and SamplingParams(4, temperature=1.0, min_p=0.1).is_filtered


def test_random_numbers_of_a_seed_and_a_counter():
    """53 bits in [0, 1), the same for a row wherever it stands, and spread evenly: of 20,000 the share below x is off by less than five standard deviations (0.018)."""
    seeds, counters = [7] * 20000, list(range(20000))
    u = sampler.uniforms(seeds, counters)
    assert u.dtype == np.float64 and float(u.min()) >= 0 and float(u.max()) < 1 and len(set(u.tolist())) == 20000
    assert sampler.uniforms([7, 9, 7], [3, 5, 4]).tolist() == [u[3], sampler.uniforms([9], [5])[0], u[4]]
    for x in (0.1, 0.5, 0.9):
        assert abs(float((u < x).mean()) - x) < 0.018
    by_seed = sampler.uniforms(range(20000), [11] * 20000)
    assert abs(float((by_seed < 0.5).mean()) - 0.5) < 0.018


def test_which_kernels_a_step_s_settings_need():
    def mode(t, p=None, k=None, m=None):
        n = len(t)
        return sampler.settings(t, p, range(n), range(n), k, m, rows=n + 1)

    assert mode([0.0, 0.0]).mode == "greedy" and mode([0.0, 1.0]).mode == "temperature" and mode([0.0, 1.0], [0.5, 1.0]).mode == "top_p"
    assert mode([0.0, 1.0], k=[5, 0]).mode == "temperature"  # (a greedy row's top_k says nothing)
    s = mode([0.0, 1.0], [1.0, 0.5], [0, 3])
    assert s.mode == "filtered" and s.uniform[0] == 0 and 0 <= s.uniform[1] < 1 and s.f32[:, 2].tolist() == [0, 1, 0, 1, 0]
    s = mode([0.7, 1.0, 0.0], [0.9, 0.5, 1.0], [0, 0, 0], [0.0, 0.25, 0.0])
    assert s.mode == "top_p+filtered" and s.uniform[0] == -1 and s.uniform[1] >= 0 and s.uniform[2] == 0
    assert s.f32[0].tolist() == pytest.approx([0.7, 0, 0, 0]) and s.f32[1].tolist() == pytest.approx([0.9, 1, 1, 1]) and s.f32[2].tolist() == [0, 1, 0, 0]
    assert mode([0.7, 1.0], [1.0, 0.5], [0, 4]).mode == "temperature+filtered"


def test_the_command_line_has_the_options():
    import argparse

    from miniserve_b200.engine.cli import add_engine_args, engine_kwargs

    ap = argparse.ArgumentParser()
    add_engine_args(ap)
    kwargs = engine_kwargs(ap.parse_args(["--max-adapters", "3", "--max-adapter-rank", "32"]))
    assert kwargs["max_adapters"] == 3 and kwargs["max_adapter_rank"] == 32 and engine_kwargs(ap.parse_args([]))["max_adapters"] == 0
