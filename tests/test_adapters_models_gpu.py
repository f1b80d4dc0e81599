"""Adapters of every family that takes them, against the same model with the adapters worked into its matrices, in 32 bits."""

from __future__ import annotations

import pytest
import torch

from miniserve_b200.engine import LLM, SamplingParams

from .test_adapters_names import pairs

pytestmark = pytest.mark.gpu

WEIGHTS = {"qkv": "w_qkv", "o": "w_o", "gate_up": "w_gate_up", "down": "w_down"}


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("name", ["vumedra-tiny", "kovusun-tiny", "tiny-a", "tiny-b"])
def test_adapters_beside_matrices_are_the_matrices_with_them(name, graphs):
    def made(**kw):
        return LLM(random=name, dtype="float32", kv_pool_tokens=2048, page_size=16, max_running=4, max_prefill_tokens=512, cuda_graph=graphs, **kw)

    prompts, params = [[3, 1, 4, 1, 5], [9, 2, 6] * 11, [5]], SamplingParams(max_new_tokens=10)
    llm = made(max_adapters=2, max_adapter_rank=8)
    given = {k: 0.2 * t for k, t in pairs(llm.model, 4, 1).items()}
    llm.engine.load_adapter("x", given, alpha=6)
    without = llm.generate(prompts, params)
    got = llm.generate(prompts, params, adapters="x")
    mixed = llm.generate(prompts, params, adapters=["x", None, "x"])
    merged = made()
    store = llm.engine.adapters
    by_matrix = {id(low): (part, product) for (part, product), low in store.products.items()}
    parts = {}  # the other model's parts, in the same order

    def walk(mine, other):
        parts[id(mine)] = other
        for a, b in zip(mine.sub_parts().values(), other.sub_parts().values()):
            walk(a, b)

    for mine, other in zip(llm.model.layers, merged.model.layers):
        walk(mine, other)
    for matrix, (low, p, first, behind) in store.places.items():
        part, product = by_matrix[id(low)]
        weight = getattr(parts[id(part)], WEIGHTS[product])
        stem = matrix.removesuffix(".weight")
        weight[first:behind] += 1.5 * (given[stem + ".lora_B.weight"].double() @ given[stem + ".lora_A.weight"].double()).float().to(weight.device)
    want = merged.generate(prompts, params)
    assert got == want and got != without and mixed == [want[0], without[1], want[2]]
