"""The 8-bit cache behind the engine where some layers have a window: several requests far past it, steps and generation, against the plain implementation over keys and values
rounded the same way; and the tokens of eager, replayed and preempted runs beside each other."""

from __future__ import annotations

import dataclasses
import random

import pytest
import torch

from miniserve_b200.cache import CacheManager
from miniserve_b200.cache.manager import group_needs
from miniserve_b200.config import Architecture, PartSpec, Qwen3Config, register_architecture, unregister_architecture
from miniserve_b200.engine import LLM, SamplingParams
from miniserve_b200.engine.loader import load_model
from miniserve_b200.engine.step import StepFunction, StepRow
from miniserve_b200.models.qwen3 import qwen3_model_spec
from tests.plain import qwen3_plain as plain
from tests.test_cache8_engine_gpu import _folder, _plain_logits8

pytestmark = pytest.mark.gpu
WINDOWS, PAGE = [24, None, 40], 8


def _window_spec(cfg: Qwen3Config):
    spec = qwen3_model_spec(cfg)
    layers = tuple(dataclasses.replace(layer, mixer=PartSpec(layer.mixer.kind, dict(layer.mixer.params, window=window))) for layer, window in zip(spec.layers, WINDOWS))
    return dataclasses.replace(spec, architecture="ToyWindow8LM", layers=layers)


@pytest.fixture(scope="module", params=[(128, 4, 2), (64, 8, 1), (80, 3, 3)], ids=str)
def folder(request, tmp_path_factory):
    register_architecture(Architecture("ToyWindow8LM", Qwen3Config.from_dict, _window_spec), replace=True)
    path, raw = tmp_path_factory.mktemp("toy_window8"), dict(plain.tiny_config_b(), architectures=["ToyWindow8LM"])
    head_dim, heads, kv_heads = request.param
    raw = dict(raw, hidden_size=256, num_attention_heads=heads, num_key_value_heads=kv_heads, head_dim=head_dim, intermediate_size=512, vocab_size=901, num_hidden_layers=3,
               tie_word_embeddings=True)
    plain.write_random_model(path, raw, seed=21, std=0.05, dtype=torch.bfloat16)
    yield dict(path=path, raw=raw, cfg=dict(plain.read_config(path), windows=WINDOWS), w=plain.read_weights(path), w16=plain.read_weights(path, torch.bfloat16))
    unregister_architecture("ToyWindow8LM")


def test_steps_of_several_requests_past_their_windows(folder, monkeypatch):
    """Portions and single tokens of three requests that have given back different numbers of pages. The bounds of the engine's other tests over an 8-bit cache: the mean of a plain
    bfloat16 run, twice its worst."""
    rng = random.Random(5)
    ids = [[rng.randrange(901) for _ in range(n)] for n in (190, 130, 260)]
    _, _, model = load_model(folder["path"], "bfloat16", "cuda:0")
    pages = [3 * 18 if need.window else 100 for need, _ in group_needs(model.entry_caches)[0]]
    cache = CacheManager(model.entry_caches, pages, PAGE, 3, dtype=model.dtype, device=model.device, poison=True, poison_on_free=True, step_tokens=90, kv_dtype="fp8")
    step = StepFunction(model, cache)
    requests, got, at = [cache.new_request() for _ in ids], [[] for _ in ids], [0] * len(ids)
    for sizes in ((60, 0, 90), (1, 40, 80), (70, 1, 1), (5, 5, 5), (1, 1, 1), (1, 1, 1), (2, 60, 1), (30, 1, 60), (1, 1, 1), (1, 1, 1)):
        rows = sorted(((i, StepRow(requests[i], ids[i][at[i]:at[i] + n], tuple(range(n)))) for i, n in enumerate(sizes) if n), key=lambda r: len(r[1].tokens))
        logits, k = step.run([r for _, r in rows]).cpu(), 0
        step.check_status()
        for i, r in rows:
            got[i].append(logits[k:k + len(r.tokens)])
            k, at[i] = k + len(r.tokens), at[i] + len(r.tokens)
    errs, noise = [], []
    for i, n in enumerate(at):
        want = _plain_logits8(monkeypatch, folder["cfg"], folder["w"], ids[i][:n])
        errs.append((torch.cat(got[i]) - want).abs().max(1).values)
        noise.append((_plain_logits8(monkeypatch, folder["cfg"], folder["w16"], ids[i][:n]).float() - want).abs().max(1).values)
    errs, noise = torch.cat(errs), torch.cat(noise)
    assert errs.mean() <= noise.mean() and errs.max() <= 2 * noise.max(), (errs.mean().item(), errs.max().item(), noise.mean().item(), noise.max().item())
    windowed = [e for e, w in enumerate(WINDOWS) if w]
    for e in range(3):
        n = requests[0].num_tokens
        if e in windowed:
            with pytest.raises(ValueError, match="left the window"):
                cache.read(requests[0], e)
        k, v = cache.read(requests[0], e, n - 20, n)
        assert k.shape[0] == 20 and bool(k.isfinite().all()) and bool(v.isfinite().all())
    for rc in requests:
        cache.release(rc)
    assert cache.is_idle()


def _runs(path, prompts, new, chunk, **all_runs):
    params, outs = SamplingParams(max_new_tokens=new), {}
    for name, kwargs in all_runs.items():
        llm = LLM(path, dtype="bfloat16", page_size=PAGE if "page_size" not in kwargs else kwargs.pop("page_size"), max_running=5, chunked_prefill_size=chunk, kv_cache_dtype="fp8",
                  poison_on_free=True, **kwargs)
        outs[name] = llm.generate(prompts, params)
        assert llm.engine.cache.is_idle()
        if name == "small":
            assert llm.engine.scheduler.num_preemptions > 0
    return outs


def _check_runs(monkeypatch, cfg, w, w16, prompts, outs):
    """Every token is the plain run's best up to what the engine's own error decides (twice a plain bfloat16 run's worst, on either side); and where two runs part, the two tokens
    are that near each other."""
    for p, *tokens in zip(prompts, *outs.values()):
        for name, o in zip(outs, tokens):
            want = _plain_logits8(monkeypatch, cfg, w, p + o)
            noise = (_plain_logits8(monkeypatch, cfg, w16, p + o).float() - want).abs().max().item()
            rows = want[len(p) - 1:-1]
            gap = rows.max(1).values - rows[torch.arange(len(o)), torch.tensor(o)]
            assert gap.max().item() <= 4 * noise, (name, gap.max().item(), noise)
            first = next((i for i, (a, b) in enumerate(zip(tokens[0], o)) if a != b), None)
            if first is not None:
                assert abs(rows[first, o[first]] - rows[first, tokens[0][first]]).item() <= 4 * noise, (name, first)


def test_generation_past_the_windows(folder, monkeypatch):
    rng = random.Random(9)
    prompts = [[rng.randrange(901) for _ in range(n)] for n in (45, 3, 110, 17, 60)]
    outs = _runs(folder["path"], prompts, 50, 32, eager=dict(cuda_graph=False, kv_pool_tokens=2048), graphs=dict(kv_pool_tokens=2048), small=dict(kv_pool_tokens=320))
    _check_runs(monkeypatch, folder["cfg"], folder["w"], folder["w16"], prompts, outs)


@pytest.mark.parametrize("head_dim,heads,kv_heads", [(128, 4, 2), (64, 4, 1)])
def test_eager_replayed_and_preempted_runs_beside_each_other(tmp_path, monkeypatch, head_dim, heads, kv_heads):
    raw = _folder(tmp_path, head_dim, heads, kv_heads)
    rng = random.Random(5)
    prompts = [[rng.randrange(raw["vocab_size"]) for _ in range(n)] for n in (70, 130, 5, 33, 200)]
    outs = _runs(tmp_path, prompts, 14, 96, eager=dict(cuda_graph=False, kv_pool_tokens=2048, page_size=16), graphs=dict(kv_pool_tokens=2048, page_size=16),
                 small=dict(kv_pool_tokens=240, page_size=16))
    cfg, w, w16 = plain.read_config(tmp_path), plain.read_weights(tmp_path), plain.read_weights(tmp_path, torch.bfloat16)
    _check_runs(monkeypatch, cfg, w, w16, prompts, outs)
