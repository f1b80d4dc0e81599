"""The 8-bit cache behind the engine: the logits of steps against the plain implementation with quantised keys and values, generation with graphs
and without, preemption, and what the manager reads back."""

from __future__ import annotations

import random

import pytest
import torch

from miniserve_b200.cache import CacheManager
from miniserve_b200.engine import LLM, SamplingParams
from miniserve_b200.engine.loader import load_model
from miniserve_b200.engine.step import StepFunction, StepRow
from tests import cache8_util as cu
from tests.plain import qwen3_plain as plain

pytestmark = pytest.mark.gpu
PAGE = 16


def _quantised(x):
    """x [n, heads, d] as the cache gives it back (float32): to the nearest code, ties to even."""
    x64 = x.double()
    e = cu.exponent64(x64)[..., None]
    y = x64 * torch.exp2(-e)
    lead = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -40))).clamp_min(-6)
    step = torch.exp2(lead - 3)
    return (torch.round(y / step) * step * torch.exp2(e)).float()


def _plain_logits8(monkeypatch, cfg, w, ids):
    """The plain float32 implementation with every layer's keys and values through the 8-bit format."""
    real = plain.causal_attention
    with monkeypatch.context() as m:
        m.setattr(plain, "causal_attention", lambda q, k, v, window=None: real(q, _quantised(k).to(q.dtype), _quantised(v).to(q.dtype), window))
        return plain.all_logits(cfg, w, ids)


def _folder(tmp_path, head_dim, heads, kv_heads, layers=2):
    raw = dict(plain.tiny_config_b(), hidden_size=256, num_attention_heads=heads, num_key_value_heads=kv_heads, head_dim=head_dim, intermediate_size=512, vocab_size=901,
               num_hidden_layers=layers, tie_word_embeddings=True)
    plain.write_random_model(tmp_path, raw, seed=21, std=0.05, dtype=torch.bfloat16)
    return raw


@pytest.mark.parametrize("head_dim,heads,kv_heads", [(128, 4, 2), (64, 8, 2), (80, 3, 3)])
def test_logits_of_portions_and_single_tokens(tmp_path, monkeypatch, head_dim, heads, kv_heads):
    """Two requests in portions of every size, one of them token by token at the end. The engine's bfloat16 arithmetic may be as far from the plain
    float32 run over the quantised cache as a plain bfloat16 run over it is (mean) and twice its worst."""
    _folder(tmp_path, head_dim, heads, kv_heads)
    cfg, w = plain.read_config(tmp_path), plain.read_weights(tmp_path)
    rng = random.Random(7)
    a, b = ([rng.randrange(901) for _ in range(n)] for n in (230, 47))
    _, _, model = load_model(tmp_path, "bfloat16", "cuda:0")
    cache = CacheManager(model.entry_caches, 30, PAGE, 3, dtype=model.dtype, device=model.device, poison=True, poison_on_free=True, kv_dtype="fp8")
    step = StepFunction(model, cache)
    ra, rb = cache.new_request(), cache.new_request()
    got = {0: [], 1: []}
    ia = ib = 0
    for na, nb in ((150, 0), (3, 40), (70, 1), (1, 1), (1, 1), (1, 2), (1, 1), (1, 1), (2, 0)):
        rows = []
        for which, rc, ids, at, n in ((0, ra, a, ia, na), (1, rb, b, ib, nb)):
            if n:
                rows.append((which, StepRow(rc, ids[at:at + n], tuple(range(n)))))
        rows.sort(key=lambda r: len(r[1].tokens))  # single tokens at the front, as the scheduler has them
        logits = step.run([r for _, r in rows]).cpu()
        step.check_status()
        at = 0
        for which, r in rows:
            got[which].append(logits[at:at + len(r.tokens)])
            at += len(r.tokens)
        ia, ib = ia + na, ib + nb
    errs, noise = [], []
    wb = plain.read_weights(tmp_path, torch.bfloat16)
    for which, ids, n in ((0, a, ia), (1, b, ib)):
        want = _plain_logits8(monkeypatch, cfg, w, ids[:n])
        errs.append((torch.cat(got[which]) - want).abs().max(1).values)
        noise.append((_plain_logits8(monkeypatch, cfg, wb, ids[:n]).float() - want).abs().max(1).values)
    errs, noise = torch.cat(errs), torch.cat(noise)
    assert errs.mean() <= noise.mean() and errs.max() <= 2 * noise.max(), (errs.mean().item(), errs.max().item(), noise.mean().item(), noise.max().item())
    # what the manager reads back is what the format holds, in both types
    for entry in range(len(cache.entry_views)):
        k, v = cache.read(ra, entry)
        k32, v32 = cache.read(ra, entry, 5, 131, dtype=torch.float32)
        assert k.dtype == torch.bfloat16 and k.shape == (ia, kv_heads, head_dim) and torch.equal(k[5:131].float(), k32) and torch.equal(v[5:131].float(), v32)
        assert torch.equal(_quantised(v32.cpu()), v32.cpu())  # a number of the format is kept as it is
    with pytest.raises(ValueError, match="positions"):
        cache.read(ra, 0, 0, ia + 1)
    cache.release(ra)
    cache.release(rb)
    assert cache.is_idle()


def test_reading_a_bfloat16_cache(tmp_path):
    _folder(tmp_path, 64, 4, 2)
    _, _, model = load_model(tmp_path, "bfloat16", "cuda:0")
    out = {}
    for kv in ("auto", "fp8"):
        cache = CacheManager(model.entry_caches, 8, PAGE, 2, dtype=model.dtype, device=model.device, kv_dtype=kv)
        rc = cache.new_request()
        StepFunction(model, cache).run([StepRow(rc, list(range(40)), (39,))])
        out[kv] = cache.read(rc, 0)
    for x, y in zip(out["auto"], out["fp8"]):  # the first layer's: the same numbers, rounded differently: 2^-8 and 2^-4, and half the smallest code (2^-10 of 2^e, e by the largest / 448)
        bound = x.float().abs() * (2.0 ** -8 + 2.0 ** -4) + 2.0 ** -10 * 2 * x.float().abs().amax(-1, keepdim=True) / 448
        assert bool(((x.float() - y.float()).abs() <= bound).all())


@pytest.mark.parametrize("head_dim,heads,kv_heads", [(128, 4, 2), (64, 4, 1)])
def test_generation_with_graphs_and_without(tmp_path, monkeypatch, head_dim, heads, kv_heads):
    """Greedy tokens through replayed decode and step graphs are those of eager steps; a pool that is too small preempts and gives the same."""
    raw = _folder(tmp_path, head_dim, heads, kv_heads)
    rng = random.Random(5)
    prompts = [[rng.randrange(raw["vocab_size"]) for _ in range(n)] for n in (70, 130, 5, 33, 200)]
    params = SamplingParams(max_new_tokens=14)
    outs = {}
    for name, kwargs in (("eager", dict(cuda_graph=False)), ("graphs", {}), ("small", dict(kv_pool_tokens=400))):
        llm = LLM(tmp_path, dtype="bfloat16", page_size=PAGE, max_running=5, chunked_prefill_size=96, kv_cache_dtype="fp8", poison_on_free=True,
                  **{"kv_pool_tokens": 2048, **kwargs})
        outs[name] = llm.generate(prompts, params)
        outs[name + " again"] = llm.generate(prompts, params)
        assert llm.engine.cache.is_idle() and llm.engine.describe()["kv_cache_dtype"] == "fp8"
    # Every token is the best of the plain run over the quantised cache, or so near that the engine's own error (twice the worst of a plain bfloat16 run, on either side) decides
    cfg, w, wb = plain.read_config(tmp_path), plain.read_weights(tmp_path), plain.read_weights(tmp_path, torch.bfloat16)
    for name, out in outs.items():
        for p, o in zip(prompts, out):
            assert len(o) == 14
            if name.endswith("again") and o == outs[name[:-6]][prompts.index(p)]:
                continue
            want = _plain_logits8(monkeypatch, cfg, w, p + o)
            noise = (_plain_logits8(monkeypatch, cfg, wb, p + o).float() - want).abs().max().item()
            rows = want[len(p) - 1:-1]
            gap = rows.max(1).values - rows[torch.arange(14), torch.tensor(o)]
            assert gap.max().item() <= 4 * noise, (name, gap.max().item(), noise)
    assert outs["graphs"] == outs["graphs again"]


def test_an_engine_that_cannot_have_it_says_so(tmp_path):
    _folder(tmp_path, 64, 4, 2)
    with pytest.raises(ValueError, match="bfloat16 model"):
        LLM(tmp_path, dtype="float32", kv_pool_tokens=256, kv_cache_dtype="fp8")
    with pytest.raises(ValueError, match="run entry|latent"):
        LLM(random="mugipel-tiny", kv_pool_tokens=256, kv_cache_dtype="fp8")
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        LLM(tmp_path, kv_pool_tokens=256, kv_cache_dtype="int4")
