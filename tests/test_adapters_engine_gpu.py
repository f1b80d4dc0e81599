"""Requests with adapters and with top_k and min_p through the engine, against the plain implementation with the adapters worked into its matrices."""

from __future__ import annotations

import random

import pytest
import torch

from miniserve_b200.engine import LLM, SamplingParams
from tests.plain import qwen3_plain as plain

pytestmark = pytest.mark.gpu

WIDE = dict(plain.tiny_config_b(), hidden_size=1024, num_attention_heads=16, num_key_value_heads=8, head_dim=128, intermediate_size=2048, vocab_size=1000,
            num_hidden_layers=2, tie_word_embeddings=True)
RAWS = {"tiny": plain.tiny_config_b(), "wide": WIDE}
MATRICES = {"all": ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj"), "some": ("q_proj", "v_proj", "up_proj")}


def adapter(w, rank, seed, matrices, std):
    """Pairs by the names of adapters' files; the product of a pair has entries of a size with the matrix's own."""
    gen, out = torch.Generator().manual_seed(seed), {}
    for name, t in w.items():
        if any(name.endswith(m + ".weight") for m in matrices):
            stem = "base_model.model." + name[:-len(".weight")]
            out[stem + ".lora_A.weight"] = (torch.randn((rank, t.shape[1]), generator=gen) * std).bfloat16()
            out[stem + ".lora_B.weight"] = (torch.randn((t.shape[0], rank), generator=gen) * 0.5).bfloat16()
    return out


def merged(w, pairs, factor):
    out = dict(w)
    for name in w:
        stem = "base_model.model." + name[:-len(".weight")]
        if stem + ".lora_A.weight" in pairs:
            out[name] = w[name] + factor * (pairs[stem + ".lora_B.weight"].float() @ pairs[stem + ".lora_A.weight"].float())
    return out


@pytest.fixture(scope="module", params=sorted(RAWS))
def held(request, tmp_path_factory):
    raw = RAWS[request.param]
    path = tmp_path_factory.mktemp(request.param)
    plain.write_random_model(path, raw, 7, std=0.05 if request.param == "tiny" else 0.02, dtype=torch.bfloat16)
    cfg, w = plain.read_config(path), plain.read_weights(path)
    std = 0.0125 if request.param == "tiny" else 0.005  # logits of up to 2 and 3 move by 1.3 to 2.6, and by 0.02 to 0.04 between the two types
    pairs = {"a": adapter(w, 4, 1, MATRICES["all"], std), "b": adapter(w, 13, 2, MATRICES["some"], std), "c": adapter(w, 16, 3, MATRICES["all"], std)}
    alpha = {"a": 8.0, "b": 13.0, "c": 8.0}
    weights = {None: w, **{n: merged(w, pairs[n], alpha[n] / (4, 13, 16)[i]) for i, n in enumerate("abc")}}
    return dict(name=request.param, raw=raw, path=path, cfg=cfg, pairs=pairs, alpha=alpha, weights=weights)


def engine(held, dtype, **kw):
    llm = LLM(held["path"], dtype=dtype, max_adapters=4, max_adapter_rank=16, **{**dict(kv_pool_tokens=4096, page_size=16, max_running=8), **kw})
    for n in "abc":
        llm.engine.load_adapter(n, held["pairs"][n], alpha=held["alpha"][n])
    return llm


def prompts_of(held, lengths, seed):
    rng = random.Random(seed)
    return [[rng.randrange(held["raw"]["vocab_size"]) for _ in range(n)] for n in lengths]


def margins(held, prompt, tokens, name, dtype):
    """How far each token's plain logit lies below the best, teacher-forced. float32: 1e-3, some thousand roundings of 2^-24 on numbers of a size of one.
    bfloat16: with w the most that the plain implementation's own logits move in bfloat16 on this sequence, the engine's may be off by 2 w (the rule of
    ``trace_util.check_bfloat16``); a token that is the engine's best is then at most 4 w below the plain one's."""
    seq = list(prompt) + list(tokens)
    logits = plain.all_logits(held["cfg"], held["weights"][name], seq)
    eps = 1e-3
    if dtype == "bfloat16":
        eps = 4 * float((plain.all_logits(held["cfg"], {k: t.bfloat16() for k, t in held["weights"][name].items()}, seq).float() - logits).abs().max())
        assert eps < 0.2 * float(logits.max()), "the bound says nothing"
    logits = logits[len(prompt) - 1:-1]
    below = logits.max(-1).values - logits.gather(1, torch.tensor(tokens)[:, None])[:, 0]
    assert float(below.max()) <= eps, (name, eps, below.tolist())


NAMES = ["a", None, "b", "a", "c", "b"]


@pytest.mark.parametrize("dtype, kw", [("float32", dict(cuda_graph=False)), ("float32", dict()), ("bfloat16", dict(cuda_graph=False)), ("bfloat16", dict()),
                                       ("bfloat16", dict(chunked_prefill_size=24)), ("bfloat16", dict(overlap=False))])
def test_requests_of_one_batch_have_their_own_adapters(held, dtype, kw):
    prompts = prompts_of(held, [5, 17, 33, 1, 9, 40], 1)
    llm = engine(held, dtype, **kw)
    outs = llm.generate(prompts, SamplingParams(max_new_tokens=12), adapters=NAMES)
    assert llm.engine.cache.is_idle()
    for p, o, n in zip(prompts, outs, NAMES):
        assert len(o) == 12
        margins(held, p, o, n, dtype)
    again = llm.generate(prompts, SamplingParams(max_new_tokens=12), adapters=NAMES)
    if dtype == "float32":
        assert again == outs


def test_requests_that_are_preempted_keep_their_adapters(held):
    prompts = prompts_of(held, [30, 12, 25, 7, 40, 18], 3)
    roomy = engine(held, "float32", chunked_prefill_size=16).generate(prompts, SamplingParams(max_new_tokens=20), adapters=NAMES)
    tight = engine(held, "float32", chunked_prefill_size=16, kv_pool_tokens=128, page_size=8)
    assert tight.generate(prompts, SamplingParams(max_new_tokens=20), adapters=NAMES) == roomy
    assert tight.engine.scheduler.num_preemptions > 0, "the pool was meant to run out"
    assert tight.engine.cache.is_idle()


def test_prompts_of_many_tokens(held):
    """Steps wide enough for the 2-CTA kernel (and, with heads of 128, its q|k|v epilogue): several prompts, decoding requests beside them, graphs replayed."""
    prompts = prompts_of(held, [700, 40, 513, 300], 2)
    llm = engine(held, "bfloat16", chunked_prefill_size=1024)
    for _ in range(3):
        outs = llm.generate(prompts, SamplingParams(max_new_tokens=4), adapters=["a", None, "c", "b"])
    for p, o, n in zip(prompts, outs, ["a", None, "c", "b"]):
        margins(held, p, o, n, "bfloat16")


def test_requests_without_adapters_run_as_in_an_engine_without(held):
    prompts = prompts_of(held, [5, 30, 12], 3)
    plain_llm = LLM(held["path"], dtype="float32", kv_pool_tokens=4096, page_size=16, max_running=8)
    want = plain_llm.generate(prompts, SamplingParams(max_new_tokens=10))
    llm = engine(held, "float32")
    assert llm.generate(prompts, SamplingParams(max_new_tokens=10)) == want
    beside = llm.generate(prompts + prompts, SamplingParams(max_new_tokens=10), adapters=[None] * 3 + ["a", "b", "c"])
    assert beside[:3] == want and beside[3:] != want


def test_adapters_come_and_go(held):
    prompts = prompts_of(held, [20, 9], 4)
    llm = engine(held, "bfloat16", max_running=4)
    req = llm.engine.add_request(prompts[0], SamplingParams(max_new_tokens=6), adapter="a")
    llm.engine.step()
    with pytest.raises(RuntimeError, match="still run"):
        llm.engine.unload_adapter("a")
    while llm.engine.has_unfinished:
        llm.engine.step()
    margins(held, prompts[0], req.output_ids, "a", "bfloat16")
    llm.engine.unload_adapter("a")
    with pytest.raises(ValueError, match="no adapter named 'a'"):
        llm.engine.add_request(prompts[0], SamplingParams(max_new_tokens=6), adapter="a")
    llm.engine.load_adapter("again", held["pairs"]["b"], alpha=held["alpha"]["b"])  # in the place of "a"
    for p, o in zip(prompts, llm.generate(prompts, SamplingParams(max_new_tokens=6), adapters="again")):
        margins(held, p, o, "b", "bfloat16")


# ------------------------------------------------------------------ filters
def test_filters_that_leave_one_token_are_greedy(held):
    prompts = prompts_of(held, [5, 30, 12], 5)
    llm = engine(held, "float32")
    want = llm.generate(prompts, SamplingParams(max_new_tokens=8))
    for kw in (dict(top_k=1), dict(min_p=1.0), dict(top_k=1, top_p=0.3), dict(top_k=900, min_p=1.0)):
        assert llm.generate(prompts, SamplingParams(max_new_tokens=8, temperature=1.3, seed=5, **kw)) == want


@pytest.mark.parametrize("graphs", [False, True])
def test_a_request_draws_the_same_wherever_it_stands(held, graphs):
    """In 32 bits: alone, beside greedy, nucleus and plain sampled ones, with and without graphs; its tokens are among the likeliest k."""
    prompts = prompts_of(held, [5, 30, 12, 8, 21, 3], 6)
    params = [SamplingParams(max_new_tokens=10, temperature=0.9, top_k=4, seed=11), SamplingParams(max_new_tokens=10, temperature=0.8, top_p=0.7, seed=12),
              SamplingParams(max_new_tokens=10), SamplingParams(max_new_tokens=10, temperature=1.2, seed=13),
              SamplingParams(max_new_tokens=10, temperature=1.1, top_p=0.9, min_p=0.2, seed=14), SamplingParams(max_new_tokens=10, temperature=1.0, top_k=1000, seed=15)]
    llm = engine(held, "float32", cuda_graph=graphs)
    together = llm.generate(prompts, params, adapters=["a", None, "b", None, "c", None])
    alone = [llm.generate([p], s, adapters=n)[0] for p, s, n in zip(prompts, params, ["a", None, "b", None, "c", None])]
    assert together == alone
    other = LLM(held["path"], dtype="float32", kv_pool_tokens=4096, page_size=16, max_running=8)
    for i in (1, 3):  # drawn by the noise, as ever
        assert other.generate([prompts[i]], params[i])[0] == together[i]
    seq = list(prompts[0])
    for t in together[0]:
        logits = plain.all_logits(held["cfg"], held["weights"]["a"], seq)[-1]
        assert float(logits[t]) >= float(logits.topk(4).values[-1]) - 1e-3
        seq.append(t)


def test_the_random_numbers_are_the_ones_of_seed_and_counter(held):
    from miniserve_b200.sampling import sampler

    prompt = prompts_of(held, [14], 7)[0]
    llm = engine(held, "float32")
    seq = list(prompt)
    (out,) = llm.generate([prompt], SamplingParams(max_new_tokens=8, temperature=0.7, top_k=6, seed=99))
    for t in out:
        logits = plain.all_logits(held["cfg"], held["weights"][None], seq)[-1].double()
        best = logits.topk(6).indices.sort().values
        sums = torch.cumsum(torch.exp((logits[best] - logits.max()) / 0.7), 0) / torch.exp((logits[best] - logits.max()) / 0.7).sum()
        u = float(sampler.uniforms([99], [len(seq)])[0])
        at = [int(best[min(int((sums <= u + d).sum()), 5)]) for d in (-1e-3, 0.0, 1e-3)]  # (a border as near as the model's rounding may be passed)
        assert t in at
        seq.append(t)


def test_graphs_of_filtered_steps_are_captured_ahead(held):
    llm = engine(held, "bfloat16", max_running=2)
    n = llm.engine.capture_graphs(("greedy", "filtered"))
    assert n == len(llm.engine.graphs._graphs) == 8  # (of one request and of two, steps with adapters and without)
    for name in (None, "b"):
        llm.generate(prompts_of(held, [5], 1), SamplingParams(max_new_tokens=4, temperature=0.5, top_k=3, seed=1), adapters=name)
        llm.generate(prompts_of(held, [5, 7], 1), SamplingParams(max_new_tokens=4), adapters=[name, None])
    assert len(llm.engine.graphs._graphs) == 8


def test_graphs_of_prompts_with_adapters_are_captured_ahead(held):
    prompt = prompts_of(held, [200], 2)
    plain_engine = engine(held, "bfloat16", step_graphs=False)
    llm = engine(held, "bfloat16")
    shapes = llm.engine.step_fn.graphs
    n = llm.engine.capture_graphs(("greedy",), prompt_tokens=300)
    captured = shapes.captures
    assert n > captured > 0
    for name in ("a", None, "c"):
        before = shapes.replayed_launches
        tokens = llm.generate(prompt, SamplingParams(max_new_tokens=4), adapters=name)[0]
        assert shapes.replayed_launches > before and shapes.captures == captured
        margins(held, prompt[0], tokens, name, "bfloat16")
        margins(held, prompt[0], plain_engine.generate(prompt, SamplingParams(max_new_tokens=4), adapters=name)[0], name, "bfloat16")
