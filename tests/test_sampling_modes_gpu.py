"""Graphs of decode steps are captured ahead for every way of sampling that a batch may need."""

from __future__ import annotations

import pytest

from miniserve_b200.engine import LLM, SamplingParams

pytestmark = pytest.mark.gpu

FILTERED = dict(temperature=0.8, top_k=5)
BATCHES = {"temperature+filtered": (dict(temperature=0.9), FILTERED, dict()), "top_p+filtered": (dict(temperature=0.9, top_p=0.6), FILTERED, dict(temperature=1.1)), "filtered": (FILTERED, dict())}


def params(kinds):
    return [SamplingParams(max_new_tokens=5, seed=i, **kw) for i, kw in enumerate(kinds)]


@pytest.mark.parametrize("mode", sorted(BATCHES))
def test_a_batch_meets_the_graphs_that_were_captured_for_it(mode):
    llm = LLM(random="tiny-b", kv_pool_tokens=1024, page_size=16, max_running=4)
    kinds = BATCHES[mode]
    prompts = [[1 + i, 2, 3] for i in range(len(kinds))]
    n = llm.engine.capture_graphs((mode,))
    buckets = [b for b in llm.engine.graphs.buckets if b > 1 or mode == "filtered"]
    assert n == len(llm.engine.graphs._graphs) == len(buckets) and {k[1] for k in llm.engine.graphs._graphs} == {mode}
    got = llm.generate(prompts, params(kinds))
    assert len(llm.engine.graphs._graphs) == n
    eager = LLM(random="tiny-b", kv_pool_tokens=1024, page_size=16, max_running=4, cuda_graph=False)
    assert [len(o) for o in got] == [len(o) for o in eager.generate(prompts, params(kinds))] == [5] * len(kinds)


def test_a_mode_that_there_is_not_is_refused():
    llm = LLM(random="tiny-b", kv_pool_tokens=1024, page_size=16, max_running=2)
    for modes in (("nucleus",), ("greedy", "filtered+top_p")):
        with pytest.raises(ValueError, match="no sampling modes"):
            llm.engine.capture_graphs(modes)
    assert not llm.engine.graphs._graphs
