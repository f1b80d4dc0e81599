"""Sampling parameters that are not numbers of tokens."""

from __future__ import annotations

import pytest

from miniserve_b200.engine import SamplingParams


@pytest.mark.parametrize("top_k", [float("inf"), float("-inf"), float("nan"), 1e30, -0.5])
def test_top_k_is_a_number_of_tokens(top_k):
    with pytest.raises(ValueError, match="top_k"):
        SamplingParams(4, temperature=1.0, top_k=top_k)
    assert SamplingParams(4, temperature=1.0, top_k=3.0).is_filtered
