"""Kernels whose CTAs write to each other's shared memory: such memory may be touched once its CTA is known to have started, so a barrier of the cluster stands ahead of the first access."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "miniserve_b200" / "csrc"
BARRIER = re.compile(r"cluster_started_wait\(\)|\b(?:cluster|group)\.sync\(\)|cluster_sync_all\(\)")


def body(name: str, kernel: str) -> str:
    """The kernel's source between its outer braces, without comments."""
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    at = text.index("{", re.search(kernel + r"\s*\(", text).end())
    depth, i = 0, at
    while True:
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        i += 1
        if depth == 0:
            return text[at:i]


# (file, kernel, what reaches another CTA's memory)
@pytest.mark.parametrize("name,kernel,reach", [("sample_filtered.cu", "sample_filtered_kernel", r"cl\.reduce<|cl\.tell\(|map_shared_rank\("),
                                               ("sampling.cu", "sample_cluster_kernel", r"nc_all_reduce<|map_shared_rank\("),
                                               ("gated_recurrence.cu", "rglru_scan_kernel", r"map_shared_rank\("), ("gemm_tc.cu", "gemm_tc_pair_kernel", r"mbar_arrive_first_cta\("),
                                               ("gemm_tc.cu", "gemm_tc_decode_kernel", r"mapa|shared::cluster\.f32"), ("gemm_tc.cu", "adapter_v_kernel", r"mapa|ld\.shared::cluster")])
def test_a_barrier_stands_ahead_of_the_first_access(name, kernel, reach):
    text = body(name, kernel)
    first = re.search(reach, text)
    assert first is not None
    barrier = BARRIER.search(text)
    assert barrier is not None and barrier.start() < first.start(), f"{kernel}: {first.group(0)} ahead of any barrier of the cluster"
    arrive = text.find("cluster_started_arrive()")
    if barrier.group(0).startswith("cluster_started"):
        assert 0 <= arrive < barrier.start() and text.count("cluster_started_arrive()") == 1
