"""Counters that launches have to themselves, taken by two host threads, without a GPU."""

from __future__ import annotations

import threading
import time
from types import SimpleNamespace

import torch

from miniserve_b200 import ops


class Slow(list):
    """A list during whose writes other threads run."""

    def __setitem__(self, at, value):
        time.sleep(0.001)
        super().__setitem__(at, value)


def test_no_two_launches_have_the_same_counters(monkeypatch):
    monkeypatch.setattr(ops.adapters, "_lib", lambda: SimpleNamespace(ms_adapter_capture_id=lambda stream: 0))
    i = torch.zeros(3, dtype=torch.int32)
    rows = ops.AdapterRows(i, i.clone())
    rows._tickets[7, 0] = Slow([None, 1000, 1000 + 8 * 200])
    taken = []
    threads = [threading.Thread(target=lambda: taken.extend([rows.tickets(7) for _ in range(50)])) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sorted(taken) == [1000 + 8 * n for n in range(150)]
