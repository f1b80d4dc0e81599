"""Per-step sampling arguments and the call into the sampling kernels.

As in miniserve/engine/sampler.py:65-100: a step whose rows are all greedy takes the plain
argmax; otherwise every row gets (temperature, top_p, seed, counter) with counter = the index
of the token being sampled in its sequence, so that a request draws the same noise wherever it
sits in a batch and whether or not it was preempted and run again. Tokens stay on the device;
the engine copies them back once per step.

Rows with top_k or min_p (which the reference does not have) are drawn by ``ops.sample_filtered`` from one random
number each, a function of (seed, counter) too; the rows beside them are drawn as they would be without.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Sequence

import numpy as np
import torch

from .. import ops


def _mix32(x: np.ndarray) -> np.ndarray:
    """Two rounds of x = ((x >> 16) ^ x) * 0x45D9F3B, then (x >> 16) ^ x, of unsigned 32-bit numbers (held in 64 bits): Thomas Mueller's integer hash."""
    for _ in range(2):
        x = (((x >> 16) ^ x) * 0x45D9F3B) & 0xFFFFFFFF
    return (x >> 16) ^ x


def uniforms(seeds: Sequence[int], counters: Sequence[int]) -> np.ndarray:
    """A random number in [0, 1) for each (seed, counter): 53 bits hashed of them, float64."""
    seed, counter = (np.asarray(x, dtype=np.uint64) & np.uint64(0xFFFFFFFF) for x in (seeds, counters))
    key = _mix32(seed ^ _mix32(counter))
    high, low = _mix32((key + 0x9E3779B9) & 0xFFFFFFFF), _mix32((key + 0x3C6EF372) & 0xFFFFFFFF)
    return ((high << np.uint64(21)) | (low >> np.uint64(11))).astype(np.float64) * 2.0 ** -53


@dataclass(frozen=True)
class Settings:
    """A step's sampling settings as rows of host tensors. ``f32`` [5, rows]: temperature and top_p of the rows drawn with noise (0 and 1 of filtered ones),
    temperature, top_p and min_p of the filtered ones; ``i64`` [2, rows]: seeds and counters; ``top_k`` int32 and ``uniform`` float64 [rows] of the filtered
    ones (below 0: the row is not filtered). ``mode``: which kernels run: "greedy", "temperature", "top_p", "filtered" (greedy rows beside), or "temperature+filtered", "top_p+filtered"."""

    mode: str
    f32: torch.Tensor
    i64: torch.Tensor
    top_k: torch.Tensor
    uniform: torch.Tensor

    @property
    def filtered(self) -> bool:
        return self.mode.endswith("filtered")


def settings(temperatures, top_ps=None, seeds=None, counters=None, top_ks=None, min_ps=None, rows: int | None = None) -> Settings:
    """``rows``: pad with greedy rows up to so many."""
    n = len(temperatures)
    rows = n if rows is None else rows
    top_ps = list(top_ps) if top_ps is not None else [1.0] * n
    top_ks = list(top_ks) if top_ks is not None else [0] * n
    min_ps = list(min_ps) if min_ps is not None else [0.0] * n
    drawn = [t > 0 for t in temperatures]
    filtered = [d and (k > 0 or m > 0) for d, k, m in zip(drawn, top_ks, min_ps)]
    noise = [d and not f for d, f in zip(drawn, filtered)]
    f32 = np.zeros((5, rows), dtype=np.float32)
    f32[1] = f32[3] = 1.0
    f32[0, :n] = np.where(noise, temperatures, 0.0)
    f32[1, :n] = np.where(filtered, 1.0, top_ps)
    f32[2, :n] = np.where(filtered, temperatures, 0.0)
    f32[3, :n] = top_ps
    f32[4, :n] = min_ps
    i64 = np.zeros((2, rows), dtype=np.int64)
    top_k, uniform = np.zeros(rows, dtype=np.int32), np.zeros(rows, dtype=np.float64)
    top_k[:n] = top_ks
    if seeds is not None:
        i64[0, :n], i64[1, :n] = seeds, counters
    if any(filtered):
        uniform[:n] = np.where(filtered, uniforms(seeds, counters), 0.0)
    mode = "greedy" if not any(noise) else "top_p" if any(p < 1 for f, p in zip(filtered, top_ps) if not f) else "temperature"
    if any(filtered):
        if any(noise):
            uniform[:n] = np.where(noise, -1.0, uniform[:n])  # those keep the token that the noise drew; greedy rows are greedy either way
            mode += "+filtered"
        else:
            mode = "filtered"
    return Settings(mode, torch.from_numpy(f32), torch.from_numpy(i64), torch.from_numpy(top_k), torch.from_numpy(uniform))


def draw(tokens: torch.Tensor, logits: torch.Tensor, mode: str, f32, i64, top_k, uniform, scratch, stream) -> None:
    """The sampling kernels of a mode, over settings on the device."""
    if mode == "greedy":
        ops.sample(tokens, logits, stream=stream)
        return
    if mode != "filtered":
        nucleus = mode.startswith("top_p")
        ops.sample(tokens, logits, temperature=f32[0], top_p=f32[1] if nucleus else None, seed=i64[0], counter=i64[1], scratch=scratch if nucleus else None, stream=stream)
    if mode.endswith("filtered"):
        ops.sample_filtered(tokens, logits, f32[2], uniform, top_k=top_k, top_p=f32[3], min_p=f32[4], stream=stream)


class Sampler:
    def __init__(self, device: torch.device | str, vocab_size: int, max_rows: int = 64):
        self.device = torch.device(device)
        self.vocab_size = vocab_size
        self._scratch = None
        self._cap = 0
        self._ensure(max_rows)

    def _ensure(self, rows: int) -> None:
        if rows <= self._cap:
            return
        self._cap = max(rows, 2 * self._cap)
        self._scratch = torch.empty(self._cap * ops.nucleus_bytes(), dtype=torch.uint8, device=self.device)

    def sample(self, logits: torch.Tensor, temperatures: Sequence[float] | None = None,
               top_ps: Sequence[float] | None = None, seeds: Sequence[int] | None = None,
               counters: Sequence[int] | None = None, stream=None, top_ks: Sequence[int] | None = None, min_ps: Sequence[float] | None = None) -> torch.Tensor:
        """``logits`` float32 [rows, vocab] -> int32 [rows] on the device."""
        rows = logits.shape[0]
        tokens = torch.empty(rows, dtype=torch.int32, device=self.device)
        if rows == 0:
            return tokens
        if temperatures is None or all(t == 0 for t in temperatures):
            ops.sample(tokens, logits, stream=stream)
            return tokens
        self._ensure(rows)
        s = settings(temperatures, top_ps, seeds, counters, top_ks, min_ps)
        f32, i64 = (x.pin_memory().to(self.device, non_blocking=True) for x in (s.f32, s.i64))
        top_k, uniform = (x.pin_memory().to(self.device, non_blocking=True) for x in (s.top_k, s.uniform)) if s.filtered else (None, None)
        draw(tokens, logits, s.mode, f32, i64, top_k, uniform, self._scratch, stream)
        return tokens
