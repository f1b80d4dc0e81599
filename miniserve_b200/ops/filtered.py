"""Sampling with temperature, top-k, top-p and min-p from given random numbers (``csrc/sample_filtered.cu``)."""

from __future__ import annotations

import ctypes
from ctypes import c_char_p, c_int, c_void_p
from functools import lru_cache

import torch

from . import build, native

_p, _i = c_void_p, c_int
FILTERS = build.Module("filters", ("sample_filtered.cu",))
MAX_VOCAB = 1 << 20


@lru_cache(maxsize=None)
def _lib():
    lib = ctypes.CDLL(str(build.ensure_built(FILTERS)))
    native._declare(lib, "ms_filters_last_error", [], c_char_p)
    native._declare(lib, "ms_filters_set_pdl", [_i], None)
    native._declare(lib, "ms_sample_filtered", [_p] * 7 + [_i] * 3 + [_p])
    lib.ms_filters_set_pdl(int(native.pdl_enabled()))
    return lib


def sample_filtered(tokens: torch.Tensor, logits: torch.Tensor, temperature: torch.Tensor, uniform: torch.Tensor, top_k: torch.Tensor | None = None,
                    top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None, stream=None) -> None:
    """tokens[r] (int32) from float32 logits [rows, vocab] and a random number ``uniform[r]`` in [0, 1) (float32 or float64), by settings of each row:
    ``temperature`` (float32; 0: the first of the likeliest tokens), ``top_k`` (int32: the k likeliest; 0 or less: all), ``top_p`` (float32: of those the
    likeliest whose mass before them is below top_p of theirs; 1 or more: all), ``min_p`` (float32: of those the ones at least min_p times as likely as the likeliest; 0: all).
    Tokens of one probability are ranked in the order of the vocabulary. What is drawn is the first token of the rest, in that order, up to which there is more than
    ``uniform[r]`` of its mass. Masses are added up exactly, so a row's token depends on nothing but the row. NaN counts as -inf, which is never drawn (a row
    of nothing else gives 0). A row whose random number is not in [0, 1) keeps the token it had."""
    rows, vocab = logits.shape
    dev = logits.get_device()
    if dev < 0 or logits.dtype is not torch.float32 or not logits.is_contiguous():
        raise ValueError(f"logits are a contiguous float32 CUDA tensor, not {logits.dtype} on {logits.device}")
    if not 1 <= vocab <= MAX_VOCAB:
        raise ValueError(f"a vocabulary of 1 to {MAX_VOCAB} tokens, not {vocab}")
    wide = uniform.dtype is torch.float64
    ptr = [_row("tokens", tokens, torch.int32, rows, dev), logits.data_ptr(), _row("temperature", temperature, torch.float32, rows, dev),
           _row("uniform", uniform, torch.float64 if wide else torch.float32, rows, dev), None if top_k is None else _row("top_k", top_k, torch.int32, rows, dev),
           None if top_p is None else _row("top_p", top_p, torch.float32, rows, dev), None if min_p is None else _row("min_p", min_p, torch.float32, rows, dev)]
    if not rows:
        return
    if torch.cuda.current_device() != dev:
        with torch.cuda.device(dev):
            return sample_filtered(tokens, logits, temperature, uniform, top_k, top_p, min_p, stream)
    rc = _lib().ms_sample_filtered(*ptr, rows, vocab, int(wide), torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream)
    native.kernel_check(rc, lib=_lib() if rc else None, errfn="ms_filters_last_error")


def _row(name: str, t: torch.Tensor, dtype: torch.dtype, rows: int, dev: int) -> int:
    """The address of a number per row."""
    if t.dtype is not dtype or t.dim() != 1 or t.shape[0] < rows or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{name} is a contiguous {dtype} tensor of {rows} rows on the logits' device, not {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()
