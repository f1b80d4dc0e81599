"""Low-rank adapters of many requests at once beside the projections that all requests share (``csrc/adapters.cu``): the matrices of one projection's
adapters (``LowRank``), which adapter each of a step's tokens has (``AdapterRows``), and the adapted products that ``ops.linear``,
``ops.linear_silu_mul`` and ``ops.qkv_norm_rope_kv`` hand over to when they are given both."""

from __future__ import annotations

import ctypes
from contextlib import nullcontext
from ctypes import c_char_p, c_int, c_void_p
from dataclasses import dataclass
from functools import lru_cache

import torch

from . import build, native

_p, _i = c_void_p, c_int
MAX_PARTS, MAX_RANK = 4, 256
ADAPTERS = build.Module("adapters", ("adapters.cu",))
_TYPES = (torch.bfloat16, torch.float32)


@dataclass(frozen=True, eq=False)
class LowRank:
    """The adapters of one projection, W [N, K]: slot s adds ``scale[s]`` B_s A_s x to W x. ``a`` [slots, parts * rank, K] and ``b`` [slots, N, rank] in the
    weight's type, ``scale`` float32 [slots]. A stacked projection (q|k|v, gate|up) has ``parts``: ``ends[p]`` is the first of W's rows behind part p (the
    last is N), a's rows [p * rank, (p + 1) * rank) and part p's rows of b belong together. An adapter of a smaller rank fills its place up with zeros."""

    a: torch.Tensor
    b: torch.Tensor
    scale: torch.Tensor
    ends: tuple[int, ...]

    def __post_init__(self):
        a, b, c = self.a, self.b, self.scale
        ends = tuple(int(e) for e in self.ends)
        if a.dtype not in _TYPES or b.dtype is not a.dtype or c.dtype is not torch.float32:
            raise TypeError(f"adapters are bfloat16 or float32, all of a projection's of one type, scales float32, not {a.dtype}, {b.dtype} and {c.dtype}")
        if a.dim() != 3 or b.dim() != 3 or c.dim() != 1 or not 1 <= len(ends) <= MAX_PARTS or b.shape[0] != a.shape[0] or c.shape[0] != a.shape[0]:
            raise ValueError(f"adapters are a [slots, parts * rank, K], b [slots, N, rank] and scale [slots] with up to {MAX_PARTS} parts, not {tuple(a.shape)}, "
                             f"{tuple(b.shape)}, {tuple(c.shape)} and {len(ends)}")
        slots, n, rank = b.shape
        if slots < 1 or a.shape[1] != len(ends) * rank or rank % 8 or not 8 <= rank <= MAX_RANK or a.shape[2] < 8 or a.shape[2] % 8:
            raise ValueError(f"adapters have a rank that is a multiple of 8 up to {MAX_RANK} (filled up with zeros) and inputs that are a multiple of 8, not a "
                             f"{tuple(a.shape)} and b {tuple(b.shape)} in {len(ends)} parts")
        if any(e <= at for at, e in zip((0,) + ends, ends)) or ends[-1] != n:
            raise ValueError(f"the parts of {n} outputs end at {ends}")
        if not (a.device == b.device == c.device) or any(not t.is_contiguous() for t in (a, b, c)) or a.data_ptr() % 16 or b.data_ptr() % 16:
            raise ValueError("an adapter's tensors lie on one device, contiguous, the matrices on 16 bytes")
        for name, value in (("ends", ends), ("slots", slots), ("rank", rank), ("parts", len(ends)), ("outputs", n), ("inputs", a.shape[2]), ("index", a.get_device())):
            object.__setattr__(self, name, value)

    @classmethod
    def zeros(cls, slots: int, inputs: int, ends: tuple[int, ...], rank: int, dtype: torch.dtype, device="cuda") -> "LowRank":
        """Adapters that add nothing, to be filled in (``scale`` too)."""
        return cls(torch.zeros((slots, len(ends) * rank, inputs), dtype=dtype, device=device), torch.zeros((slots, ends[-1], rank), dtype=dtype, device=device),
                   torch.zeros((slots,), dtype=torch.float32, device=device), tuple(ends))


class AdapterRows:
    """Which adapter each token of a step has: ``slot_of_row`` int32 [rows], the slot of each request (below 0: none), and ``row_of_token`` int32
    [tokens], the request of each token, tokens in the order of the requests. Made once per step and used by all its layers, on one stream. A slot that the
    adapters do not have raises the status word, and the token counts as one without an adapter."""

    def __init__(self, slot_of_row: torch.Tensor, row_of_token: torch.Tensor):
        for t in (slot_of_row, row_of_token):
            if t.dtype is not torch.int32 or t.dim() != 1 or not t.is_contiguous():
                raise ValueError("slots and rows are contiguous int32 tensors of one dimension")
        if slot_of_row.device != row_of_token.device:
            raise ValueError("slots and rows lie on one device")
        self.slot_of_row, self.row_of_token = slot_of_row, row_of_token
        self.rows, self.tokens, self.index = slot_of_row.shape[0], row_of_token.shape[0], slot_of_row.get_device()


class _Adapters(ctypes.Structure):
    """``Adapters`` of csrc/adapters.cu."""

    _fields_ = [(n, _p) for n in ("a", "b", "scale", "slot_of_row", "row_of_token", "status")] + [("slots", _i), ("rank", _i), ("parts", _i), ("ends", _i * MAX_PARTS)]


@lru_cache(maxsize=None)
def _lib():
    lib = ctypes.CDLL(str(build.ensure_built(ADAPTERS)))
    native._declare(lib, "ms_adapters_last_error", [], c_char_p)
    native._declare(lib, "ms_adapters_set_pdl", [_i], None)
    native._declare(lib, "ms_adapter_shrink", [_p, _p, _p, _i, _i, _i, _i, _p])
    native._declare(lib, "ms_adapter_expand", [_p, _p, _p, _i, _i, _i, _i, _i, _p])
    lib.ms_adapters_set_pdl(int(native.pdl_enabled()))
    return lib


def _check(rc: int) -> None:
    native.kernel_check(rc, lib=_lib() if rc else None, errfn="ms_adapters_last_error")


def on_stream(stream: int, device: torch.device):
    """Allocations in the order of ``stream`` (a handle), where that is not the current one."""
    if stream == torch.cuda.current_stream(device).cuda_stream:
        return nullcontext()
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device))


def check(x: torch.Tensor, weight: torch.Tensor, out: torch.Tensor | None, low_rank: LowRank, rows: AdapterRows, gated: bool) -> None:
    if not isinstance(low_rank, LowRank) or not isinstance(rows, AdapterRows):
        raise TypeError("an adapted product takes low_rank (ops.LowRank) and adapter_rows (ops.AdapterRows), both")
    if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != low_rank.inputs or tuple(weight.shape) != (low_rank.outputs, low_rank.inputs):
        raise ValueError(f"x is {tuple(x.shape)}, the weight {tuple(weight.shape)}, its adapters take {low_rank.inputs} and give {low_rank.outputs}")
    if x.shape[0] != rows.tokens:
        raise ValueError(f"x has {x.shape[0]} tokens, adapter_rows {rows.tokens}")
    if x.dtype is not low_rank.a.dtype or weight.dtype is not x.dtype:
        raise TypeError(f"x, the weight and its adapters are of one type, not {x.dtype}, {weight.dtype} and {low_rank.a.dtype}")
    if not (x.get_device() == weight.get_device() == low_rank.index == rows.index >= 0) or not x.is_contiguous() or not weight.is_contiguous() or x.data_ptr() % 16:
        raise ValueError("kernel operands must be contiguous CUDA tensors on one device, x on 16 bytes")
    out_columns = low_rank.outputs // 2 if gated else low_rank.outputs
    if gated and (low_rank.outputs % 2 or out.dtype is not x.dtype):
        raise ValueError(f"a gate|up projection of {low_rank.outputs} rows, out {out.dtype} for x {x.dtype}")
    if out is not None and (tuple(out.shape) != (x.shape[0], out_columns) or out.get_device() != low_rank.index or not out.is_contiguous()
                            or out.dtype not in ((torch.float32,) if x.dtype is torch.float32 else _TYPES)):
        raise ValueError(f"out is {out.dtype} {tuple(out.shape)}, not a contiguous [{x.shape[0]}, {out_columns}]")


def _struct(low_rank: LowRank, rows: AdapterRows) -> _Adapters:
    from . import device_status

    return _Adapters(low_rank.a.data_ptr(), low_rank.b.data_ptr(), low_rank.scale.data_ptr(), rows.slot_of_row.data_ptr(), rows.row_of_token.data_ptr(),
                     device_status(low_rank.a.device).data_ptr(), low_rank.slots, low_rank.rank, low_rank.parts,
                     (_i * MAX_PARTS)(*low_rank.ends, *[low_rank.outputs] * (MAX_PARTS - low_rank.parts)))


def _code(dtype: torch.dtype) -> int:
    return 0 if dtype is torch.float32 else 1


def add(y: torch.Tensor, x: torch.Tensor, low_rank: LowRank, rows: AdapterRows, stream: int) -> None:
    """y [T, N] += what the tokens' adapters make of x."""
    t, k = x.shape
    ad = _struct(low_rank, rows)
    with on_stream(stream, x.device):
        v = torch.empty((t, low_rank.parts * low_rank.rank), dtype=torch.float32, device=x.device)
    _check(_lib().ms_adapter_shrink(v.data_ptr(), x.data_ptr(), ctypes.addressof(ad), t, low_rank.outputs, k, _code(x.dtype), stream))
    _check(_lib().ms_adapter_expand(y.data_ptr(), v.data_ptr(), ctypes.addressof(ad), t, low_rank.outputs, k, _code(x.dtype), _code(y.dtype), stream))


def linear(x, weight, out, stream: int, low_rank: LowRank, rows: AdapterRows) -> torch.Tensor:
    from . import linear as shared

    check(x, weight, out, low_rank, rows, False)
    out = shared(x, weight, out=out, stream=stream)
    if x.shape[0]:
        add(out, x, low_rank, rows, stream)
    return out


def linear_silu_mul(x, weight, out, scratch, stream: int, low_rank: LowRank, rows: AdapterRows) -> torch.Tensor:
    from . import silu_mul

    check(x, weight, out, low_rank, rows, True)
    if not x.shape[0]:
        return out
    if scratch is None:
        with on_stream(stream, x.device):
            scratch = torch.empty((x.shape[0], low_rank.outputs), dtype=x.dtype, device=x.device)
    gate_up = linear(x, weight, scratch, stream, low_rank, rows)
    silu_mul(out, gate_up, stream=stream)
    return out
