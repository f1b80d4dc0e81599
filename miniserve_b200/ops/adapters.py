"""Low-rank adapters of many requests at once beside the projections that all requests share (``csrc/adapters.cu``): the matrices of one projection's
adapters (``LowRank``), which adapter each of a step's tokens has (``AdapterRows``), and the adapted products that ``ops.linear``,
``ops.linear_silu_mul`` and ``ops.qkv_norm_rope_kv`` hand over to when they are given both."""

from __future__ import annotations

import ctypes
from contextlib import nullcontext
from ctypes import c_char_p, c_int, c_ulonglong, c_void_p
from dataclasses import dataclass
from functools import lru_cache

import torch

from . import build, native

_p, _i = c_void_p, c_int
MAX_PARTS, MAX_RANK, TILE = 4, 256, 256  # TILE: tokens of a row tile of the plan
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
    [tokens], the request of each token, tokens in the order of the requests. Made once per step and used by all its layers: steps of many tokens have a plan, which the
    first product of a stream (or of a capture) makes of what the tensors hold then. A slot that the adapters do not have raises the status word, and the
    token counts as one without an adapter."""

    def __init__(self, slot_of_row: torch.Tensor, row_of_token: torch.Tensor):
        for t in (slot_of_row, row_of_token):
            if t.dtype is not torch.int32 or t.dim() != 1 or not t.is_contiguous():
                raise ValueError("slots and rows are contiguous int32 tensors of one dimension")
        if slot_of_row.device != row_of_token.device:
            raise ValueError("slots and rows lie on one device")
        self.slot_of_row, self.row_of_token = slot_of_row, row_of_token
        self.rows, self.tokens, self.index = slot_of_row.shape[0], row_of_token.shape[0], slot_of_row.get_device()
        self._plans: dict = {}

    def plan(self, slots: int, stream: int) -> "_Plan":
        """The adapters of each row tile, for projections with ``slots`` of them."""
        key = (slots, stream, _lib().ms_adapter_capture_id(stream))
        held = self._plans.get(key)
        if held is None:
            held = self._plans[key] = _Plan(self, slots, stream)
        return held


class _Adapters(ctypes.Structure):
    """``Adapters`` of csrc/adapters.cuh."""

    _fields_ = [(n, _p) for n in ("a", "b", "scale", "slot_of_row", "row_of_token", "status")] + [("slots", _i), ("rank", _i), ("parts", _i), ("ends", _i * MAX_PARTS)]


class _Product(ctypes.Structure):
    """``AdaptedProduct`` of csrc/adapters.cuh."""

    _fields_ = [("ad", _Adapters), ("v", _p), ("tile_first", _p), ("block_slot", _p), ("max_blocks", _i)]


class _Plan:
    def __init__(self, rows: AdapterRows, slots: int, stream: int):
        from . import device_status

        device, t = rows.slot_of_row.device, rows.tokens
        tiles = -(-t // TILE)
        # a request of several tiles has a block in each, and each request behind the first may add one to a tile that it shares
        self.max_blocks = max(1, min(tiles * min(slots, TILE), tiles + rows.rows - 1))
        with on_stream(stream, device):
            self.ints = torch.empty(tiles + 1 + 2 * self.max_blocks + t, dtype=torch.int32, device=device)
        at = self.ints.data_ptr()
        self.tile_first, self.block_slot = at, at + 4 * (tiles + 1)
        self.block_tile = self.block_slot + 4 * self.max_blocks
        self.token_slot = self.block_tile + 4 * self.max_blocks
        ad = _Adapters(None, None, None, rows.slot_of_row.data_ptr(), rows.row_of_token.data_ptr(), device_status(device).data_ptr(), slots, 0, 0)
        _check(_lib().ms_adapter_plan(self.tile_first, self.block_slot, self.block_tile, self.token_slot, ctypes.addressof(ad), t, self.max_blocks, stream))


@lru_cache(maxsize=None)
def _lib():
    lib = ctypes.CDLL(str(build.ensure_built(ADAPTERS)))
    native._declare(lib, "ms_adapters_last_error", [], c_char_p)
    native._declare(lib, "ms_adapters_set_pdl", [_i], None)
    native._declare(lib, "ms_adapter_capture_id", [_p], c_ulonglong)
    native._declare(lib, "ms_adapter_plan", [_p] * 5 + [_i, _i, _p])
    native._declare(lib, "ms_adapter_shrink", [_p, _p, _p, _i, _i, _i, _i, _p])
    native._declare(lib, "ms_adapter_shrink_blocks", [_p] * 7 + [_i] * 5 + [_p])
    native._declare(lib, "ms_adapter_expand", [_p] * 4 + [_i] * 6 + [_p])
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


FEW_TOKENS = 48  # up to so many, v is made token by token


def _v(x: torch.Tensor, low_rank: LowRank, rows: AdapterRows, ad: _Adapters, stream: int) -> torch.Tensor:
    """What the adapters' A make of x, float32 [T, parts * rank]."""
    t, k = x.shape
    with on_stream(stream, x.device):
        v = torch.empty((t, low_rank.parts * low_rank.rank), dtype=torch.float32, device=x.device)
    if x.dtype is torch.float32 or t <= FEW_TOKENS:
        _check(_lib().ms_adapter_shrink(v.data_ptr(), x.data_ptr(), ctypes.addressof(ad), t, low_rank.outputs, k, _code(x.dtype), stream))
    else:
        plan = rows.plan(low_rank.slots, stream)
        _check(_lib().ms_adapter_shrink_blocks(v.data_ptr(), x.data_ptr(), ctypes.addressof(ad), plan.tile_first, plan.block_slot, plan.block_tile, plan.token_slot, t,
                                               low_rank.outputs, k, plan.max_blocks, 1, stream))
    return v


def product(x: torch.Tensor, low_rank: LowRank, rows: AdapterRows, stream: int) -> tuple:
    """What a product on the 2-CTA tcgen05 kernel takes of the adapters, and the V it points to."""
    t, k = x.shape
    ad, plan = _struct(low_rank, rows), rows.plan(low_rank.slots, stream)
    with on_stream(stream, x.device):
        v = torch.empty((plan.max_blocks * TILE, low_rank.parts * low_rank.rank), dtype=torch.bfloat16, device=x.device)
    _check(_lib().ms_adapter_shrink_blocks(v.data_ptr(), x.data_ptr(), ctypes.addressof(ad), plan.tile_first, plan.block_slot, plan.block_tile, plan.token_slot, t,
                                           low_rank.outputs, k, plan.max_blocks, 0, stream))
    return _Product(ad, v.data_ptr(), plan.tile_first, plan.block_slot, plan.max_blocks), v


def _in_its_sums(x, weight, out, epilogue: str) -> bool:
    """Whether the product runs on the 2-CTA tcgen05 kernel, which takes the adapters in its own sums."""
    from . import tc_gemm_ok

    return x.dtype is torch.bfloat16 and out.dtype is torch.bfloat16 and x.shape[0] > FEW_TOKENS and tc_gemm_ok(x, weight, out, epilogue)


def _run(x, weight, out, stream: int, low_rank: LowRank, rows: AdapterRows, gated: bool) -> None:
    from . import TC_EPILOGUE, device_status
    from . import linear as shared

    t, k = x.shape
    epilogue = "silu_mul" if gated else "bf16"
    if _in_its_sums(x, weight, out, epilogue):
        held, v = product(x, low_rank, rows, stream)
        lib = native.gemm_tc()
        native.kernel_check(lib.ms_gemm_tc_adapted_bf16(out.data_ptr(), x.data_ptr(), weight.data_ptr(), t, out.shape[1], k, TC_EPILOGUE[epilogue], ctypes.addressof(held),
                                                        device_status(x.device).data_ptr(), stream), lib=lib, errfn="ms_gemm_tc_last_error")
        return
    # the shared product in float32, so that the sum is rounded once
    ad = _struct(low_rank, rows)
    if out.dtype is torch.float32 and not gated:
        y = out
    else:
        with on_stream(stream, x.device):
            y = torch.empty((t, low_rank.outputs), dtype=torch.float32, device=x.device)
    shared(x, weight, out=y, stream=stream)
    v = _v(x, low_rank, rows, ad, stream)
    _check(_lib().ms_adapter_expand(out.data_ptr(), y.data_ptr(), v.data_ptr(), ctypes.addressof(ad), t, low_rank.outputs, k, _code(x.dtype), _code(out.dtype), int(gated), stream))


def _here(call, x, weight, out, stream, low_rank: LowRank, rows: AdapterRows) -> torch.Tensor:
    """The call on its tensors' device, and its stream (None: that device's current one)."""
    device = low_rank.a.device
    if stream is None:
        stream = torch.cuda.current_stream(device).cuda_stream
    if torch.cuda.current_device() == low_rank.index:
        return call(x, weight, out, stream, low_rank, rows)
    with torch.cuda.device(device):
        return call(x, weight, out, stream, low_rank, rows)


def linear(x, weight, out, stream, low_rank: LowRank, rows: AdapterRows) -> torch.Tensor:
    check(x, weight, out, low_rank, rows, False)
    return _here(_linear, x, weight, out, stream, low_rank, rows)


def linear_silu_mul(x, weight, out, stream, low_rank: LowRank, rows: AdapterRows) -> torch.Tensor:
    check(x, weight, out, low_rank, rows, True)
    return _here(_linear_silu_mul, x, weight, out, stream, low_rank, rows)


def _linear(x, weight, out, stream: int, low_rank: LowRank, rows: AdapterRows) -> torch.Tensor:
    if out is None:
        with on_stream(stream, x.device):
            out = torch.empty((x.shape[0], low_rank.outputs), dtype=x.dtype, device=x.device)
    if x.shape[0]:
        _run(x, weight, out, stream, low_rank, rows, False)
    return out


def _linear_silu_mul(x, weight, out, stream: int, low_rank: LowRank, rows: AdapterRows) -> torch.Tensor:
    if x.shape[0]:
        _run(x, weight, out, stream, low_rank, rows, True)
    return out
