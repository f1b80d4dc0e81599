"""Low-rank adapters of many requests at once beside the projections that all requests share (``csrc/adapters.cu``): the matrices of one projection's
adapters (``LowRank``), which adapter each of a step's tokens has (``AdapterRows``), and the adapted products that ``ops.linear``,
``ops.linear_silu_mul`` and ``ops.qkv_norm_rope_kv`` hand over to when they are given both."""

from __future__ import annotations

import ctypes
import struct
import sys
import threading
from contextlib import nullcontext
from ctypes import c_char_p, c_int, c_longlong, c_ulonglong, c_void_p
from dataclasses import dataclass
from functools import lru_cache

import torch

from . import build, native

_p, _i = c_void_p, c_int
MAX_PARTS, MAX_RANK, TILE = 4, 256, 256  # TILE: tokens of a row tile of the plan
TICKETS = 256  # pairs of counters that a step makes at a time
BLOCK_BYTES = 48  # of an ``AdapterBlock`` (csrc/adapters.cuh)
ADAPTERS = build.Module("adapters", ("adapters.cu",))
_TYPES = (torch.bfloat16, torch.float32)
_Q = struct.Struct("Q").pack


def _ops():
    """The package that imports this module."""
    return sys.modules[__package__]


@dataclass(frozen=True, eq=False)
class LowRank:
    """The adapters of one projection, W [N, K]: slot s adds ``scale[s]`` B_s A_s x to W x. ``a`` [slots, parts * rank, K] and ``b`` [slots, N, rank] in the
    weight's type, ``scale`` float32 [slots]. A stacked projection (q|k|v, gate|up) has ``parts``: ``ends[p]`` is the first of W's rows behind part p (the
    last is N), a's rows [p * rank, (p + 1) * rank) and part p's rows of b belong together. An adapter of a smaller rank fills its place up with zeros.
    All are finite: in a step of many tokens other requests' tokens meet an adapter with zeros for v."""

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
        # what every call asks for: sizes, the device's index (-1: the host), the two ends of the kernels' ``Adapters``
        for name, value in (("ends", ends), ("slots", slots), ("rank", rank), ("parts", len(ends)), ("outputs", n), ("inputs", a.shape[2]), ("index", a.get_device()),
                            ("dtype", a.dtype), ("numbers", len(ends) * rank), ("weight_shape", (n, a.shape[2])), ("head", struct.pack("3Q", a.data_ptr(), b.data_ptr(), c.data_ptr())),
                            ("tail", struct.pack("7i4x", slots, rank, len(ends), *ends, *[n] * (MAX_PARTS - len(ends))))):
            object.__setattr__(self, name, value)

    @classmethod
    def zeros(cls, slots: int, inputs: int, ends: tuple[int, ...], rank: int, dtype: torch.dtype, device="cuda") -> "LowRank":
        """Adapters that add nothing, to be filled in (``scale`` too)."""
        return cls(torch.zeros((slots, len(ends) * rank, inputs), dtype=dtype, device=device), torch.zeros((slots, ends[-1], rank), dtype=dtype, device=device),
                   torch.zeros((slots,), dtype=torch.float32, device=device), tuple(ends))


class AdapterRows:
    """Which adapter each token of a step has: ``slot_of_row`` int32 [rows], the slot of each request (below 0: none), and ``row_of_token`` int32
    [tokens], the request of each token, tokens in the order of the requests. Made once per step and used by all its layers: products of many tokens work by a plan of the two,
    which is written once for each stream (or capture, whose replays write it again) and kept. Writing to the tensors in place makes it anew, as far as torch counts what is
    written (``Tensor._version``); behind writes that it does not count (a kernel of one's own, ``.data``, a replayed graph) call ``refresh``. Tensors of inference mode, whose
    writes nobody counts, have no plan that is kept. A slot that the adapters do not have, or a row that there is not, raises the status word, and the token counts as one
    without an adapter."""

    def __init__(self, slot_of_row: torch.Tensor, row_of_token: torch.Tensor):
        for t in (slot_of_row, row_of_token):
            if t.dtype is not torch.int32 or t.dim() != 1 or not t.is_contiguous():
                raise ValueError("slots and rows are contiguous int32 tensors of one dimension")
        if slot_of_row.device != row_of_token.device:
            raise ValueError("slots and rows lie on one device")
        self.slot_of_row, self.row_of_token = slot_of_row, row_of_token
        self.rows, self.tokens, self.index = slot_of_row.shape[0], row_of_token.shape[0], slot_of_row.get_device()
        self._plans: dict = {}  # (slots, stream, capture) -> (what the tensors' versions were, the plan)
        self._tickets: dict = {}
        self._taking = threading.Lock()
        if self.index >= 0:
            self.status = _ops().device_status(slot_of_row.device).data_ptr()
            self.middle = struct.pack("3Q2i", slot_of_row.data_ptr(), row_of_token.data_ptr(), self.status, self.rows, 0)
            self.sms = _ops()._sm_count(slot_of_row.device)

    def plan(self, slots: int, stream: int) -> "_Plan":
        """The adapters of each row tile, for projections with ``slots`` of them, of what the tensors hold now."""
        key, version = (slots, stream, _lib().ms_adapter_capture_id(stream)), self._version()
        held = self._plans.get(key)
        if held is None or held[0] != version or version is None:
            held = self._plans[key] = (version, _Plan(self, slots, stream))
        return held[1]

    def _version(self) -> tuple | None:
        """How often torch has seen the tensors written (None: it does not count)."""
        if self.slot_of_row.is_inference() or self.row_of_token.is_inference():
            return None
        return self.slot_of_row._version, self.row_of_token._version

    def refresh(self) -> None:
        """Forget the plans: the tensors were written in a way that torch does not count."""
        self._plans.clear()

    def tickets(self, stream: int) -> int:
        """The address of two zeros on the device that no launch has had: a launch leaves its counts in them."""
        key = (stream, _lib().ms_adapter_capture_id(stream))
        with self._taking:  # (two host threads: a pair is one launch's)
            held = self._tickets.get(key)
            if held is None or held[1] == held[2]:
                with on_stream(stream, self.slot_of_row.device):
                    zeros = torch.zeros(2 * TICKETS, dtype=torch.int32, device=self.slot_of_row.device)
                held = self._tickets[key] = [zeros, zeros.data_ptr(), zeros.data_ptr() + 8 * TICKETS]
            held[1] += 8
            return held[1] - 8


class _Plan:
    def __init__(self, rows: AdapterRows, slots: int, stream: int):
        device, t = rows.slot_of_row.device, rows.tokens
        tiles = -(-t // TILE)
        # a request of several tiles has a block in each, and each request behind the first may add one to a tile that it shares
        self.max_blocks = max(1, min(tiles * min(slots, TILE), tiles + rows.rows - 1))
        with on_stream(stream, device):
            self.ints = torch.empty(BLOCK_BYTES // 4 * self.max_blocks + tiles + 1, dtype=torch.int32, device=device)
        self.blocks = self.ints.data_ptr()
        self.tile_first = self.blocks + BLOCK_BYTES * self.max_blocks
        ad = bytes(24) + rows.middle + struct.pack("7i4x", slots, 0, 0, 0, 0, 0, 0)
        _check(_lib().ms_adapter_plan(self.tile_first, self.blocks, ad, t, self.max_blocks, stream))


@lru_cache(maxsize=None)
def _lib():
    lib = ctypes.CDLL(str(build.ensure_built(ADAPTERS)))
    native._declare(lib, "ms_adapters_last_error", [], c_char_p)
    native._declare(lib, "ms_adapters_set_pdl", [_i], None)
    native._declare(lib, "ms_adapter_capture_id", [_p], c_ulonglong)
    native._declare(lib, "ms_adapter_plan", [_p] * 2 + [c_char_p, _i, _i, _p])
    native._declare(lib, "ms_adapter_shrink", [_p, _p, c_char_p, _i, _i, _i, _i, _p, c_longlong, _p])
    native._declare(lib, "ms_adapter_expand", [_p, _p, _p, c_char_p] + [_i] * 6 + [_p])
    lib.ms_adapters_set_pdl(int(native.pdl_enabled()))
    return lib


def _check(rc: int) -> None:
    native.kernel_check(rc, lib=_lib() if rc else None, errfn="ms_adapters_last_error")


_now = torch._C._cuda_getCurrentRawStream  # the handle of a device's current stream (what torch.cuda.current_stream(index).cuda_stream is, in a tenth of its time)
_HERE = nullcontext()


def on_stream(stream: int, device: torch.device):
    """Allocations in the order of ``stream`` (a handle), where that is not the current one."""
    if stream == _now(device.index):
        return _HERE
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device))


def check(x: torch.Tensor, weight: torch.Tensor, out: torch.Tensor | None, low_rank: LowRank, rows: AdapterRows, gated: bool) -> None:
    if not isinstance(low_rank, LowRank) or not isinstance(rows, AdapterRows):
        raise TypeError("an adapted product takes low_rank (ops.LowRank) and adapter_rows (ops.AdapterRows), both")
    shape, dtype, index = x.shape, x.dtype, low_rank.index
    if len(shape) != 2 or shape[1] != low_rank.inputs or weight.shape != low_rank.weight_shape:
        raise ValueError(f"x is {tuple(shape)}, the weight {tuple(weight.shape)}, its adapters take {low_rank.inputs} and give {low_rank.outputs}")
    if shape[0] != rows.tokens:
        raise ValueError(f"x has {shape[0]} tokens, adapter_rows {rows.tokens}")
    if dtype is not low_rank.dtype or weight.dtype is not dtype:
        raise TypeError(f"x, the weight and its adapters are of one type, not {dtype}, {weight.dtype} and {low_rank.dtype}")
    if (not (x.get_device() == weight.get_device() == index == rows.index >= 0) or not x.is_contiguous() or not weight.is_contiguous() or x.data_ptr() % 16
            or weight.data_ptr() % 16):
        raise ValueError("kernel operands must be contiguous CUDA tensors on one device, x and the weight on 16 bytes")
    if gated and (low_rank.outputs % 2 or out.dtype is not dtype):
        raise ValueError(f"a gate|up projection of {low_rank.outputs} rows, out {out.dtype} for x {dtype}")
    if out is not None and (out.shape != (shape[0], low_rank.outputs // 2 if gated else low_rank.outputs) or out.get_device() != index or not out.is_contiguous()
                            or (out.dtype is not dtype and out.dtype is not torch.float32) or out.data_ptr() % 16):
        raise ValueError(f"out is {out.dtype} {tuple(out.shape)} for {shape[0]} tokens and {low_rank.outputs} outputs{' (gate and up)' if gated else ''}: a contiguous tensor on the "
                         "adapters' device, of x's type or float32, on 16 bytes")


def _code(dtype: torch.dtype) -> int:
    return 0 if dtype is torch.float32 else 1


WAY: str | None = None  # tests and measurements: "stream", "decode", "pair" or "apart" instead of the rules'
# Up to so many products (tokens x numbers x k) v is made token by token, beyond by a plan on the tensor cores. Token by token / by a plan, us, of one adapter and of 16: 64 tokens, 96
# numbers, k 4,096 7.6 / 8.4 and 7.6 / 15.8; 48 numbers, k 12,288 8.6 / 10.2 and 10.7 / 19.6; 96 numbers, k 12,288 14.2 / 11.9 and 17.8 / 27.8.
TOKEN_WISE = 48 << 20
# A weight of up to so many bytes is asked into L2 by the launch that makes v, while the kernels before it still run. A decode step of 0.6b with adapters, ms, without / with: 1 request 1.157 /
# 1.128, 8 on eight adapters 1.338 / 1.291; a product behind a short kernel loses 0.1 to 0.2 us. Beside larger weights it loses (12288 -> 4096 22.3 / 28.5 us: the product asks for them itself).
AHEAD = 16 << 20
FEW_TOKENS = 32  # up to so many (in some cases twice so many), the products are the decode steps' tcgen05 kernel
# That kernel makes v itself where the weight is at least OWN_WEIGHT MiB and the numbers (tokens x rank x parts) are few beside it (the square of the MiB over 128: 18 beside 48
# MiB, 288 beside 192): it then fetches the weights while the kernels before it still run, and v is ready before they have come; in a launch ahead v comes sooner where it is much. In a launch ahead / its own work, us, behind a norm, rank
# 16: 1 token of 4096 -> 6144 17.1 / 15.7, gated 2048 -> 2 x 6144 16.0 / 13.5, 4096 -> 2 x 12288 39.2 / 35.6 and 8 of eight adapters 41.2 / 38.1; but 8 of 12288 -> 4096 22.4 / 24.9, 8 of 4096 -> 6144 18.2 / 20.6, of 2048 -> 2 x
# 6144 18.1 / 21.6, 1 of 4096 -> 4096 11.7 / 14.3.
OWN_WEIGHT = 48


def makes_its_own(numbers: int, weight: int) -> bool:
    return weight >= OWN_WEIGHT and 128 * numbers <= weight * weight


def _terms(x: torch.Tensor, low_rank: LowRank, rows: AdapterRows, ad: bytes, stream: int, weight: torch.Tensor | None = None) -> torch.Tensor:
    """What the adapters' A make of x, float32 [T, parts * rank]. ``weight``: the one of the product behind, which the launch may ask into L2."""
    t, k = x.shape
    size = 2 * k * low_rank.outputs
    ahead = size if weight is not None and size <= AHEAD else 0
    with on_stream(stream, x.device):
        v = torch.empty((t, low_rank.numbers), dtype=torch.float32, device=x.device)
    if t * low_rank.numbers * k <= TOKEN_WISE or x.dtype is torch.float32 or not _ops().tc_gemm_enabled():
        _check(_lib().ms_adapter_shrink(v.data_ptr(), x.data_ptr(), ad, t, low_rank.outputs, k, _code(x.dtype), weight.data_ptr() if ahead else None, ahead, stream))
    else:
        _by_plan(v, x, rows.plan(low_rank.slots, stream), ad, rows, True, stream)
    return v


def _by_plan(v: torch.Tensor, x: torch.Tensor, plan: _Plan, ad: bytes, rows: AdapterRows, compact: bool, stream: int) -> None:
    lib = native.gemm_tc()
    native.kernel_check(lib.ms_gemm_tc_adapter_v(v.data_ptr(), x.data_ptr(), ad, plan.tile_first, plan.blocks, x.shape[0], x.shape[1], plan.max_blocks, int(compact), rows.status,
                                                 stream), lib=lib, errfn="ms_gemm_tc_last_error")


def product(x: torch.Tensor, low_rank: LowRank, rows: AdapterRows, stream: int) -> tuple:
    """What a product on the 2-CTA tcgen05 kernel takes of the adapters (``AdaptedProduct``), and the V that it points to."""
    ad, plan = low_rank.head + rows.middle + low_rank.tail, rows.plan(low_rank.slots, stream)
    with on_stream(stream, x.device):
        v = torch.empty((plan.max_blocks * TILE, low_rank.numbers), dtype=torch.bfloat16, device=x.device)
    _by_plan(v, x, plan, ad, rows, False, stream)
    return ad + struct.pack("3Qi4x", v.data_ptr(), plan.tile_first, plan.blocks, plan.max_blocks), v


def way_of(tokens: int, outputs: int, inputs: int, rank: int, gated: bool, sms: int) -> str:
    """The way of a bfloat16 product with adapters. "stream": the weight-streaming kernel of decode steps, a thread's terms behind an output's sum. "decode": the swapped-operand tcgen05 kernel of decode steps, the terms on its idle epilogue warps. "pair": the 2-CTA tcgen05 kernel, which
    takes the adapters in its own sums. "apart": the shared product in float32 wherever ``linear`` sends it (beyond 16 rows of bfloat16 the vendor
    library's), the terms added behind.

    Up to 16 tokens stream, where k is at most 2,048, the weight at most 12 MiB and tokens times rank at most 256. decode / stream, us, behind a norm: 8 tokens of rank 16, 1024 -> 4096 9.1 / 6.9,
    1 token 7.4 / 6.2, 16 10.4 / 8.4, 8 of rank 32 9.3 / 8.9, gated 1024 -> 2 x 3 Ki 9.6 / 7.7 (rank 32: 9.9 / 11.0), 2048 -> 1024 8.1 / 7.3; but 16 tokens of 2048 -> 4096 10.6 / 11.1, 8 of
    rank 32 9.7 / 10.5, 4 of rank 64 9.8 / 10.8.

    Else up to 32 tokens decode; up to 64 too at ranks up to 32, and beyond that rank where it is not gated and the outputs are at most twice k. decode / apart / pair, us, one adapter of
    rank 16: 32 tokens of 4096 -> 6144 14.9 / 21.7, of 2048 -> 4096 9.4 / 12.7, of 12288 -> 4096 22.9 / 33.8, gated 4096 -> 2 x 12288 43.2 / 48.7; 64 tokens of 4096 -> 4096 15.0 / 18.4 / 27
    (of 16 adapters 16.7 / 25.6 / 37), of 12288 -> 4096 25.7 / 34.2 / 65, of 1024 -> 4096 13.0 / 12.5 / 11.1 (16 adapters 14.7 / 17.4 / 19.2), gated 4096 -> 2 x 12288 51.7 / 56.9 / 55.2; rank
    64: 4096 -> 4096 18.6 / 28.0 / 27, 1024 -> 4096 16.1 / 19.0 / 11.1, gated 2048 -> 2 x 6144 29.7 / 35.0 / 20.6.

    Beyond, by what both take (us, fitted to a B200): a round of tiles of 256 x 256 on pairs of SMs goes with k; apart is the weights or the operations, three launches, and the outputs
    read and written again. pair / apart: 4096 -> 4096 at 64 tokens 27 / 19, at 512 28 / 33 (rank 64: 29 / 48); 4096 -> 6144 at 200 28 / 33; 12288 -> 4096 at 200 66 / 50, at 700 68 / 79;
    1024 -> 4096 at 64 11 / 13, at 1,100 19 / 36; gated 4096 -> 2 x 12288 at 64 55 / 58, at 200 56 / 90. (Over a hundred such cases the rule's way takes 1 % longer than the best one's.)"""
    rows = outputs * (2 if gated else 1)
    if tokens <= 16 and inputs <= 2048 and inputs * rows <= 6 << 20 and tokens * rank <= 256:
        return "stream"
    if tokens <= FEW_TOKENS or (tokens <= 2 * FEW_TOKENS and (rank <= 32 or (not gated and outputs <= 2 * inputs))):
        return "decode"
    tiles = -(-tokens // TILE) * -(-outputs // (128 if gated else 256))
    apart = max(2.4 * inputs * rows / 6.3e6, 2 * tokens * inputs * rows / 1.2e9) + 10 + (2 + 0.2 * rank) * 1e-6 * tokens * rows
    return "pair" if 6 + -(-tiles // (sms // 2)) * inputs * 0.0048 <= apart else "apart"


def _run(x, weight, out, stream: int, low_rank: LowRank, rows: AdapterRows, gated: bool) -> None:
    t, k = x.shape
    n, ad, device = out.shape[1], low_rank.head + rows.middle + low_rank.tail, x.device
    if x.dtype is torch.bfloat16 and out.dtype is torch.bfloat16 and _ops().tc_gemm_enabled():
        lib = native.gemm_tc()
        way = WAY or way_of(t, n, k, low_rank.rank, gated, rows.sms)
        if way == "stream":
            v = _terms(x, low_rank, rows, ad, stream, weight)
            native.kernel_check(native.kernels().ms_gemm_skinny_adapted_bf16(out.data_ptr(), x.data_ptr(), weight.data_ptr(), t, n, k, int(gated),
                                                                             b"".join((_Q(v.data_ptr()), ad, _Q(0))), stream))
            return
        if way == "decode":
            if makes_its_own(t * low_rank.numbers, 2 * k * low_rank.outputs >> 20):
                tickets = rows.tickets(stream)
                with on_stream(stream, device):
                    v = torch.empty((t, low_rank.numbers), dtype=torch.float32, device=device)
            else:
                v, tickets = _terms(x, low_rank, rows, ad, stream, weight), 0
            term = b"".join((_Q(v.data_ptr()), ad, _Q(tickets)))
            rc = lib.ms_gemm_tc_decode_adapted_bf16(out.data_ptr(), x.data_ptr(), weight.data_ptr(), t, n, k, int(gated), term, rows.status, stream)
            native.kernel_check(rc, lib=lib, errfn="ms_gemm_tc_last_error")
            return
        if way == "pair":
            held, v = product(x, low_rank, rows, stream)
            rc = lib.ms_gemm_tc_adapted_bf16(out.data_ptr(), x.data_ptr(), weight.data_ptr(), t, n, k, 2 if gated else 0, held, rows.status, stream)
            native.kernel_check(rc, lib=lib, errfn="ms_gemm_tc_last_error")
            return
    # the shared product in float32, so that the sum is rounded once
    y = out
    if out.dtype is not torch.float32 or gated:
        with on_stream(stream, device):
            y = torch.empty((t, low_rank.outputs), dtype=torch.float32, device=device)
    _ops().linear(x, weight, out=y, stream=stream)
    v = _terms(x, low_rank, rows, ad, stream)
    _check(_lib().ms_adapter_expand(out.data_ptr(), y.data_ptr(), v.data_ptr(), ad, t, low_rank.outputs, k, _code(x.dtype), _code(out.dtype), int(gated), stream))


def _call(x, weight, out, stream, low_rank: LowRank, rows: AdapterRows, gated: bool) -> torch.Tensor:
    """The call on its tensors' device, and its stream (None: that device's current one)."""
    if torch.cuda.current_device() != low_rank.index:
        with torch.cuda.device(low_rank.index):
            return _call(x, weight, out, stream, low_rank, rows, gated)
    if stream is None:
        stream = _now(low_rank.index)
    if out is None:
        with on_stream(stream, x.device):
            out = torch.empty((x.shape[0], low_rank.outputs), dtype=x.dtype, device=x.device)
    if x.shape[0]:
        _run(x, weight, out, stream, low_rank, rows, gated)
    return out


def linear(x, weight, out, stream, low_rank: LowRank, rows: AdapterRows) -> torch.Tensor:
    check(x, weight, out, low_rank, rows, False)
    return _call(x, weight, out, stream, low_rank, rows, False)


def linear_silu_mul(x, weight, out, stream, low_rank: LowRank, rows: AdapterRows) -> torch.Tensor:
    check(x, weight, out, low_rank, rows, True)
    return _call(x, weight, out, stream, low_rank, rows, True)
