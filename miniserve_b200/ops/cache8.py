"""The paged cache in 8 bits (``csrc/cache8.cuh``): its pools, the write of a step's keys and values, reading them back, and attention over
them. ``ops.qk_norm_rope_kv`` and ``ops.attention`` take a ``Pool8`` where they take a pool of bfloat16, and come here."""

from __future__ import annotations

import ctypes
import struct
from contextlib import nullcontext
from ctypes import c_char_p, c_float, c_int, c_longlong, c_ulonglong, c_void_p
from dataclasses import dataclass
from functools import lru_cache

import torch

from . import build, native

_p, _i, _f, _ll = c_void_p, c_int, c_float, c_longlong
MIN_PAGE = 8
EXPONENT_BIAS = 127
LARGEST, EXPONENTS = 448.0, (-60, 7)


@dataclass(frozen=True, eq=False)
class Pool8:
    """Keys (or values) of one cache entry in 8 bits. ``codes`` uint8 [pages, kv_heads, page_size, d] (bits of ``torch.float8_e4m3fn``) and
    ``exponents`` uint8 [pages, kv_heads, page_size]: number i of a head's vector is code_i * 2^(exponent - 127). The writer takes the smallest
    exponent at which the vector's largest number is at most 448, within 2^-60 and 2^7; a vector with a number that is not finite gets 255 and zero
    codes, and reads as NaN. Other exponents follow the formula too: 0, an empty pool's, is 2^-127."""

    codes: torch.Tensor
    exponents: torch.Tensor

    def __post_init__(self):
        c, e = self.codes, self.exponents
        if c.dtype != torch.uint8 or e.dtype != torch.uint8 or c.dim() != 4 or c.shape[:3] != e.shape:
            raise ValueError(f"an 8-bit pool is uint8 codes [pages, kv_heads, page_size, d] and uint8 exponents of the first three sizes, not "
                             f"{c.dtype} {tuple(c.shape)} and {e.dtype} {tuple(e.shape)}")
        if c.shape[3] % 16 or not 16 <= c.shape[3] <= 256:
            raise ValueError(f"an 8-bit cache takes head sizes that are multiples of 16 up to 256, not {c.shape[3]}")
        if c.shape[2] < MIN_PAGE or c.shape[2] & (c.shape[2] - 1):
            raise ValueError(f"an 8-bit cache takes pages of a power of two of at least {MIN_PAGE} tokens, not {c.shape[2]}")
        if c.device != e.device or not c.is_contiguous() or not e.is_contiguous() or c.data_ptr() % 16 or e.data_ptr() % 8:
            raise ValueError("an 8-bit pool's tensors lie on one device, contiguous, codes on 16 bytes and exponents on 8")
        # what every call asks for: sizes, the device's index (-1: the host), addresses
        for name, value in (("sizes", tuple(c.shape)), ("index", c.get_device()), ("pointers", (c.data_ptr(), e.data_ptr()))):
            object.__setattr__(self, name, value)

    @classmethod
    def empty(cls, pages: int, kv_heads: int, page_size: int, head_dim: int, device="cuda") -> "Pool8":
        """A pool of zeros."""
        return cls(torch.zeros((pages, kv_heads, page_size, head_dim), dtype=torch.uint8, device=device),
                   torch.zeros((pages, kv_heads, page_size), dtype=torch.uint8, device=device))

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def device(self) -> torch.device:
        return self.codes.device


def takes(head_dim: int, page_size: int) -> bool:
    """Whether an 8-bit cache can hold heads of this size in pages of this many tokens."""
    return head_dim % 16 == 0 and 16 <= head_dim <= 256 and page_size >= MIN_PAGE and page_size & (page_size - 1) == 0


CACHE8 = build.Module("cache8", ("cache8.cu",))
_WRITE, _READ = struct.Struct("16Qq9if").pack, struct.Struct("12Qq8i").pack  # ``Write8`` and ``Read8`` of csrc/cache8.cu


def module_for(head_dim: int) -> build.Module:
    return build.Module(f"attn_cache8_d{head_dim}", ("attention_cache8.cu",), defines=(f"MS_HEAD_DIM={head_dim}",))


@lru_cache(maxsize=None)
def _cache_lib():
    lib = ctypes.CDLL(str(build.ensure_built(CACHE8)))
    native._declare(lib, "ms_cache8_last_error", [], c_char_p)
    native._declare(lib, "ms_cache8_set_pdl", [_i], None)
    native._declare(lib, "ms_cache8_write", [c_char_p])
    native._declare(lib, "ms_cache8_read", [c_char_p])
    native._declare(lib, "ms_cache8_unpack", [_p] * 12 + [_i] * 8 + [_ll, _i, _i, _p, _p])
    native._declare(lib, "ms_cache8_capture_id", [_p], c_ulonglong)
    lib.ms_cache8_set_pdl(int(native.pdl_enabled()))
    return lib


def _cache_check(rc: int) -> None:
    native.LAUNCHES[0] += 1
    if rc:
        native.kernel_check(rc, lib=_cache_lib(), errfn="ms_cache8_last_error", launches=0)


class _Split(ctypes.Structure):
    """``Split8`` of csrc/attention_cache8.cu."""

    _fields_ = [(n, _p) for n in ("cu_q", "q_start", "page_indptr", "page_indices", "status", "part", "cut")] + [
        (n, _i) for n in ("rows", "tile0", "tiles", "nq", "nkv", "window", "sink", "page_size", "ctas")] + [("scale", _f), ("num_pages", _i), ("behind", _i), ("all_rows", _i), ("num_entries", _i), ("ahead", _i)]


class _AttnLib:
    """The attention kernels of one head size."""

    def __init__(self, head_dim: int):
        lib = ctypes.CDLL(str(build.ensure_built(module_for(head_dim))))
        pre = f"ms_attn_cache8_d{head_dim}_"
        self.last_error = native._declare(lib, pre + "last_error", [], c_char_p)
        native._declare(lib, pre + "set_pdl", [_i], None)(int(native.pdl_enabled()))
        self.split = native._declare(lib, pre + "split", [_p, _i, _i] + [_p] * 7)
        self.part_floats = native._declare(lib, pre + "part_floats", [_i], _ll)
        self.slice, self.switch = (native._declare(lib, pre + name, [])() for name in ("slice", "switch_slices"))
        self.warps, self.alone_most = (native._declare(lib, pre + name, [_i]) for name in ("warps", "alone_most"))
        self.most_rows = native._declare(lib, pre + "most_rows", [])()
        self.max_units = native._declare(lib, pre + "max_units", [])()


@lru_cache(maxsize=None)
def _attn_lib(head_dim: int) -> _AttnLib:
    return _AttnLib(head_dim)


def _stream_of(stream, device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream if stream is None else stream


_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32


def _check_tables(index: int, *tensors: torch.Tensor) -> None:
    for t in tensors:
        if t.dtype is not _I32 or t.get_device() != index or not t.is_contiguous():
            raise ValueError("positions, rows, page tables and the status word are contiguous int32 tensors on the pools' device")


def _check_pools(k: Pool8, v: Pool8) -> None:
    if not isinstance(k, Pool8) or not isinstance(v, Pool8):
        raise TypeError("keys and values are both in 8 bits or both not")
    if k.sizes != v.sizes or k.index != v.index:
        raise ValueError(f"the pools of keys and values differ: {k.sizes} on {k.device}, {v.sizes} on {v.device}")
    if k.index < 0:
        raise ValueError("kernel operands must be contiguous CUDA tensors")


def qk_norm_rope_kv(q_out, k_pool: Pool8, v_pool: Pool8, qkv, q_norm_w, k_norm_w, inv_freq, rotary_dim: int, eps: float, positions, row_of_token,
                    page_indptr, page_indices, page_size: int, status, stream=None, cos_sin=None) -> None:
    """``ops.qk_norm_rope_kv`` with keys and values quantised into 8-bit pools: what is rounded is the float32 number behind norm and rotation
    (values: as projected). ``page_indptr`` [rows + 1], ``page_indices``: entry 0 of row r's table lies at ``page_indptr[r]``, which may be outside the tables where a window gave
    its pages back; the last number is where all tables end. A token whose position leads outside them, or to no page of the pool, raises the status word and is not written;
    two tokens of a call do not share a place."""
    _check_pools(k_pool, v_pool)
    t, nq, d = q_out.shape
    pages, nkv, held, dim = k_pool.sizes
    dev = k_pool.index
    if held != page_size or dim != d or qkv.shape != (t, (nq + 2 * nkv) * d):
        raise ValueError(f"q is {tuple(q_out.shape)}, the projection {tuple(qkv.shape)}, the pools {k_pool.sizes}, the page size {page_size}")
    pq, px, pw, pk = q_out.data_ptr(), qkv.data_ptr(), 0 if q_norm_w is None else q_norm_w.data_ptr(), 0 if k_norm_w is None else k_norm_w.data_ptr()
    for x, at, n in ((q_out, pq, 0), (qkv, px, 0), (q_norm_w, pw, d), (k_norm_w, pk, d)):
        if x is not None and (x.dtype is not _BF16 or x.get_device() != dev or not x.is_contiguous() or at % 16 or (n and x.numel() != n)):
            raise ValueError("an 8-bit cache is written from contiguous bfloat16 tensors on its device, on 16 bytes; norm weights have the head's size")
    freq = table = 0
    if inv_freq is not None:
        if inv_freq.dtype is not _F32 or inv_freq.numel() != rotary_dim // 2 or inv_freq.get_device() != dev or not inv_freq.is_contiguous():
            raise ValueError("inv_freq is float32 [rotary_dim / 2] on the pools' device")
        freq = inv_freq.data_ptr()
        if cos_sin is not None:
            if cos_sin.dtype is not _F32 or cos_sin.shape != (t, rotary_dim) or cos_sin.get_device() != dev or not cos_sin.is_contiguous():
                raise ValueError("cos_sin is float32 [tokens, rotary_dim], contiguous, on the pools' device")
            table = cos_sin.data_ptr()
    _check_tables(dev, positions, row_of_token, page_indptr, page_indices, status)
    if positions.numel() < t or row_of_token.numel() < t:
        raise ValueError(f"{t} tokens need as many positions and rows")
    kc, ke = k_pool.pointers
    vc, ve = v_pool.pointers
    _cache_check(_cache_lib().ms_cache8_write(_WRITE(
        pq, kc, ke, vc, ve, px, pw, pk, freq, table, positions.data_ptr(), row_of_token.data_ptr(), page_indptr.data_ptr(), page_indices.data_ptr(),
        status.data_ptr(), _stream_of(stream, k_pool.device), pages, dev, page_indptr.numel() - 1, page_indices.numel(), t, nq,
        nkv, d, rotary_dim if freq else 0, page_size, eps)))


def read_cache(k_out: torch.Tensor, v_out: torch.Tensor, k_pool: Pool8, v_pool: Pool8, positions: torch.Tensor, row_of_token: torch.Tensor,
               page_indptr: torch.Tensor, page_indices: torch.Tensor, status: torch.Tensor, stream=None) -> None:
    """The cached keys and values of given tokens as dense rows: ``k_out``, ``v_out`` [N, kv_heads, d], bfloat16 (exact) or float32 (exact), row i what
    the cache holds at position ``positions[i]`` of row ``row_of_token[i]`` of the page tables (as ``qk_norm_rope_kv`` takes them). A position that leads outside the tables, or to no
    page of the pool, raises the status word and leaves its row as it was; of a window's group, only positions that were not given back are asked for."""
    _check_pools(k_pool, v_pool)
    pages, nkv, page_size, d = k_pool.sizes
    dev, shape = k_pool.index, k_out.shape
    n = shape[0]
    if shape != (n, nkv, d) or v_out.shape != shape or positions.numel() < n or row_of_token.numel() < n:
        raise ValueError(f"rows {tuple(shape)} and {tuple(v_out.shape)} of pools {k_pool.sizes}, {positions.numel()} positions, {row_of_token.numel()} rows")
    dtype = k_out.dtype
    if (dtype is not _BF16 and dtype is not _F32) or v_out.dtype is not dtype:
        raise TypeError(f"a cache is read as bfloat16 or float32, not {dtype} and {v_out.dtype}")
    pk, pv = k_out.data_ptr(), v_out.data_ptr()
    if k_out.get_device() != dev or v_out.get_device() != dev or not k_out.is_contiguous() or not v_out.is_contiguous() or pk % 16 or pv % 16:
        raise ValueError("the rows are contiguous, on 16 bytes, on the pools' device")
    _check_tables(dev, positions, row_of_token, page_indptr, page_indices, status)
    kc, ke = k_pool.pointers
    vc, ve = v_pool.pointers
    _cache_check(_cache_lib().ms_cache8_read(_READ(
        pk, pv, kc, ke, vc, ve, positions.data_ptr(), row_of_token.data_ptr(), page_indptr.data_ptr(), page_indices.data_ptr(), status.data_ptr(),
        _stream_of(stream, k_pool.device), pages, dev, page_indptr.numel() - 1, page_indices.numel(), n, nkv, d, page_size, 0 if dtype is _F32 else 1)))


# ------------------------------------------------------------------ attention

def _on_stream(ctx, device: torch.device):
    """Allocations (and their zeroing) in the order of the step's stream, where that is not the current one."""
    if ctx.stream == torch.cuda.current_stream(device).cuda_stream:
        return nullcontext()
    return torch.cuda.stream(_stream(ctx, device))


def _stream(ctx, device: torch.device) -> torch.cuda.Stream:
    return torch.cuda.ExternalStream(ctx.stream, device=device) if ctx.stream else torch.cuda.default_stream(device)


def _workspace(ctx, floats: int, device) -> torch.Tensor:
    """Partial results of steps that run one after the other. What is outgrown stays alive for graphs that hold its address; a capture that needs
    more than there is gets its own."""
    held = ctx.scratch.get("cache8")
    if held is not None and held.numel() >= floats:
        return held
    with _on_stream(ctx, device):
        new = torch.empty(floats, dtype=torch.float32, device=device)
    ctx.scratch.setdefault("retired", []).append(new)
    if not torch.cuda.is_current_stream_capturing():
        ctx.scratch["cache8"] = new
    return new


def _alone(ctx, lib: _AttnLib, rows: range, tiles: range, tile_rows: int, heads: int, nkv: int, window: int) -> bool:
    """Whether the kernel would give every item (tile of query rows of a request, and kv head) a CTA of its own, by its own rule: then none is cut, and the second
    kernel need not run."""
    if len(ctx.host_q_len) < rows.stop:
        return False
    total = longest = 0
    for r in rows:
        start, most = ctx.host_q_start[r], ctx.host_q_len[r] * heads
        for row0 in range(tiles.start * tile_rows, min(tiles.stop * tile_rows, most), tile_rows):
            low = max(0, start + row0 // heads - window + 1) if window else 0
            n = max(1, -(-(start + (min(row0 + tile_rows, most) - 1) // heads + 1) // lib.slice) - low // lib.slice)
            total, longest = total + n + lib.switch, max(longest, n)
    warps = lib.warps(tile_rows)
    return -(-longest // warps) <= lib.alone_most(-(-total * nkv // (ctx.sm_count * warps)))


def _plans(ctx, group: int, ranges: list, key: tuple, device) -> list:
    """The launches over ``ranges`` of a step's rows, ``(first, rows, the most new tokens of one)``, the same for every layer with these sizes and this window:
    ``(plan, its address, query rows of a tile, the most of a request, launches)``."""
    nq, nkv, d, scale, window, sink, page_size, pages = key
    lib = _attn_lib(d)
    _check_tables(device.index, ctx.cu_q, ctx.q_start, ctx.page_indptr[group], ctx.page_indices[group], ctx.status)
    ctas = ctx.sm_count
    floats = lib.part_floats(ctas)
    part = _workspace(ctx, floats + 4 * ctas, device)
    fixed = not ctx.graph_bucket and not torch.cuda.is_current_stream_capturing()  # (a graph may be replayed for other lengths)
    out = []
    for begin, rows_all, most_tokens in ranges:
        most = most_tokens * (nq // nkv)
        tiles = -(-most // lib.most_rows)  # as few as there have to be, of one size
        tile_rows = -(-most // (8 * tiles)) * 8
        tiles_each = min(tiles, lib.max_units)
        rows_each = lib.max_units // tiles_each
        for first in range(begin, begin + rows_all, rows_each):
            skip, rows = 4 * first, min(rows_each, begin + rows_all - first)  # the per-row tables are int32
            for tile0 in range(0, tiles, tiles_each):
                here = min(tiles_each, tiles - tile0)
                whole = fixed and rows * here * nkv <= ctas and _alone(ctx, lib, range(first, first + rows), range(tile0, tile0 + here), tile_rows, nq // nkv, nkv, window)
                plan = _Split(ctx.cu_q.data_ptr() + skip, ctx.q_start.data_ptr() + skip, ctx.page_indptr[group].data_ptr() + skip, ctx.page_indices[group].data_ptr(),
                              ctx.status.data_ptr(), part.data_ptr(), part.data_ptr() + 4 * floats, rows, tile0, here, nq, nkv, window, sink, page_size, ctas, scale, pages,
                              not whole, ctx.num_rows - first, ctx.page_indices[group].numel(), bool(getattr(ctx, "tables_ahead", False)))
                out.append((plan, ctypes.addressof(plan), tile_rows, most, 1 if whole else 2))
    return out


def _of_one_size(ctx, first: int, heads: int, lib: _AttnLib) -> list:
    """Rows [first, num_rows) in ranges that a launch takes whole, as far as that goes: tiles are counted by a range's longest row."""
    out = []
    for r in range(first, ctx.num_rows):
        n = ctx.host_q_len[r]
        if out:
            at, rows, most = out[-1]
            if (rows + 1) * -(-max(n, most) * heads // lib.most_rows) <= lib.max_units:
                out[-1] = (at, rows + 1, max(n, most))
                continue
        out.append((r, 1, n))
    return [x for x in out if x[2]]


def _split(out, q, k_pool: Pool8, v_pool: Pool8, ctx, group: int, scale: float, window: int, sink: bool, first: int, rows: int, most_tokens: int | None, nq: int) -> None:
    """Rows [first, first + rows) of the step, of at most ``most_tokens`` new tokens (None: of as many as the host's list says), on the kernel that shares out keys."""
    pages, nkv, page_size, d = k_pool.sizes
    key = ("cache8", group, first, rows, most_tokens, nq, nkv, d, scale, window, sink, page_size, pages)
    held = ctx.step_cache.get(key)
    if held is None:
        lib = _attn_lib(d)
        ranges = _of_one_size(ctx, first, nq // nkv, lib) if most_tokens is None else [(first, rows, most_tokens)]
        held = ctx.step_cache[key] = (lib, _plans(ctx, group, ranges, (nq, nkv, d, float(scale), window, int(sink), page_size, pages), k_pool.device))
    lib, plans = held
    for plan, at, tile_rows, most, launches in plans:
        native.LAUNCHES[0] += launches
        if lib.split(at, tile_rows, most, out.data_ptr(), q.data_ptr(), *k_pool.pointers, *v_pool.pointers, ctx.stream):
            raise native.NativeError(lib.last_error().decode())


# Steps of several tokens a request have two ways: the kernel that shares out keys reads the codes again for every 16 query rows of a kv head (24 at head sizes up to 64); or their
# pages are unpacked to bfloat16 and attended over by a bfloat16 cache's kernels. Measured (one B200, us, keys shared out / unpacked):
#   head size 128, unpacked for the tcgen05 kernel (256 query rows a tile), by query rows of a request:   64      96     128     256
#     1 request behind 2,000 tokens                                                                      26/34   26/34   28/36   34/40
#     16 behind 2,000                                                                                    75/93   99/93  126/89  226/101
#     1 behind 32,000                                                                                    65/108  87/108 108/108 191/116
#   others, unpacked for the mma.sync kernel (64 query rows a CTA, which walks all their keys), by new tokens of a request:
#     head size 64, 8 heads a kv head, 4 requests behind 3,000 tokens     32: 43/190   128: 111/197   1,024: 919/1034
#                                      4 behind 500                       32: 25/45    128: 49/51     512: 203/156   1,024: 436/344
#                                      8 from the beginning               64: 31/20    128: 63/31     512: 315/131
#     head size 64, 1 head a kv head, 1 from the beginning                512: 31/37   4,096: 313/414;   8 so  512: 86/86   4,096: 2325/2387
#     head size 80, 2 heads a kv head, 1 from the beginning               512: 33/43   2,048: 121/156;   8 so  512: 115/96  2,048: 917/801;   4 behind 3,000  512: 278/446
#     head size 256, 4 heads a kv head, 1 from the beginning              256: 20/31   1,024: 72/96;     8 so  256: 92/70   1,024: 585/436;   4 behind 3,000  256: 242/293
# So up to SPLIT_ROWS query rows always share out keys. Beyond, the tcgen05 kernel takes what it takes: right for many requests and for many keys; a lone request of 128 or 256 query rows behind
# 2,000 keys is 6 to 8 us slower for it. Of other shapes the mma.sync kernel takes steps with no more keys behind them
# than new tokens where 8 heads and more share a kv head, or where 2 and more do and 4 requests and more come: it has many CTAs then, of few keys each.
SPLIT_ROWS = 96
UNPACKED_BYTES = 1 << 30  # of pages unpacked at a time, unless a single request has more


def _shares_out(q, k_pool: Pool8, ctx, first: int) -> bool:
    """Whether rows [first, num_rows), some of more than SPLIT_ROWS query rows, go to the kernel that shares out keys."""
    from . import attention_tc_ok  # (this module is imported by theirs)

    rows, heads = ctx.num_rows - first, q.shape[1] // k_pool.sizes[1]
    if not (heads >= 8 or (heads >= 2 and rows >= 4)):
        return not attention_tc_ok(q, k_pool)
    key = ("cache8_more_behind", first)
    more_behind = ctx.step_cache.get(key)
    if more_behind is None:
        more_behind = ctx.step_cache[key] = sum(ctx.host_q_start[first:ctx.num_rows]) > sum(ctx.host_q_len[first:ctx.num_rows])
    return more_behind and not attention_tc_ok(q, k_pool)


class _Unpacked:
    """A step's context whose pages of one group are the unpacked ones, by tables of their own: rows [first, num_rows). Plans are its own (those of the context are of all rows)."""

    def __init__(self, ctx, group: int, num_rows: int, indptr: torch.Tensor, ids: torch.Tensor, scratch: dict):
        self.__dict__.update(ctx.__dict__)
        self.num_rows, self.scratch, self.step_cache = num_rows, scratch, {}
        self.page_indptr, self.page_indices = list(ctx.page_indptr), list(ctx.page_indices)
        self.page_indptr[group], self.page_indices[group] = indptr, ids


def _parts(ctx, first: int, window: int, page_size: int, page_bytes: int) -> list:
    """Rows [first, num_rows) in parts whose pages fit: ``(first row, row behind, pages)``. A row's pages begin with the first that its window reaches."""
    out, at, entries = [], first, 0
    for r in range(first, ctx.num_rows):
        start, tokens = ctx.host_q_start[r], ctx.host_q_len[r]
        n = -(-(start + tokens) // page_size) - (max(0, start - window + 1) // page_size if window else 0) if tokens else 0
        if entries and (entries + n) * page_bytes > UNPACKED_BYTES:
            out.append((at, r, entries))
            at, entries = r, 0
        entries += n
    out.append((at, ctx.num_rows, entries))
    return [x for x in out if x[2]]


def _unpacked(ctx, capture: int, numbers: int, ints: int, device: torch.device) -> tuple:
    """Pages of K and of V (``numbers`` each) and ``ints`` entries of tables for steps that run one after the other, and the scratch that they are kept in. What a launch reads of them it
    has written before. ``capture``: which one, 0: none."""
    scratch = ctx.step_cache.setdefault(("cache8_scratch", capture), {}) if capture else ctx.scratch
    held = scratch.get("cache8_pages")  # with the stream they were made on
    if held is not None and held[0].numel() >= numbers and held[2].numel() >= ints:
        if held[3] != ctx.stream:  # (outgrown, they go back to the stream they came from, which is not to use them before this one is done)
            for t in held[:3]:
                t.record_stream(_stream(ctx, device))
        return *held[:3], scratch
    if held is not None:  # (a context grows portion by portion: twice as much the next time, up to what a step of several rows may take)
        numbers = max(numbers, min(2 * held[0].numel(), UNPACKED_BYTES // 4)) if held[0].numel() < numbers else held[0].numel()
        ints = max(ints, 2 * held[2].numel())
        # the old ones go first: here, and what the step keeps of them
        del scratch["cache8_pages"], held
        for key in [x for x in ctx.step_cache if x[0] == "cache8_unpacked" and x[-1] == capture]:
            del ctx.step_cache[key]
    with _on_stream(ctx, device):
        new = tuple(torch.empty(n, dtype=t, device=device) for n, t in ((numbers, torch.bfloat16), (numbers, torch.bfloat16), (ints, torch.int32)))
    scratch["cache8_pages"] = *new, ctx.stream
    return *new, scratch


def _dense(out, q, k_pool: Pool8, v_pool: Pool8, ctx, group: int, scale: float, window: int, sink: bool, first: int) -> None:
    """Rows [first, num_rows) of the step over pages unpacked to bfloat16. A captured graph has scratch of its own, the prompt kernels' included, from the graph's memory:
    what eager steps outgrow may go, and what a kernel finds zero at its start the graph makes so."""
    from . import attention_bf16, attention_tc_ok, attention_tc_prefill  # (this module is imported by theirs)

    pages, nkv, page_size, d = k_pool.sizes
    key = ("cache8_unpacked", group, first, q.shape[1], nkv, page_size, d, window, ctx.stream, _cache_lib().ms_cache8_capture_id(ctx.stream))
    parts, scope = ctx.step_cache.get(key), nullcontext()
    if parts is None:
        scope = _on_stream(ctx, k_pool.device)  # (what the prompt kernels make at a first call is made, and zeroed, there)
        _check_tables(k_pool.index, ctx.cu_q, ctx.q_start, ctx.page_indptr[group], ctx.page_indices[group], ctx.status)
        page = nkv * page_size * d
        parts = _parts(ctx, first, window, page_size, 4 * page)
        most = max((n for _, _, n in parts), default=0)
        rows, num_ids = ctx.num_rows + 1, most + ctx.page_indices[group].numel()
        *pools, tables, scratch = _unpacked(ctx, key[-1], most * page, rows + num_ids, k_pool.device)
        k, v = (x[:most * page].view(most, nkv, page_size, d) for x in pools)
        indptr, ids = tables[:rows], tables[rows:rows + num_ids]
        parts = ctx.step_cache[key] = (k, v, [(a, n, _Unpacked(ctx, group, b, indptr, ids, scratch)) for a, b, n in parts])
    k, v, parts = parts
    with scope:
        for a, entries, view in parts:
            _cache_check(_cache_lib().ms_cache8_unpack(
                k.data_ptr(), v.data_ptr(), view.page_indices[group].data_ptr(), view.page_indptr[group].data_ptr(), *k_pool.pointers, *v_pool.pointers, ctx.cu_q.data_ptr(),
                ctx.q_start.data_ptr(), ctx.page_indptr[group].data_ptr(), ctx.page_indices[group].data_ptr(), a, view.num_rows, ctx.num_rows, entries, nkv, d, window, page_size,
                pages, ctx.page_indices[group].numel(), view.page_indices[group].numel(), ctx.status.data_ptr(), ctx.stream))
            if attention_tc_ok(q, k):
                attention_tc_prefill(out, q, k, v, view, group, scale, window or None, a, sink)
            else:
                attention_bf16.run_prefill(out, q, k, v, view, group, scale, window or None, a, sink)


def attention(out: torch.Tensor, q: torch.Tensor, k_pool: Pool8, v_pool: Pool8, ctx, group: int, scale: float, window: int | None, sink: bool = False) -> None:
    """``ops.attention`` over an 8-bit cache: causal attention of the step's new tokens (bfloat16 queries and output) over the pages of cache group
    ``group``, window and sink as there. Single tokens, drafted ones and what else the rule at SPLIT_ROWS says go to the kernel that shares out keys
    (``csrc/attention_cache8.cu``); other prompts to a bfloat16 cache's kernels, over pages unpacked first. A page that a row looks at and the tables or
    the pool do not have raises the status word (without a window a row's table ends where the next one begins). Single and drafted
    tokens go by the lengths on the device; other prompts' pages are counted by ``ctx.host_q_start`` and ``ctx.host_q_len``, and rows that turn out to have more of
    them raise the status word. Workspaces lie in ``ctx.scratch``: steps of one context (and graphs captured of them) run one after the other."""
    if not isinstance(v_pool, Pool8) or k_pool.sizes != v_pool.sizes or k_pool.index != v_pool.index or k_pool.index < 0:
        _check_pools(k_pool, v_pool)
    shape = q.shape
    nq, d = shape[1], shape[2]
    _, nkv, _, dim = k_pool.sizes
    dev = k_pool.index
    if not (out.shape == shape and q.dtype is torch.bfloat16 and out.dtype is torch.bfloat16 and q.get_device() == dev and out.get_device() == dev
            and q.is_contiguous() and out.is_contiguous()):
        raise ValueError("attention over an 8-bit cache takes contiguous bfloat16 queries and output of one shape on the pools' device")
    window, heads = window or 0, nq // nkv
    if dim != d or nq % nkv or window < 0:
        raise ValueError(f"{nq} query heads of {d} over pools {k_pool.sizes}, window {window}")
    if getattr(ctx, "recorder", None) is not None:
        # a pass that is captured for steps of other lengths too: launched anew for each, between the graphs
        ctx.recorder.defer(lambda step: attention(out, q, k_pool, v_pool, step, group, scale, window, sink))
        return
    if not shape[0]:
        return
    if torch.cuda.current_device() != dev:
        with torch.cuda.device(dev):
            attention(out, q, k_pool, v_pool, ctx, group, scale, window, sink)
        return
    if ctx.max_q_len * heads <= SPLIT_ROWS:
        _split(out, q, k_pool, v_pool, ctx, group, scale, window, sink, 0, ctx.num_rows, ctx.max_q_len, nq)
        return
    single = ctx.leading_single_rows
    if single:
        _split(out, q, k_pool, v_pool, ctx, group, scale, window, sink, 0, single, 1, nq)
    if single == ctx.num_rows:
        return
    if _shares_out(q, k_pool, ctx, single):
        _split(out, q, k_pool, v_pool, ctx, group, scale, window, sink, single, ctx.num_rows - single, None, nq)
    else:
        _dense(out, q, k_pool, v_pool, ctx, group, scale, window, sink, single)
