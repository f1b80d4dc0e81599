"""The 8-bit cache in plain 64-bit arithmetic: the format from its bits, quantising, attention; and batches over random pages."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from miniserve_b200 import ops
from tests import kernel_util as ku

EXP_MIN, EXP_MAX, TOP = -60, 7, 448.0


def values64(codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    """float64 [..., d] of codes uint8 [..., d] and exponents uint8 [...]."""
    c = codes.long()
    field, man = (c >> 3) & 15, (c & 7).double()
    mag = torch.where(field > 0, (1 + man / 8) * torch.exp2(field.double() - 7), man / 8 * 2.0 ** -6)
    mag = torch.where((c & 127) == 127, math.nan, mag)
    x = torch.where(c >= 128, -mag, mag) * torch.exp2(exps.double() - 127)[..., None]
    return torch.where((exps == 255)[..., None], math.nan, x)


def exponent64(x: torch.Tensor) -> torch.Tensor:
    """The exponent that a vector x [..., d] (float64, finite) is held with."""
    amax = x.abs().amax(-1)
    e = torch.full_like(amax, EXP_MIN)
    for n in range(EXP_MIN, EXP_MAX):
        e = torch.where(amax > TOP * 2.0 ** n, torch.full_like(e, n + 1), e)
    return e


def check_held(codes: torch.Tensor, exps: torch.Tensor, x: torch.Tensor, slack: float) -> None:
    """Codes and exponents stand for x (float64 [..., d], finite) to half a step of e4m3; ``slack``: relative error that x itself may
    have had before it was rounded (float32 arithmetic)."""
    got, e = values64(codes, exps), exps.double() - 127
    amax = x.abs().amax(-1)
    assert bool(((e >= EXP_MIN) & (e <= EXP_MAX)).all())
    assert bool(((amax <= TOP * torch.exp2(e) * (1 + slack)) | (e == EXP_MAX)).all()), "an exponent is too small"
    assert bool(((amax > TOP * torch.exp2(e - 1) * (1 - slack)) | (e == EXP_MIN)).all()), "an exponent is too large"
    clipped = x.clamp(-TOP * 2.0 ** EXP_MAX, TOP * 2.0 ** EXP_MAX)
    # half a step: 2^-4 of the number, or half of the smallest code (2^-9) of the vector's scale
    bound = torch.maximum(clipped.abs() * 2.0 ** -4, (2.0 ** -10 * torch.exp2(e))[..., None].expand_as(x)) + slack * amax[..., None]
    off = (got - clipped).abs() - bound
    assert bool((off <= 0).all()), f"a code is {off.max().item()} beyond half a step"


def random_pool(pages, kv_heads, page, d, gen, spread=0.7) -> ops.Pool8:
    """A pool of random codes that a writer could have made (no NaN), exponents of vectors of different sizes."""
    codes = torch.randint(0, 256, (pages, kv_heads, page, d), generator=gen, device="cuda", dtype=torch.uint8)
    codes = torch.where((codes & 127) == 127, codes - 1, codes)
    codes = torch.where((codes & 127) > 0x58, codes - 0x20 * ((codes & 127) > 0x58).to(torch.uint8), codes)  # few of the largest
    exps = (127 - 6 + spread * torch.randn((pages, kv_heads, page), generator=gen, device="cuda")).round().to(torch.uint8)
    return ops.Pool8(codes, exps)


class Batch8(ku.PagedBatch):
    """Rows (start, q_len) over random pages of random 8-bit pools; every slot that no row holds is poison."""

    def __init__(self, rows, page, kv_heads, d, seed=0, spread=0.7):
        super().__init__(rows, page, kv_heads, d, torch.bfloat16, seed)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.k8 = random_pool(self.num_pages, kv_heads, page, d, gen, spread)
        self.v8 = random_pool(self.num_pages, kv_heads, page, d, gen, spread)
        held = torch.zeros((self.num_pages, page), dtype=torch.bool)
        for (s, n), t in zip(rows, self.tables):
            for i, p in enumerate(t):
                held[p, :max(0, min(page, s + n - i * page))] = True
        gone = (~held).cuda()[:, None, :].expand(-1, kv_heads, -1)
        for pool in (self.k8, self.v8):
            pool.codes[gone] = 0x7F
            pool.exponents[gone] = 255

    def dense64(self, r: int):
        """Keys and values of row r, float64 [kv_len, kv_heads, d]."""
        n = sum(self.rows[r])
        t = torch.tensor(self.tables[r], device="cuda")
        out = []
        for pool in (self.k8, self.v8):
            x = values64(pool.codes[t], pool.exponents[t])  # [pages, kv_heads, page, d]
            out.append(x.permute(0, 2, 1, 3).reshape(-1, x.shape[1], x.shape[3])[:n])
        return out


def attention64(q, k, v, q_positions, scale, window=None, sink=False):
    """Attention in 64 bits, and sum_j p_j |v_j| beside it (what rounding the weights can move)."""
    n, heads, d = q.shape
    group = heads // k.shape[1]
    key = torch.arange(k.shape[0], device=q.device)
    pos = torch.as_tensor(q_positions, device=q.device)[:, None]
    seen = key <= pos
    if window:
        seen &= key > pos - window
    out, mass = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    for h in range(heads):
        s = torch.where(seen, (q[:, h].double() @ k[:, h // group].T) * scale, -math.inf)
        m = s.amax(1, keepdim=True).clamp_min(-1e300)
        p = torch.where(seen, torch.exp(s - m), 0.0)
        total = p.sum(1, keepdim=True) + (torch.exp(-m) if sink else 0.0)
        p = torch.where(total > 0, p / total, 0.0)
        vh = torch.where(seen.any(0)[:, None], v[:, h // group], 0.0)
        out[:, h], mass[:, h] = p @ vh, p @ vh.abs()
    return out, mass


def packed_tables(rows, page: int, window, tables) -> tuple[list, list]:
    """``page_indptr`` and ``page_indices`` as the engine's packer lays them out for rows (start, q_len) of a group with ``window``: pages that the window had passed when the step began were
    given back. ``tables``: the pages of every row, from position 0 on."""
    from miniserve_b200.cache import BlockAllocator
    from miniserve_b200.ops import native

    alloc = BlockAllocator(sum(len(t) for t in tables) + 1, page)
    held, name = [], {}
    for s, n in rows:
        t = alloc.new_table()
        t.append_tokens(s)
        if window:
            t.release_below(s - window + 1)
        t.append_tokens(n)
        held.append(t)
    for t, pages in zip(held, tables):
        for block, p in zip(t.blocks, pages):
            if block >= 0:
                assert block not in name
                name[block] = p
    arr = lambda x: np.asarray(x, dtype=np.int32)  # noqa: E731
    count, total = len(rows), sum(n for _, n in rows)
    arena, offsets = np.zeros(8 * total + 64 * count + sum(len(t) for t in tables) + 256, dtype=np.int32), (ctypes.c_longlong * 11)()
    handles = (ctypes.c_void_p * count)(*[t.handle for t in held])
    qs, ql, ids, slots, want, pad = arr([s for s, _ in rows]), arr([n for _, n in rows]), arr([0] * total), arr([0] * count), arr([]), arr([0])
    end = native.host().ms_pack_step(arena.ctypes.data, arena.size, offsets, count, 0, qs.ctypes.data, ql.ctypes.data, ids.ctypes.data, slots.ctypes.data, want.ctypes.data, 0, 1, handles,
                                     pad.ctypes.data, 0, 0, 0, 1, page)
    assert end > 0
    indptr = arena[offsets[8]:offsets[8] + count + 1].tolist()
    return indptr, [name.get(b, -1) for b in arena[offsets[9]:offsets[9] + indptr[-1]].tolist()]


class Packed8(Batch8):
    """Rows in the packer's layout for a group with ``window``: the pages that it has passed are not in the tables, and poison."""

    def __init__(self, rows, page, kv_heads, d, window, seed=0):
        super().__init__(rows, page, kv_heads, d, seed)
        i32 = dict(dtype=torch.int32, device="cuda")
        indptr, indices = packed_tables(rows, page, window, self.tables)
        self.page_indptr, self.page_indices = torch.tensor(indptr, **i32), torch.tensor(indices, **i32)
        gone = sorted({p for t in self.tables for p in t} - set(indices))
        for pool in (self.k8, self.v8):
            pool.codes[gone] = 0x7F
            pool.exponents[gone] = 255
