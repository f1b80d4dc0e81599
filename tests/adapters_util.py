"""Helpers of the adapters' tests: inputs, the formula in 64 bits, and how far a result may be from it."""

from __future__ import annotations

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a step of a type, relative


def made(rows, k, parts, rank, slots, dtype, seed=0, device="cuda"):
    """x, weight, LowRank, AdapterRows for requests ``rows`` of (tokens, slot)."""
    from miniserve_b200 import ops

    gen = torch.Generator(device=device).manual_seed(seed)
    n, tokens = sum(parts), sum(c for c, _ in rows)

    def draw(*shape, std):
        return (torch.randn(shape, generator=gen, device=device) * std).to(dtype)

    x, w = draw(tokens, k, std=1.0), draw(n, k, std=k ** -0.5)
    ends = [sum(parts[:i + 1]) for i in range(len(parts))]
    low = ops.LowRank(draw(slots, len(parts) * rank, k, std=k ** -0.5), draw(slots, n, rank, std=rank ** -0.5),
                      0.5 + torch.rand((slots,), generator=gen, device=device), tuple(ends))
    return x, w, low, rows_of(rows, device)


def rows_of(rows, device="cuda"):
    from miniserve_b200 import ops

    i32 = dict(dtype=torch.int32, device=device)
    return ops.AdapterRows(torch.tensor([s for _, s in rows], **i32), torch.tensor([i for i, (c, _) in enumerate(rows) for _ in range(c)], **i32))


def formula(x, w, low, rows):
    """(y, tolerance) float64 [T, N]: the shared product and the adapters', token by token. The tolerance counts: the shared product stored in the
    type and the sum stored again (half a step each), the adapter's r numbers stored in the type (half a step of each term of B's sum), and sums of
    K and r terms in 32 bits, each addition off by 2^-24 of a partial sum that is no larger than the sum of the terms' magnitudes."""
    x64, w64 = x.double(), w.double()
    half = HALF[x.dtype]
    base, mags = x64 @ w64.T, x64.abs() @ w64.abs().T
    y, tol = base.clone(), 2.0 ** -24 * (x.shape[1] + 2) * mags
    slot = rows.slot_of_row[rows.row_of_token.long()].tolist()
    r, k = low.rank, x.shape[1]
    for t, s in enumerate(slot):
        if not 0 <= s < low.slots:
            continue
        a, b, c = low.a[s].double(), low.b[s].double(), float(low.scale[s])
        v, va = c * (a @ x64[t]), c * (a.abs() @ x64[t].abs())
        at = 0
        for p, end in enumerate(low.ends):
            bp = b[at:end]
            y[t, at:end] += bp @ v[p * r:(p + 1) * r]
            tol[t, at:end] += half * (bp.abs() @ v[p * r:(p + 1) * r].abs()) + 2.0 ** -24 * (k + r + 4) * (bp.abs() @ va[p * r:(p + 1) * r])
            at = end
    return y, tol + half * (base.abs() + y.abs()) + 1e-30


def gated(y, tol, dtype):
    """(silu(gate) * up, tolerance) of stacked gate|up columns: |silu'| is below 1.1; the exponential and the division of the kernels' fast forms
    are good to 2^-20."""
    g, u = y.chunk(2, 1)
    dg, du = tol.chunk(2, 1)
    out = g * torch.sigmoid(g) * u
    return out, 1.1 * dg * (u.abs() + du) + (g * torch.sigmoid(g)).abs() * du + (HALF[dtype] + 2.0 ** -20) * out.abs() + 1e-30


def close(got, want, tol):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} outside, worst {((got.double() - want).abs() / tol).nan_to_num(1e9).max().item():.3f} of the tolerance, first {bad.nonzero()[0].tolist()}"
