"""CPU restatement, in float64, of the 4-bit K/V cache (test oracle).

TEST INFRASTRUCTURE ONLY -- see ``oracle/__init__.py``.

The package's format (``include/loopfuse_b200.h``): groups of 64 dims, ``low = min x``,
``s = bf16((max - low) / 15)``, ``n = rint((x - low) / s)``, value ``n * s + low``; a page of one KV
head is ``18 * D`` bytes.  ``pack`` / ``unpack`` move codes one by one by the header's formulas.
"""
from __future__ import annotations

import math
from typing import List, Tuple

import torch

PAGE, GROUP = 16, 64


def quantise(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(codes int64 [..., D], s [..., D/64], low [..., D/64])`` (float64) of ``x [..., D]``."""
    g = x.double().unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1), g.amax(-1)
    span = (high - low).float()
    bad = ~(span < 2.0 ** 60) | torch.isnan(g).any(-1)
    s = (span.double() / 15).to(torch.bfloat16).double()
    n = ((g - low[..., None]) / torch.where(s > 0, s, torch.ones_like(s))[..., None]).round()
    n = torch.where((s > 0)[..., None] & ~bad[..., None], n.clamp(0, 15), torch.zeros_like(n))
    nan = torch.full_like(s, math.nan)
    return (torch.nan_to_num(n).long().flatten(-2), torch.where(bad, nan, s), torch.where(bad, nan, low))


def value(n: torch.Tensor, s: torch.Tensor, low: torch.Tensor) -> torch.Tensor:
    """Values (float64) the codes stand for."""
    return (n.unflatten(-1, (-1, GROUP)).double() * s[..., None] + low[..., None]).flatten(-2)


def places(D: int):
    """Byte offset and bit shift in a block of every K code and V code, each ``[16, D]``."""
    ng = D // GROUP
    t, d = torch.arange(PAGE)[:, None], torch.arange(D)[None, :]
    e = d % 8
    bit = 4 * (e // 2) + 16 * (e % 2) + 0 * t
    k_at = t * 32 * ng + (d % 64 // 16) * 8 * ng + (d // 64) * 8 + (d % 16 // 8) * 4 + bit // 8
    v_at = 8 * D + (t // 8) * 256 * ng + ((d % 64 // 8) * 4 + t % 8 // 2) * 8 * ng + (d // 64) * 8 \
        + (d % 8 // 4) * 4 + (t % 2) * 2 + d % 4 // 2
    return (k_at, bit % 8), (v_at, 4 * (d % 2) + 0 * t)


def write_token(pages: torch.Tensor, page: int, head: int, tok: int, k: torch.Tensor, v: torch.Tensor) -> None:
    """Quantise one token's ``k, v [D]`` into ``pages [P, Hkv, 18 * D]`` (uint8, CPU) in place."""
    D = k.shape[-1]
    ng = D // GROUP
    blk = pages[page, head]
    for which, (x, (at, up)) in enumerate(zip((k, v), places(D))):
        n, s, low = quantise(x)
        for d in range(D):
            a, u = int(at[tok, d]), int(up[tok, d])
            blk[a] = (int(blk[a]) & ~(15 << u) & 255) | (int(n[d]) << u)
        par = torch.stack([s, low], -1).to(torch.bfloat16).contiguous().view(torch.uint8).flatten()
        p0 = 16 * D + (tok * 2 + which) * ng * 4
        blk[p0:p0 + 4 * ng] = par


def unpack(pages: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``k, v [..., 16, D]`` (float64) of blocks ``[..., 18 * D]`` and V's ``s * |n - 8|``."""
    D = pages.shape[-1] // 18
    ng = D // GROUP
    par = pages[..., 16 * D:].contiguous().view(torch.bfloat16).double().unflatten(-1, (PAGE, 2, ng, 2))
    out = []
    for which, (at, up) in enumerate(places(D)):
        n = (pages[..., at].long() >> up) & 15
        s, low = par[..., which, :, 0], par[..., which, :, 1]
        out.append(value(n, s, low))
    spread = ((n - 8).abs().unflatten(-1, (ng, GROUP)).double() * s[..., None]).flatten(-2)
    return out[0], out[1], spread


def decode(q: torch.Tensor, pages: torch.Tensor, table: torch.Tensor, lens: List[int], scale: float):
    """``o [N, Hq, D]``, ``lse [N, Hq]`` and a bound on the kernel's error of each, float64.

    The bound counts: o's rounding to bf16 (half a step, 2^-8); the rounding of ``p s`` to bf16,
    which multiplies ``n - 8`` (2^-8 of ``sum p s |n - 8|``); the scores' fp32 sums of products
    ``q n s`` and of ``b sum(q)``, seven additions of magnitude at most ``(15 s + |b|) sum |q|`` with
    2^-22 each (truncating accumulators; where a long prefix is taken in tiles, 17 additions of 2^-23, half
    of them while the sum is still growing: 13.5 of 2^-23); fp32 exponentials and sums (2^-20 of ``sum p |v|``)."""
    N, Hq, D = q.shape
    Hkv = pages.shape[1]
    G, ng = Hq // Hkv, D // GROUP
    o = torch.zeros(N, Hq, D, dtype=torch.float64)
    lse = torch.full((N, Hq), -math.inf, dtype=torch.float64)
    tol_o, tol_l = torch.zeros_like(o), torch.zeros_like(lse)
    for i, L in enumerate(lens):
        if L == 0:
            continue
        blk = pages[table[i, :-(-L // PAGE)].long()]
        k, v, spread = (x.transpose(1, 2).reshape(-1, Hkv, D)[:L] for x in unpack(blk))
        par = blk[..., 16 * D:].contiguous().view(torch.bfloat16).double().unflatten(-1, (PAGE, 2, ng, 2))[..., 0, :, :]
        par = par.transpose(1, 2).reshape(-1, Hkv, ng, 2)[:L]
        most = 15 * par[..., 0] + par[..., 1].abs()
        for h in range(Hq):
            x = q[i, h].double()
            sc = scale * (k[:, h // G] @ x)
            size = (most[:, h // G] * x.abs().unflatten(0, (ng, GROUP)).sum(-1)).sum(-1).max()
            delta = float(abs(scale) * 7 * 2 ** -22 * size) + 2 ** -21
            lse[i, h] = torch.logsumexp(sc, 0)
            p = torch.softmax(sc, 0)
            o[i, h] = p @ v[:, h // G]
            around = p @ v[:, h // G].abs()
            tol_o[i, h] = 2 ** -8 * o[i, h].abs() + 2 ** -8 * (p @ spread[:, h // G]) * (1 + 2 ** -6) \
                + (2 * delta + 2 ** -20) * around + 1e-30
            tol_l[i, h] = 2 * delta + 2 ** -22 * lse[i, h].abs()
    return o, lse, tol_o, tol_l
