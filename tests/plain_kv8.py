"""The 8-bit cache of keys and values in plain torch: its numbers, its pages, attention over it in 64 bits."""
from __future__ import annotations

import math

import torch

LOWEST, HIGHEST = -60, 40
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}       # half a step, relative


def power(e: torch.Tensor) -> torch.Tensor:
    """2^e in 64 bits, exactly."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def quantise(x: torch.Tensor):
    """32-bit rows ``[..., n]`` -> (the values kept, in 64 bits; scale bytes; number bytes)."""
    assert x.dtype == torch.float32
    amax = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
    m, e = torch.frexp(amax.double())                                  # 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e - 9 + (m > 0.875).to(e.dtype), torch.full_like(e, LOWEST)).clamp(LOWEST, HIGHEST)
    y = x.double() / power(e).unsqueeze(-1)
    y = torch.where(torch.isfinite(x), y.clamp(-448, 448), torch.full_like(y, math.nan))
    codes = y.float().to(torch.float8_e4m3fn)                          # (y has at most 24 bits: nothing is lost on the way)
    return codes.double() * power(e).unsqueeze(-1), (e + 127).to(torch.uint8), codes.view(torch.uint8)


def rotate(qk: torch.Tensor, cos_sin: torch.Tensor, pairing: int) -> torch.Tensor:
    """32-bit heads ``[T, h, hd]`` turned step by step in 32 bits; ``cos_sin [T, hd/2, 2]``."""
    half = qk.shape[-1] // 2
    a, b = (qk[..., :half], qk[..., half:]) if pairing == 0 else (qk[..., 0::2], qk[..., 1::2])
    if cos_sin is None:
        ra, rb = a, b
    else:
        c, s = cos_sin[:, None, :, 0], cos_sin[:, None, :, 1]
        ra, rb = a * c - b * s, a * s + b * c
    return torch.stack([ra, rb], -1).flatten(2) if pairing == 1 else torch.cat([ra, rb], -1)


def page_bytes(nkv: int, P: int, hd: int) -> int:
    return -(-2 * nkv * P * (hd + 1) // 16) * 16


def split(pages: torch.Tensor, nkv: int, P: int, hd: int):
    """Views: numbers ``[pages, 2, nkv, P, hd]`` and scale bytes ``[pages, 2, nkv, P]``."""
    n = 2 * nkv * P * hd
    return pages[:, :n].unflatten(1, (2, nkv, P, hd)), pages[:, n:n + 2 * nkv * P].unflatten(1, (2, nkv, P))


def case(seqs, nh, nkv, hd, P, dtype, seed, sequential=False, freed_before=None, spread=0.0, junk=True):
    """Queries and an 8-bit cache for sequences given as (keys, rows): ``keys`` and ``values`` hold what the cache stands for.
    ``spread``: powers of two by which tokens' keys and values differ.  What no row was written to is junk, NaN among it."""
    g = torch.Generator().manual_seed(seed)
    blocks = [-(-c // P) for c, _ in seqs]
    total = sum(blocks) + 3
    perm = list(range(total - 1, -1, -1)) if sequential else torch.randperm(total, generator=g).tolist()
    pages = torch.randint(0, 256, (total, page_bytes(nkv, P, hd)), generator=g, dtype=torch.uint8)
    data, scale = split(pages, nkv, P, hd)
    if not junk:
        pages.zero_()
    table = torch.full((len(seqs), max(blocks)), -1, dtype=torch.int32)
    keys, values, rows_q, token_seq, positions, start = [], [], [], [], [], [0]
    for s, (ctx, n) in enumerate(seqs):
        kept = []
        for _ in range(2):
            x = torch.randn(ctx, nkv, hd, generator=g)
            x = x * torch.exp2(torch.round(spread * torch.randn(ctx, nkv, 1, generator=g)))
            kept.append(quantise(x))
        for j in range(blocks[s]):
            page, m = perm.pop(), min(P, ctx - j * P)
            if freed_before and j * P + P <= freed_before[s]:
                continue
            table[s, j] = page
            for w in range(2):
                data[page, w, :, :m] = kept[w][2][j * P:j * P + m].transpose(0, 1)
                scale[page, w, :, :m] = kept[w][1][j * P:j * P + m].transpose(0, 1)
        keys.append(kept[0][0])
        values.append(kept[1][0])
        rows_q.append(torch.randn(n, nh, hd, generator=g).to(dtype))
        token_seq += [s] * n
        positions += list(range(ctx - n, ctx))
        start.append(start[-1] + n)
    ints = lambda v: torch.tensor(v, dtype=torch.int32)   # noqa: E731
    return dict(q=torch.cat(rows_q).reshape(-1, nh * hd), pages=pages, table=table, token_seq=ints(token_seq),
                positions=ints(positions), seq_start=ints(start), keys=keys, values=values, query_lens=[n for _, n in seqs],
                heads=(nh, nkv, hd, P), dtype=dtype)


def attend(c, scale: float, window: int = 0, weights_step: float = 0.0):
    """(outputs in 64 bits ``[T, nh*hd]``, how far each may be off).

    The bound, number by number, for a kernel that forms scores and sums in 32 bits and rounds its weights by at most ``weights_step``
    of themselves: a score is off by at most ds = (hd + 8) 2^-24 scale sum|q k| + 2^-22 |score| (the sum's roundings; the exponent's
    argument); a weight by exp(ds) - 1 and 2^-21 (the exponential) and ``weights_step``; their sums by (keys + 8) 2^-24 of what they add up;
    the quotient then by twice that of sum p|v| / sum p, and the result's own rounding by half a step of its type."""
    nh, nkv, hd, P = c["heads"]
    outs, offs, row = [], [], 0
    for s, n in enumerate(c["query_lens"]):
        k, v = c["keys"][s], c["values"][s]
        L = k.shape[0]
        q = c["q"][row:row + n].double().view(n, nh, hd)
        pos = c["positions"][row:row + n].long()
        at = torch.arange(L)
        there = (c["table"][s, at // P] >= 0)
        seen = (at <= pos[:, None]) & there
        if window:
            seen &= at > pos[:, None] - window
        o, f = torch.zeros(n, nh, hd, dtype=torch.float64), torch.zeros(n, nh, hd, dtype=torch.float64)
        for h in range(nh):
            kh, vh = k[:, h // (nh // nkv)], v[:, h // (nh // nkv)]
            dot = q[:, h] @ kh.T * scale
            ds = (hd + 8) * 2.0 ** -24 * scale * (q[:, h].abs() @ kh.abs().T) + 2.0 ** -22 * dot.abs()
            ds = torch.where(seen, ds, torch.zeros_like(ds))
            masked = dot.masked_fill(~seen, -1e300)
            p = torch.softmax(masked, -1) * seen
            # p (exp(ds) - 1), in a form that holds where p is below the smallest number; results and bound lie among the values
            grown = (torch.exp((torch.log_softmax(masked, -1) + ds).clamp(max=50)) - p).clamp(min=0) * seen
            each = grown + p * (2.0 ** -21 + weights_step + (L + 8) * 2.0 ** -24)
            o[:, h] = p @ vh
            f[:, h] = torch.minimum(each @ vh.abs() + each.sum(-1, keepdim=True) * (p @ vh.abs()), 2 * vh.abs().amax(0))
        outs.append(o.flatten(1))
        offs.append(f.flatten(1))
        row += n
    o, f = torch.cat(outs), torch.cat(offs)
    return o, f + STEP[c["dtype"]] * o.abs() + 1e-30
