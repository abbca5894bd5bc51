"""Attention over the 8-bit cache where keys and values differ in size by tens of powers of two and the scores stay moderate, so that weights of
all sizes meet values of all sizes and a result says something about each."""
import math

import pytest
import torch

import plain_kv8 as plain
from test_kv8_gpu import DECODE, WEIGHTS, ops, portions, run   # noqa: F401

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("portions")]


def spread_case(seqs, nh, nkv, hd, P, dtype, seed, keys, values):
    """Keys of up to 2^keys and down to 2^-60 of that, none so large that a score passes some tens; values whose size grows and falls by
    2^values or more along a sequence, in step with weights that do the opposite."""
    c = plain.case(seqs, nh, nkv, hd, P, dtype, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    c["q"] = (c["q"].float() * 2.0 ** -keys * 3).to(dtype)
    data, scale = plain.split(c["pages"], nkv, P, hd)
    row = 0
    for s, (ctx, n) in enumerate(seqs):
        k = torch.randn(ctx, nkv, hd, generator=g) * torch.exp2(keys - torch.randint(0, 2, (ctx, nkv, 1), generator=g)
                                                               * torch.randint(0, 60, (ctx, nkv, 1), generator=g).float())
        # the score that the sequence's last row gives each key, in powers of two: the value shrinks by as much, or nearly so
        q = c["q"][row + n - 1].float().view(nkv, nh // nkv, hd)[:, 0]
        bits = torch.einsum("lkd,kd->lk", k, q) / math.sqrt(hd) * math.log2(math.e)
        size = torch.round(values * torch.sin(torch.arange(ctx) * 0.37 + seed))[:, None] * (torch.rand(ctx, 1, generator=g) < 0.2) - torch.round(bits)
        v = torch.randn(ctx, nkv, hd, generator=g).abs() * torch.exp2(size)[..., None] * torch.where(torch.arange(hd) % 2 == 0, 1.0, -1.0)
        for w, x in ((0, k), (1, v)):
            kept, byte, code = plain.quantise(x.contiguous())
            (c["keys"], c["values"])[w][s] = kept
            for j in range(-(-ctx // P)):
                m = min(P, ctx - j * P)
                data[int(c["table"][s, j]), w, :, :m] = code[j * P:j * P + m].transpose(0, 1)
                scale[int(c["table"][s, j]), w, :, :m] = byte[j * P:j * P + m].transpose(0, 1)
        row += n
    return c


def weights_floor(c, scale):
    """How much further the bfloat16 kernel for single rows may be off, by the numbers that its weights are held in.

    A weight times its value's scale, W_j = p_j 2^(b_j), is held as w = 2^8 W_j / R in two e4m3 numbers, hi + lo / 16, against a reference R no
    less than any W of the key's 32 (neighbours from a multiple of 32 on).  |w - hi| is at most 2^-4 w, or 2^-10 below 2^-6; lo is
    16 (w - hi) within 2^-4 of itself, or within 2^-10 below 2^-6.  So w is off by at most 2^-8 of itself (which the other bound counts) or by
    2^-10 / 16 = 2^-14, and W_j by 2^-22 R.  R is at most 2^4 of the 32 keys' largest W, or 2^-30 of the row's largest.  The value's
    numbers are v_j / 2^(b_j), so the sum of 2^-18 W_max(32 of j) |v_j| / 2^(b_j) bounds it all, with 2^-52 W_max for the rest."""
    nh, nkv, hd, P = c["heads"]
    _, scales = plain.split(c["pages"], nkv, P, hd)
    outs, row = [], 0
    for s, n in enumerate(c["query_lens"]):
        k, v = c["keys"][s], c["values"][s]
        L = k.shape[0]
        at = torch.arange(L)
        bits = scales[c["table"][s, at // P].long(), 1, :, at % P].to(torch.int64) - 127                      # [L, nkv]
        seen = at <= c["positions"][row:row + n].long()[:, None]
        q = c["q"][row:row + n].double().view(n, nh, hd)
        out = torch.zeros(n, nh, hd, dtype=torch.float64)
        for h in range(nh):
            g = h // (nh // nkv)
            p = torch.softmax((q[:, h] @ k[:, g].T * scale).masked_fill(~seen, -1e300), -1) * seen
            unit = plain.power(bits[:, g])
            pad = torch.zeros(n, -L % 32, dtype=torch.float64)
            W = torch.cat([p * unit, pad], 1).view(n, -1, 32).amax(-1).repeat_interleave(32, 1)[:, :L]
            out[:, h] = ((2.0 ** -18 * W + 2.0 ** -52 * W.amax(-1, keepdim=True)) * seen) @ (v[:, g].abs() / unit[:, None])
        outs.append(out.flatten(1))
        row += n
    return torch.cat(outs)


def expectation(c):
    hd = c["heads"][2]
    half = c["dtype"] == torch.bfloat16
    want, off = plain.attend(c, 1.0 / math.sqrt(hd), 0, WEIGHTS if half else 0.0)
    if half:
        off = off + weights_floor(c, 1.0 / math.sqrt(hd))
    # the bound says something: zeros, the wrong sign, a tenth more all fail
    assert float((off < 0.1 * want.abs()).double().mean()) > 0.95
    return want, off


SHAPES = [(8, 2, 128, 16), (8, 8, 64, 16), (6, 3, 48, 4), (16, 1, 128, 64)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("keys,values", [(0, 3), (0, 30), (-40, 12), (25, 30)])
@pytest.mark.parametrize("seqs", [DECODE, [(700, 300), (65, 65)], [(2100, 1), (1900, 20)]], ids=["decode", "portions", "long"])
def test_values_and_keys_of_unequal_size(ops, dtype, keys, values, seqs):   # noqa: F811
    for shape in SHAPES:
        c = spread_case(seqs, *shape, dtype, 5, keys, values)
        want, off = expectation(c)
        got = run(ops, c, 1.0 / math.sqrt(shape[2]))
        assert float(((got - want).abs() / off).max()) <= 1.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 2])
@pytest.mark.parametrize("where", [0, 1, 777, 69999])
def test_one_key_far_above_many(ops, dtype, n, where):   # noqa: F811
    """A key that takes nearly all of the softmax, whose value is small in half of its columns: there the sum of 70000 weights, each
    2^-23 of the largest, is what counts."""
    nh, nkv, hd, P = 4, 1, 64, 64
    ctx = 70000 + n - 1
    c = plain.case([(ctx, n)], nh, nkv, hd, P, dtype, seed=where)
    data, scale = plain.split(c["pages"], nkv, P, hd)
    g = torch.Generator().manual_seed(1)
    c["q"] = torch.zeros_like(c["q"])
    c["q"].view(n, nh, hd)[:, :, 0] = 8.0
    k = torch.zeros(ctx, nkv, hd)
    k[:, :, 1:] = torch.randn(ctx, nkv, hd - 1, generator=g)
    k[where, :, 0] = 16.0                                       # a score of 16, so exp(16) = 2^23 of the others' weight
    v = 1.0 + 0.25 * torch.randn(ctx, nkv, hd, generator=g)
    v[where] = torch.where(torch.arange(hd) % 2 == 0, 1.0, 2.0 ** -8)
    for w, x in ((0, k), (1, v)):
        kept, byte, code = plain.quantise(x.contiguous())
        (c["keys"], c["values"])[w][0] = kept
        for j in range(-(-ctx // P)):
            m = min(P, ctx - j * P)
            data[int(c["table"][0, j]), w, :, :m] = code[j * P:j * P + m].transpose(0, 1)
            scale[int(c["table"][0, j]), w, :, :m] = byte[j * P:j * P + m].transpose(0, 1)
    want, off = expectation(c)
    assert float(want[0, 1]) > 1.5 * 2.0 ** -8                  # (the many are more than the one here)
    assert float(((run(ops, c, 1.0 / math.sqrt(hd)) - want).abs() / off).max()) <= 1.0
