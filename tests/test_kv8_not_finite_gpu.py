"""The 8-bit cache where keys or values are not finite: they reach the rows that see them, and no other, whatever kernel runs."""
import pytest
import torch

import plain_kv8 as plain
from test_kv8_gpu import WEIGHTS, ops, portions, run   # noqa: F401

pytestmark = pytest.mark.gpu

DECODE = [(700, 1), (129, 1), (64, 1), (300, 1), (1, 1)]
MIXED = [(700, 1), (900, 120), (300, 300), (64, 2), (333, 40), (77, 1), (2, 2)]


def spoil(c, places):
    """NaN into the cache at (sequence, key, KV head, channel or None: all, 0: the key, 1: the value)."""
    nh, nkv, hd, P = c["heads"]
    data, _ = plain.split(c["pages"], nkv, P, hd)
    for i, (s, key, head, channel, w) in enumerate(places):
        at = slice(None) if channel is None else channel
        page = int(c["table"][s, key // P])
        assert page >= 0
        data[page, w, head, key % P, at] = 0x7f if i % 2 else 0xff
        (c["keys"], c["values"])[w][s][key, head, at] = 0.0


def expected(c, scale, window, places):
    """(outputs in 64 bits, how far they may be off, which of them are NaN)."""
    want, off = plain.attend(c, scale, window, WEIGHTS if c["dtype"] == torch.bfloat16 else 0.0)
    nh, nkv, hd, P = c["heads"]
    nan = torch.zeros(len(want), nh, hd, dtype=torch.bool)
    for s, key, head, channel, w in places:
        for r in range(len(want)):
            pos = int(c["positions"][r])
            if int(c["token_seq"][r]) == s and key <= pos and (not window or key > pos - window):
                heads = slice(head * (nh // nkv), (head + 1) * (nh // nkv))
                nan[r, heads, slice(None) if channel is None or w == 0 else channel] = True
    return want, off, nan.flatten(1)


def check(ops, c, window, places):   # noqa: F811
    spoil(c, places)
    want, off, nan = expected(c, 0.09, window, places)
    assert bool(nan.any()) and not bool(nan.all())
    got = run(ops, c, 0.09, window)
    assert torch.equal(torch.isnan(got), nan)
    assert float(((got - want).abs() / off)[~nan].max()) <= 1.0


def places_of(seqs, nkv, hd, w):
    """The newest row's; one between; one behind the windows below; whole rows and single channels."""
    out = []
    for s, (keys, n) in enumerate(seqs):
        if s % 3 == 2:
            continue                                       # (some sequences stay whole)
        for key, channel in ((keys - 1, s % hd), (max(keys - n // 2 - 1, 0), hd - 1), (max(keys - 150, 0), None if s % 2 else 7)):
            out.append((s, key, (s + key) % nkv, channel, w))
    return out


SHAPES = [(8, 2, 128, 16), (4, 4, 64, 8), (16, 1, 128, 64), (128, 1, 64, 256), (6, 3, 48, 4), (3, 1, 32, 8)]


@pytest.mark.usefixtures("portions")
@pytest.mark.parametrize("w", [0, 1], ids=["keys", "values"])
@pytest.mark.parametrize("nh,nkv,hd,P", SHAPES)
@pytest.mark.parametrize("seqs", [DECODE, MIXED], ids=["decode", "mixed"])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_reach_the_rows_that_see_them(ops, w, nh, nkv, hd, P, seqs, window, dtype):   # noqa: F811
    c = plain.case(seqs, nh, nkv, hd, P, dtype, seed=hd + w)
    check(ops, c, window, places_of(seqs, nkv, hd, w))


@pytest.mark.parametrize("query_tiles,slices", [(1, 1), (1, 2), (1, 4), (1, 8), (2, 1), (2, 2), (2, 4), (2, 8)])
@pytest.mark.parametrize("nh,nkv,hd,P", SHAPES[:4])
@pytest.mark.parametrize("window", [0, 100])
def test_in_any_cut_of_portions(ops, query_tiles, slices, nh, nkv, hd, P, window, monkeypatch):   # noqa: F811
    from allpaca_b200.ops import kv8
    monkeypatch.setattr(kv8, "plan_portions", lambda lens, per_tile, *a: (
        query_tiles, sum(-(-n // (query_tiles * per_tile)) for n in lens), slices))
    monkeypatch.setattr(kv8, "rows_are_faster", lambda *a: False)
    for seqs in ([(1500, 2), (700, 70), (129, 129), (1, 1), (2000, 300)], [(257, 2), (40, 40)]):
        c = plain.case(seqs, nh, nkv, hd, P, torch.bfloat16, seed=slices)
        check(ops, c, window, places_of(seqs, nkv, hd, 1))


def test_every_value(ops):   # noqa: F811
    """All values of a sequence: its rows are NaN, its neighbours' are as without it."""
    seqs = [(300, 200), (500, 60), (90, 90)]
    for window in (0, 50):
        c = plain.case(seqs, 8, 2, 128, 16, torch.bfloat16, seed=1)
        check(ops, c, window, [(1, key, head, None, 1) for key in range(500) for head in range(2)])


def test_a_key_that_a_page_given_back_held(ops):   # noqa: F811
    """NaN in a page that is no longer the sequence's is nobody's."""
    c = plain.case([(900, 120), (300, 70)], 8, 2, 128, 16, torch.bfloat16, seed=4, freed_before=[600, 0])
    gone = torch.ones(c["pages"].shape[0], dtype=torch.bool)
    gone[c["table"][c["table"] >= 0].long()] = False
    c["pages"][gone] = 0x7f
    check(ops, c, 0, [(0, 899, 1, 3, 1), (1, 250, 0, None, 1)])


@pytest.mark.parametrize("every", [1, 128])
@pytest.mark.parametrize("window", [0, 1000])
def test_a_long_portion_full_of_them(ops, every, window):   # noqa: F811
    """Every value, or one column of every 128th key: a result for every row, in a bounded time."""
    nh, nkv, hd, P, rows, keys = 8, 2, 128, 16, 2048, 10240
    g = torch.Generator().manual_seed(1)
    pages = keys // P
    cache = torch.randint(0, 120, (pages, ops.kv8_page_bytes(nkv, P, hd)), generator=g, dtype=torch.uint8)
    data, scale = plain.split(cache, nkv, P, hd)
    scale.fill_(119)
    if every == 1:
        data[:, 1] = 0x7f
    else:
        data[::every // P, 1, :, 3, 77] = 0xff              # keys 3, 131, 259 ...
    args = [t.cuda() for t in (cache, torch.arange(pages).int().view(1, -1), torch.zeros(rows, dtype=torch.int32),
                               torch.arange(keys - rows, keys).int())]
    q = torch.randn(rows, nh * hd, generator=g).bfloat16().cuda()
    out = torch.zeros_like(q)
    kw = dict(seq_start=torch.tensor([0, rows], dtype=torch.int32, device="cuda"), query_lens=[rows], contexts=[keys])
    times = []
    for _ in range(3):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        ops.attention_kv8(q, out, *args, nh, nkv, hd, P, 0.05, window, **kw)
        end.record()
        torch.cuda.synchronize()
        times.append(start.elapsed_time(end))
    ops.check_kernel_status()
    nan = torch.isnan(out.view(rows, nh, hd)).cpu()
    want = torch.ones_like(nan)
    if every > 1:
        want[:, :, :] = torch.arange(hd) == 77
    assert torch.equal(nan, want)
    assert min(times) < 100, times
