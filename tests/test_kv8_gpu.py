"""The 8-bit cache of keys and values: what is stored, what comes back, attention over it, each against 64 bits."""
import math

import pytest
import torch

import plain_kv8 as plain

pytestmark = pytest.mark.gpu

# heads, KV heads, head size, page size
SHAPES = [(4, 2, 16, 16), (3, 1, 32, 8), (6, 3, 48, 4), (8, 8, 64, 16), (8, 2, 128, 16), (5, 1, 80, 32), (20, 1, 16, 16),
          (32, 8, 128, 16), (16, 2, 64, 128), (4, 1, 256, 5), (40, 2, 64, 64), (16, 1, 128, 1)]
# (keys, rows): single rows, portions, both, lengths at tiles' and pages' edges
DECODE = [(700, 1), (129, 1), (64, 1), (1, 1), (65, 1), (33, 1), (32, 1), (1500, 1)]
MIXED = [(700, 1), (300, 1), (1, 1), (129, 129), (64, 2), (333, 40), (77, 1), (65, 65), (2, 2)]


@pytest.fixture(scope="module")
def ops():
    from allpaca_b200 import ops as o
    return o


@pytest.fixture(params=["by rule", "tensor cores"])
def portions(request, monkeypatch):
    """Portions by the kernel that the rule names, then all by the one for portions, however small."""
    from allpaca_b200.ops import kv8
    if request.param == "tensor cores":
        monkeypatch.setattr(kv8, "rows_are_faster", lambda *a: False)


def dev(t):
    return t.to("cuda") if t is not None else None


def store_case(T, nh, nkv, hd, P, dtype, slices, seed, blocks=3):
    """Rows of two sequences at scattered positions, each with a page of its own place."""
    g = torch.Generator().manual_seed(seed)
    width = (nh + 2 * nkv) * hd
    x = torch.randn(slices, T, width, generator=g) * torch.exp2(torch.randint(-3, 4, (slices, T, 1), generator=g).float())
    qkv = x if slices > 1 else x[0].to(dtype)
    blocks = max(blocks, -(-T // P))
    seq = torch.randint(0, 2, (T,), generator=g)
    pos = torch.stack([torch.randperm(blocks * P, generator=g)[:T] for _ in range(2)])[seq, torch.arange(T)]
    table = torch.randperm(2 * blocks, generator=g).view(2, blocks)
    turn = torch.randn(T, hd // 2, generator=g)
    return (qkv, pos.int(), seq.int(), table.int(), torch.stack([turn.cos(), turn.sin()], -1), 2 * blocks)


def kept_rows(qkv, cos_sin, pairing, nh, nkv, hd):
    x = qkv.float()
    if x.dim() == 3:
        y = x[0]
        for i in range(1, x.shape[0]):
            y = y + x[i]
        x = y
    x = x.view(x.shape[0], nh + 2 * nkv, hd)
    return plain.rotate(x[:, :nh + nkv], cos_sin, pairing), x[:, nh + nkv:]


@pytest.mark.parametrize("nh,nkv,hd,P", SHAPES)
@pytest.mark.parametrize("T", [1, 7, 200])
@pytest.mark.parametrize("pairing", [0, 1, 2])
@pytest.mark.parametrize("dtype,slices", [(torch.bfloat16, 1), (torch.float32, 1), (torch.bfloat16, 3)])
def test_store_gives_the_formulas_bytes(ops, nh, nkv, hd, P, T, pairing, dtype, slices):
    qkv, pos, seq, table, cos_sin, pages = store_case(T, nh, nkv, hd, P, dtype, slices, seed=hd + T)
    cache = torch.full((pages, ops.kv8_page_bytes(nkv, P, hd)), 77, dtype=torch.uint8, device="cuda")
    q = torch.full((T, nh * hd), float("nan"), dtype=dtype, device="cuda")
    ops.rope_kv8_store(dev(qkv), q, cache, dev(pos), dev(seq), dev(table), dev(cos_sin), pairing, nh, nkv, hd, P)
    qk, v = kept_rows(qkv, cos_sin, pairing, nh, nkv, hd)
    assert torch.equal(q.cpu(), qk[:, :nh].flatten(1).to(dtype))
    want = torch.full((pages, ops.kv8_page_bytes(nkv, P, hd)), 77, dtype=torch.uint8)
    data, scale = plain.split(want, nkv, P, hd)
    page, slot = table.long()[seq.long(), pos.long() // P], pos.long() % P
    for w, x in enumerate((qk[:, nh:], v)):
        _, byte, code = plain.quantise(x.contiguous())
        data[page, w, :, slot] = code
        scale[page, w, :, slot] = byte
    got, got_scale = plain.split(cache.cpu(), nkv, P, hd)
    assert torch.equal(got_scale, scale)
    assert torch.equal(torch.where(got == 128, 0, got), torch.where(data == 128, 0, data))       # (-0 and 0 are one number)
    assert torch.equal(cache.cpu()[:, 2 * nkv * P * (hd + 1):], want[:, 2 * nkv * P * (hd + 1):])
    for out in (torch.float32, torch.bfloat16):
        k, vv = (torch.empty((T, nkv * hd), dtype=out, device="cuda") for _ in range(2))
        ops.kv8_read(cache, dev(pos), dev(seq), dev(table), k, vv, nkv, hd, P)
        for got, x in ((k, qk[:, nh:]), (vv, v)):
            assert torch.equal(got.cpu().double(), plain.quantise(x.contiguous())[0].flatten(1))


def test_rows_of_zeros_extremes_and_what_is_not_finite(ops):
    nh, nkv, hd, P = 2, 1, 64, 8
    x = torch.randn(8, 4, hd, generator=torch.Generator().manual_seed(3))
    x[0, 2:] = 0
    x[1, 2:] = 1e-40                       # below the lowest scale: subnormal numbers, then zeros
    x[2, 2:] *= 2.0 ** -70
    x[3, 2:] *= 2.0 ** 100                 # above the highest: the largest numbers
    x[4, 2:, 5] = math.inf
    x[5, 2:, 6] = math.nan
    x[6, 2:] = math.inf
    x[7, 2:, 7] = 448.0 * 2 ** 5           # a row's largest number on the border of two scales
    x = x.flatten(1)
    pos, seq, table = torch.arange(8, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    cache = torch.zeros((1, ops.kv8_page_bytes(nkv, P, hd)), dtype=torch.uint8, device="cuda")
    q = torch.empty((8, nh * hd), device="cuda")
    ops.rope_kv8_store(dev(x), q, cache, dev(pos), dev(seq), dev(table), None, 0, nh, nkv, hd, P)
    k, v = (torch.empty((8, hd), device="cuda") for _ in range(2))
    ops.kv8_read(cache, dev(pos), dev(seq), dev(table), k, v, nkv, hd, P)
    for got, at in ((k, 2), (v, 3)):
        want = plain.quantise(x.view(8, 4, hd)[:, at].contiguous())[0]
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got.cpu().double()), torch.nan_to_num(want))
    assert float(got.cpu()[3].abs().max()) == 448.0 * 2.0 ** 40


def test_rows_without_a_page(ops):
    """Positions and sequences outside the block table, pages given back and ids outside the cache: not kept, read as zeros."""
    nh, nkv, hd, P = 2, 2, 32, 8
    pos = torch.tensor([0, -1, 16, 9, 3, 3, 4], dtype=torch.int32)
    seq = torch.tensor([0, 0, 0, 0, 1, 2, -1], dtype=torch.int32)
    table = torch.tensor([[1, -1], [7, 0]], dtype=torch.int32)       # sequence 1's first page lies outside the cache
    x = torch.randn(7, (nh + 2 * nkv) * hd, generator=torch.Generator().manual_seed(1))
    cache = torch.zeros((2, ops.kv8_page_bytes(nkv, P, hd)), dtype=torch.uint8, device="cuda")
    q = torch.empty((7, nh * hd), device="cuda")
    ops.rope_kv8_store(dev(x), q, cache, dev(pos), dev(seq), dev(table), None, 0, nh, nkv, hd, P)
    assert torch.equal(q.cpu(), x[:, :nh * hd])
    k, v = (torch.full((7, nkv * hd), 5.0, device="cuda") for _ in range(2))
    ops.kv8_read(cache, dev(pos), dev(seq), dev(table), k, v, nkv, hd, P)
    assert int((k != 0).any(1).sum()) == 1 and bool((k[0] != 0).any())
    assert torch.equal(v.cpu()[0].double(), plain.quantise(x[:1, (nh + nkv) * hd:].view(1, nkv, hd).contiguous())[0].flatten())
    data, scale = plain.split(cache.cpu(), nkv, P, hd)
    assert int((scale != 0).sum()) == 2 * nkv                        # one row's scales
    k.fill_(5.0)
    ops.kv8_read(cache, dev(pos), dev(seq), dev(table), k, None, nkv, hd, P)
    assert bool((k[0] != 5).any())


def run(ops, c, scale, window=0, metadata=True, **more):
    nh, nkv, hd, P = c["heads"]
    q = dev(c["q"])
    out = torch.full_like(q, float("nan"))
    kept = []

    def scratch(name, shape, dtype):
        kept.append(torch.full(shape, float("nan"), dtype=dtype, device="cuda"))
        return kept[-1]
    kw = {}
    if metadata:
        held = [k for (k, n) in zip([len(x) for x in c["keys"]], c["query_lens"]) if n == 1]
        kw = dict(seq_start=dev(c["seq_start"]), query_lens=c["query_lens"], max_context=max(held or [1]),
                  mean_context=sum(held) // max(len(held), 1), scratch=scratch)
    ops.attention_kv8(q, out, dev(c["pages"]), dev(c["table"]), dev(c["token_seq"]), dev(c["positions"]), nh, nkv, hd, P, scale,
                      window, **kw, **more)
    ops.check_kernel_status()
    return out.cpu().double()


# what a bfloat16 kernel's weights may be off by before they meet the values: half a step of bfloat16
WEIGHTS = 2.0 ** -8


def check(got, c, scale, window=0):
    want, off = plain.attend(c, scale, window, WEIGHTS if c["dtype"] == torch.bfloat16 else 0.0)
    worst = ((got - want).abs() / off).max()
    assert float(worst) <= 1.0, float(worst)


@pytest.mark.usefixtures("portions")
@pytest.mark.parametrize("nh,nkv,hd,P", SHAPES)
@pytest.mark.parametrize("seqs", [DECODE, MIXED], ids=["decode", "mixed"])
@pytest.mark.parametrize("window", [0, 37, 200])
@pytest.mark.parametrize("dtype,metadata", [(torch.float32, True), (torch.bfloat16, True), (torch.bfloat16, False)])
def test_attention(ops, nh, nkv, hd, P, seqs, window, dtype, metadata):
    c = plain.case(seqs, nh, nkv, hd, P, dtype, seed=hd + P, sequential=P == 64)
    check(run(ops, c, 0.8 / math.sqrt(hd), window, metadata), c, 0.8 / math.sqrt(hd), window)


@pytest.mark.usefixtures("portions")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("spread", [4.0, 12.0])
@pytest.mark.parametrize("seqs", [DECODE, [(700, 300), (65, 65)]], ids=["decode", "portions"])
def test_attention_over_rows_of_unequal_size(ops, dtype, spread, seqs):
    """Keys and values whose sizes differ by many powers of two from token to token: scores of all sizes, weights that matter only
    through their values."""
    for nh, nkv, hd, P in ((8, 2, 128, 16), (8, 8, 64, 16), (6, 3, 48, 4)):
        c = plain.case(seqs, nh, nkv, hd, P, dtype, seed=5, spread=spread)
        c["q"] = (c["q"].float() * 2.0 ** -spread).to(dtype)
        check(run(ops, c, 1.0 / math.sqrt(hd)), c, 1.0 / math.sqrt(hd))


@pytest.mark.usefixtures("portions")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("far", [0, 3, 15, 16, 31, 32, 63, 64, 127, 128, 500, 1023])
def test_finds_one_far_key(ops, dtype, far):
    """One key among a thousand wins the softmax; its value must come out."""
    for hd in (64, 128):
        nh, nkv, P = 4, 2, 16
        for seqs in ([(1024, 1)], [(1024, 5)], [(1024, 100)]):
            c = plain.case(seqs, nh, nkv, hd, P, dtype, seed=far)
            data, scale = plain.split(c["pages"], nkv, P, hd)
            row = c["q"][-1].view(nh, hd)
            k = torch.stack([row[2 * h].float() * 40 / row[2 * h].float().norm() for h in range(nkv)])
            v = torch.stack([torch.full((hd,), 3.0 + h) for h in range(nkv)])
            page = int(c["table"][0, far // P])
            for w, x in ((0, k), (1, v)):
                kept, byte, code = plain.quantise(x)
                data[page, w, :, far % P], scale[page, w, :, far % P] = code, byte
                (c["keys"], c["values"])[w][0][far] = kept
            want, off = plain.attend(c, 1.0, 0, WEIGHTS if dtype == torch.bfloat16 else 0.0)
            assert abs(float(want[-1].view(nh, hd)[0].mean()) - 3.0) < 0.1
            got = run(ops, c, 1.0)
            assert float(((got - want).abs() / off).max()) <= 1.0


@pytest.mark.usefixtures("portions")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("seqs", [[(900, 1), (500, 1), (149, 1)], [(900, 70), (500, 3), (300, 149)]], ids=["decode", "portions"])
def test_pages_given_back(ops, dtype, seqs):
    """Pages behind the window are gone (their ids are -1); then, without a window, rows that see only what is left, or nothing."""
    for nh, nkv, hd, P in ((8, 2, 128, 16), (4, 4, 64, 8), (6, 3, 48, 4)):
        freed = [ctx - n - 150 + 1 for ctx, n in seqs]
        c = plain.case(seqs, nh, nkv, hd, P, dtype, seed=9, freed_before=freed)
        check(run(ops, c, 0.08, 150), c, 0.08, 150)
        c = plain.case(seqs, nh, nkv, hd, P, dtype, seed=9, freed_before=[freed[0], 500 - seqs[1][1] // 2, 10000])
        check(run(ops, c, 0.08), c, 0.08)


def test_no_rows(ops):
    cache = torch.zeros((2, ops.kv8_page_bytes(2, 16, 64)), dtype=torch.uint8, device="cuda")
    none, table = torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    q = torch.zeros((0, 4 * 64), dtype=torch.bfloat16, device="cuda")
    ops.rope_kv8_store(torch.zeros((0, 8 * 64), dtype=torch.bfloat16, device="cuda"), q, cache, none, none, table, None, 0, 4, 2, 64, 16)
    ops.kv8_read(cache, none, none, table, q[:, :128].contiguous(), None, 2, 64, 16)
    ops.attention_kv8(q, torch.zeros_like(q), cache, table, none, none, 4, 2, 64, 16, 1.0)
    assert int(cache.sum()) == 0


def test_refusals(ops):
    nh, nkv, hd, P = 4, 2, 64, 16
    cache = torch.zeros((2, ops.kv8_page_bytes(nkv, P, hd)), dtype=torch.uint8, device="cuda")
    one = torch.zeros(3, dtype=torch.int32, device="cuda")
    table = torch.zeros((3, 1), dtype=torch.int32, device="cuda")
    x = torch.zeros((3, (nh + 2 * nkv) * hd), dtype=torch.bfloat16, device="cuda")
    q = torch.zeros((3, nh * hd), dtype=torch.bfloat16, device="cuda")
    k = torch.zeros((3, nkv * hd), device="cuda")
    E = ops.KernelError

    def bad(call, *args, **kw):
        with pytest.raises(E):
            call(*args, **kw)
    store = ops.rope_kv8_store
    bad(store, x, q, cache.cpu(), one, one, table, None, 0, nh, nkv, hd, P)
    bad(store, x, q, cache.view(torch.int8), one, one, table, None, 0, nh, nkv, hd, P)
    bad(store, x, q, cache, one, one, table, None, 0, nh, nkv, hd, 8)               # another page size
    bad(store, x, q, cache, one, one, table, None, 0, nh, nkv, 72, P)
    bad(store, x, q, cache, one, one, table, None, 3, nh, nkv, hd, P)
    bad(store, x[:2], q, cache, one, one, table, None, 0, nh, nkv, hd, P)
    bad(store, x.half(), q, cache, one, one, table, None, 0, nh, nkv, hd, P)
    bad(store, x, q.float(), cache, one, one, table, None, 0, nh, nkv, hd, P)       # narrower input than the queries
    bad(store, x[None].expand(2, -1, -1).contiguous(), q, cache, one, one, table, None, 0, nh, nkv, hd, P)   # 16-bit slices
    bad(store, x, q, cache, one.long(), one, table, None, 0, nh, nkv, hd, P)
    bad(store, x, q, cache, one[:2], one, table, None, 0, nh, nkv, hd, P)
    bad(store, x, q, cache, one, one, table[:0], None, 0, nh, nkv, hd, P)
    bad(store, x, q, cache, one, one, table, torch.zeros((3, hd, 2), device="cuda"), 0, nh, nkv, hd, P)
    shifted = torch.zeros(cache.numel() + 8, dtype=torch.uint8, device="cuda")[8:].view_as(cache)
    bad(store, x, q, shifted, one, one, table, None, 0, nh, nkv, hd, P)
    bad(ops.kv8_read, cache, one, one, table, k.half(), None, nkv, hd, P)
    bad(ops.kv8_read, cache, one, one, table, k, k.bfloat16(), nkv, hd, P)
    bad(ops.kv8_read, cache, one, one, table, k[:2], None, nkv, hd, P)
    bad(ops.kv8_read, cache, one, one, table, k.cpu(), None, nkv, hd, P)
    att = ops.attention_kv8
    bad(att, q, q[:2], cache, table, one, one, nh, nkv, hd, P, 1.0)
    bad(att, q.half(), q.half(), cache, table, one, one, nh, nkv, hd, P, 1.0)
    bad(att, q, torch.zeros_like(q), cache, table, one, one, nh, 3, hd, P, 1.0)
    bad(att, q, torch.zeros_like(q), cache, table, one, one, nh, nkv, hd, P, 1.0, -1)
    bad(att, q, torch.zeros_like(q), cache, table, one, one, nh, nkv, hd, P, 1.0, seq_start=one, query_lens=[1, 1])
    bad(att, q.float(), torch.zeros_like(q), cache, table, one, one, nh, nkv, hd, P, 1.0)


@pytest.mark.parametrize("ctas,cluster", [(1, 0), (2, 0), (3, 0), (7, 0), (31, 0), (100, 0), (148, 0), (400, 0), (1, 1), (1, 2), (1, 4), (1, 8), (1, 16)])
@pytest.mark.parametrize("nh,nkv,hd,P", [(8, 2, 128, 16), (16, 1, 128, 64), (40, 2, 64, 16), (6, 2, 96, 5), (8, 8, 32, 16), (4, 1, 256, 7)])
def test_any_cut_of_the_work(ops, ctas, cluster, nh, nkv, hd, P, monkeypatch):
    """Runs of tiles that end inside a pair, hold many pairs, or none; pairs cut into many parts; all on scratch full of junk."""
    from allpaca_b200.ops import kv8
    monkeypatch.setattr(kv8, "plan_rows", lambda *a: (ctas, cluster))
    for seqs in (DECODE, [(3000, 1), (700, 9), (333, 5), (3, 3)]):
        c = plain.case(seqs, nh, nkv, hd, P, torch.bfloat16, seed=ctas + hd)
        check(run(ops, c, 0.09), c, 0.09)


@pytest.mark.parametrize("query_tiles,slices", [(1, 1), (1, 2), (1, 4), (1, 8), (2, 1), (2, 2), (2, 4), (2, 8)])
@pytest.mark.parametrize("nh,nkv,hd,P", [(8, 2, 128, 16), (16, 1, 128, 64), (32, 2, 64, 8), (4, 4, 64, 128), (128, 1, 64, 256), (8, 8, 128, 32)])
@pytest.mark.parametrize("window", [0, 100])
def test_portions_on_tensor_cores(ops, query_tiles, slices, nh, nkv, hd, P, window, monkeypatch):
    """Portions of two rows to several CTAs' worth, key slices that hold many tiles, one or none, one-row sequences among them."""
    from allpaca_b200.ops import kv8
    monkeypatch.setattr(kv8, "plan_portions", lambda lens, per_tile, *a: (
        query_tiles, sum(-(-n // (query_tiles * per_tile)) for n in lens), slices))
    monkeypatch.setattr(kv8, "rows_are_faster", lambda *a: False)
    monkeypatch.setattr(kv8, "WIDE_SCRATCH", (1 << 30) if slices < 4 else 1)          # all sequences together, or one by one
    for seqs in ([(1500, 2), (700, 70), (129, 129), (1, 1), (64, 1), (2, 2), (3000, 300)], [(130, 130)], [(257, 2)]):
        c = plain.case(seqs, nh, nkv, hd, P, torch.bfloat16, seed=slices + hd)
        check(run(ops, c, 0.09, window), c, 0.09, window)
