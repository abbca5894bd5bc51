"""The operators of the 8-bit cache as they are used: one after the other, captured, on several streams, in padded batches."""
import math

import pytest
import torch

import plain_kv8 as plain
from test_kv8_gpu import DECODE, WEIGHTS, dev, ops, portions, run   # noqa: F401

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("portions")]


def rows_of(seqs):
    """Positions and sequences of the rows that sequences of (keys, rows) bring, and where each begins."""
    pos = torch.cat([torch.arange(c - n, c) for c, n in seqs]).int()
    seq = torch.repeat_interleave(torch.arange(len(seqs)), torch.tensor([n for _, n in seqs])).int()
    return pos, seq, torch.tensor([0] + torch.tensor([n for _, n in seqs]).cumsum(0).tolist()).int()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh,nkv,hd,P,pairing", [(8, 2, 128, 16, 2), (4, 4, 64, 8, 0), (6, 2, 96, 7, 1)])
def test_a_conversation(ops, dtype, nh, nkv, hd, P, pairing):   # noqa: F811
    """Prompts are stored and attend, then tokens come one by one through one captured graph whose rows change behind it (a sequence
    ends meanwhile: its row goes on as padding), then everything is read back."""
    g = torch.Generator().manual_seed(hd)
    prompts, steps, ends = [150, 61, 1], 24, 9
    blocks = -(-(max(prompts) + steps) // P)
    table = torch.randperm(3 * blocks + 2, generator=g)[:3 * blocks].view(3, blocks).int()
    cache = torch.randint(0, 256, (3 * blocks + 2, ops.kv8_page_bytes(nkv, P, hd)), generator=g, dtype=torch.uint8).cuda()
    width, scale = (nh + 2 * nkv) * hd, 0.7 / math.sqrt(hd)
    keys, values = ([torch.zeros(0, nkv, hd, dtype=torch.float64) for _ in prompts] for _ in range(2))

    def step_inputs(seqs):
        pos, seq, start = rows_of(seqs)
        x = torch.randn(len(pos), width, generator=g).to(dtype)
        turn = torch.randn(len(pos), hd // 2, generator=g)
        return x, torch.stack([turn.cos(), turn.sin()], -1), pos, seq, start

    def expect(x, cos_sin, pos, seq, seqs):
        heads = x.float().view(len(pos), nh + 2 * nkv, hd)
        qk = plain.rotate(heads[:, :nh + nkv], cos_sin, pairing)
        for i in range(len(prompts)):
            mine = seq == i
            keys[i] = torch.cat([keys[i], plain.quantise(qk[mine][:, nh:].contiguous())[0]])
            values[i] = torch.cat([values[i], plain.quantise(heads[mine][:, nh + nkv:].contiguous())[0]])
        c = dict(q=qk[:, :nh].flatten(1).to(dtype), table=table, positions=pos, keys=keys, values=values,
                 query_lens=[int((seq == i).sum()) for i in range(len(prompts))], heads=(nh, nkv, hd, P), dtype=dtype)
        return plain.attend(c, scale, 0, WEIGHTS if dtype == torch.bfloat16 else 0.0)

    def near(got, want, off):
        assert float(((got.cpu().double() - want).abs() / off).max()) <= 1.0

    seqs = [(n, n) for n in prompts]
    x, cs, pos, seq, start = step_inputs(seqs)
    q = torch.empty((len(pos), nh * hd), dtype=dtype, device="cuda")
    out = torch.empty_like(q)
    dtable = dev(table)
    ops.rope_kv8_store(dev(x), q, cache, dev(pos), dev(seq), dtable, dev(cs), pairing, nh, nkv, hd, P)
    ops.attention_kv8(q, out, cache, dtable, dev(seq), dev(pos), nh, nkv, hd, P, scale, seq_start=dev(start), query_lens=prompts)
    near(out, *expect(x, cs, pos, seq, seqs))

    # one graph for all steps: its buffers are filled anew before every replay
    gx, gcs = torch.zeros((3, width), dtype=dtype, device="cuda"), torch.zeros((3, hd // 2, 2), device="cuda")
    gpos, gseq = (torch.full((3,), -1, dtype=torch.int32, device="cuda") for _ in range(2))
    gq, gout = (torch.zeros((3, nh * hd), dtype=dtype, device="cuda") for _ in range(2))
    gstart = torch.arange(4, dtype=torch.int32, device="cuda")
    kept = {}

    def scratch(name, shape, t):
        return kept.setdefault(name, torch.full(shape, float("nan"), dtype=t, device="cuda"))

    def step():
        ops.rope_kv8_store(gx, gq, cache, gpos, gseq, dtable, gcs, pairing, nh, nkv, hd, P)
        ops.attention_kv8(gq, gout, cache, dtable, gseq, gpos, nh, nkv, hd, P, scale, seq_start=gstart, query_lens=[1, 1, 1],
                          max_context=blocks * P, scratch=scratch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    lens = list(prompts)
    for n in range(steps):
        live = [i for i in range(3) if not (i == 1 and n >= ends)]
        x, cs, _, _, _ = step_inputs([(lens[i] + 1, 1) for i in range(3)])
        pos = torch.tensor([lens[i] if i in live else -1 for i in range(3)], dtype=torch.int32)
        seq = torch.tensor([i if i in live else -1 for i in range(3)], dtype=torch.int32)
        for to, what in ((gx, x), (gcs, cs), (gpos, pos), (gseq, seq)):
            to.copy_(what)
        gout.fill_(float("nan"))
        graph.replay()
        rows = torch.tensor(live)
        near(gout.cpu()[rows], *expect(x[rows], cs[rows], pos[rows], seq[rows], None))
        assert bool((gout.cpu()[[i for i in range(3) if i not in live]] == 0).all())
        for i in live:
            lens[i] += 1
    pos, seq, _ = rows_of([(n, n) for n in lens])
    k, v = (torch.empty((len(pos), nkv * hd), device="cuda") for _ in range(2))
    ops.kv8_read(cache, dev(pos), dev(seq), dtable, k, v, nkv, hd, P)
    assert torch.equal(k.cpu().double(), torch.cat(keys).flatten(1)) and torch.equal(v.cpu().double(), torch.cat(values).flatten(1))
    ops.check_kernel_status()


def arguments(c):
    nh, nkv, hd, P = c["heads"]
    q = dev(c["q"])
    return q, torch.zeros_like(q), dev(c["pages"]), dev(c["table"]), dev(c["token_seq"]), dev(c["positions"]), nh, nkv, hd, P, 0.1


@pytest.mark.parametrize("seqs", [DECODE, [(3000, 1)], [(700, 1)] * 40, [(900, 120), (300, 300)], [(2000, 9)]],
                         ids=["ragged", "long", "many", "portions", "few rows"])
def test_the_same_bits_every_time_and_on_two_streams(ops, seqs):   # noqa: F811
    c = plain.case(seqs, 8, 2, 128, 16, torch.bfloat16, seed=2)
    kw = dict(seq_start=dev(c["seq_start"]), query_lens=c["query_lens"])
    args = arguments(c)
    ops.attention_kv8(*args, **kw)
    want = args[1].clone()
    outs = [torch.zeros_like(want) for _ in range(40)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        with torch.cuda.stream(streams[i % 2]):
            ops.attention_kv8(args[0], out, *args[2:], **kw)
    torch.cuda.synchronize()
    ops.check_kernel_status()
    for out in outs:
        assert torch.equal(out, want)


def test_two_graphs_on_one_scratch(ops):   # noqa: F811
    """Captured calls of different shapes that share a workspace, replayed in any order."""
    kept = {}

    def scratch(name, shape, t):
        if name not in kept or kept[name].numel() < math.prod(shape):
            kept[name] = torch.full((max(math.prod(shape), 1 << 22),), float("nan"), dtype=t, device="cuda")
        return kept[name][:math.prod(shape)].view(shape)
    calls = []
    for n, seqs in enumerate(([(3000, 1)] * 3, [(1500, 1)] * 60, [(800, 100), (40, 40)], [(2500, 1)] * 7)):
        c = plain.case(seqs, 8, 2, 64, 16, torch.bfloat16, seed=n)
        args, kw = arguments(c), dict(seq_start=dev(c["seq_start"]), query_lens=c["query_lens"], scratch=scratch)
        ops.attention_kv8(*args, **kw)
        want = args[1].clone()
        calls.append((args, kw, want))
    graphs = []
    for args, kw, want in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            ops.attention_kv8(*args, **kw)
    for i in (0, 1, 2, 3, 3, 0, 0, 2, 1, 2, 3, 1, 0):
        calls[i][0][1].fill_(float("nan"))
        graphs[i].replay()
        assert torch.equal(calls[i][0][1], calls[i][2])
    ops.check_kernel_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_are_not_there(ops, dtype):   # noqa: F811
    """Rows without a sequence or a position, and what lies behind the last row."""
    for nh, nkv, hd, P in ((8, 2, 128, 16), (4, 4, 64, 5)):
        c = plain.case([(100, 1)] * 6, nh, nkv, hd, P, dtype, seed=3)
        want, off = plain.attend(c, 0.1, 0, WEIGHTS if dtype == torch.bfloat16 else 0.0)
        q, _, pages, table, seq, pos, *rest = arguments(c)
        seq[1], seq[2], pos[3], seq[4] = -1, 6, -1, 2 ** 31 - 1
        big, out = (torch.full((9, nh * hd), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        big[:6] = q
        ops.attention_kv8(big, out, pages, table, seq, torch.cat([pos, pos]), *rest)
        got = out.cpu().double()
        assert bool((got[1:5] == 0).all()) and bool((got[6:] == 7).all())
        for r in (0, 5):
            assert float(((got[r] - want[r]).abs() / off[r]).max()) <= 1.0
    ops.check_kernel_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_positions_past_the_block_table(ops, dtype):   # noqa: F811
    """A row past the last page that its table names sees all keys there are."""
    for seqs in ([(96, 1), (96, 1)], [(96, 40), (96, 3)]):
        c = plain.case(seqs, 4, 2, 64, 16, dtype, seed=4)
        last = torch.tensor([c["query_lens"][0] - 1, -1])
        want, off = plain.attend(c, 0.1, 0, WEIGHTS if dtype == torch.bfloat16 else 0.0)
        args = list(arguments(c))
        # (rows of a sequence follow one another in their positions: all of them move)
        args[5] = args[5] + 96
        ops.attention_kv8(*args, seq_start=dev(c["seq_start"]), query_lens=c["query_lens"])
        got = args[1].cpu().double()
        assert float(((got[last] - want[last]).abs() / off[last]).max()) <= 1.0
    ops.check_kernel_status()


def test_many_rows(ops):   # noqa: F811
    """More single rows than one launch takes, several of a sequence, in no order; and more rows than sequences in a table."""
    c = plain.case([(70, 70), (300, 300), (1, 1), (600, 230)], 8, 2, 64, 16, torch.bfloat16, seed=6)
    want, off = plain.attend(c, 0.1, 0, WEIGHTS)
    order = torch.randperm(len(c["token_seq"]), generator=torch.Generator().manual_seed(1))
    args = list(arguments(c))
    for i in (0, 4, 5):
        args[i] = args[i][order.cuda()].contiguous()
    ops.attention_kv8(*args)
    assert float(((args[1].cpu().double() - want[order]).abs() / off[order]).max()) <= 1.0
    twice = torch.cat([order[:5], order[:5]])                    # the same row twice
    args = list(arguments(c))
    for i in (0, 4, 5):
        args[i] = args[i][twice.cuda()].contiguous()
    out = torch.zeros_like(args[0])
    ops.attention_kv8(args[0], out, *args[2:])
    assert torch.equal(out[:5], out[5:])
    ops.check_kernel_status()


@pytest.mark.parametrize("scale", [0.0, -0.1, 8.0])
def test_any_scale(ops, scale):   # noqa: F811
    for seqs in (DECODE, [(300, 40), (129, 129)]):
        for dtype in (torch.bfloat16, torch.float32):
            c = plain.case(seqs, 8, 2, 64, 16, dtype, seed=7)
            want, off = plain.attend(c, abs(scale), 0, WEIGHTS if dtype == torch.bfloat16 else 0.0)
            if scale < 0:                                        # the same as turning the queries round
                c["q"] = -c["q"]
            got = run(ops, c, scale)
            assert float(((got - want).abs() / off).max()) <= 1.0


def test_queries_that_are_not_finite(ops):   # noqa: F811
    """They spoil their own row and head, no other."""
    for seqs in (DECODE, [(300, 40), (129, 129)]):
        for dtype in (torch.bfloat16, torch.float32):
            c = plain.case(seqs, 8, 2, 64, 16, dtype, seed=8)
            want, off = plain.attend(c, 0.1, 0, WEIGHTS if dtype == torch.bfloat16 else 0.0)
            q = c["q"].view(-1, 8, 64)
            q[2, 3, 5], q[0, 1, 0] = math.nan, math.nan
            got = run(ops, c, 0.1).view(-1, 8, 64)
            bad = torch.isnan(got).all(-1)
            assert bad[2, 3] and bad[0, 1] and int(torch.isnan(got).any(-1).sum()) == 2
            near = (got - want.view_as(got)).abs() / off.view_as(got)
            assert float(near[~bad].max()) <= 1.0


def test_long_tables(ops):   # noqa: F811
    """A table that names far more pages than a sequence has: what lies behind its rows is never looked at."""
    c = plain.case([(50, 1), (700, 1)], 8, 2, 128, 16, torch.bfloat16, seed=9)
    p = plain.case([(50, 50), (700, 65)], 8, 2, 128, 16, torch.bfloat16, seed=9)
    for case in (c, p):
        wide = torch.full((2, 5000), 2 ** 31 - 1, dtype=torch.int32)
        wide[:, :case["table"].shape[1]] = torch.where(case["table"] < 0, 2 ** 31 - 1, case["table"])
        case["table"], narrow = wide, case["table"]
        got = run(ops, case, 0.1)
        case["table"] = narrow
        want, off = plain.attend(case, 0.1, 0, WEIGHTS)
        assert float(((got - want).abs() / off).max()) <= 1.0


@pytest.mark.parametrize("seqs", [[(50, 0), (90, 2)], [(90, 2), (40, 0), (70, 1)], [(64, 1), (30, 0), (200, 70)], [(30, 0), (70, 1), (65, 1)]])
def test_sequences_that_bring_nothing(ops, seqs):   # noqa: F811
    for dtype in (torch.bfloat16, torch.float32):
        c = plain.case(seqs, 8, 2, 64, 16, dtype, seed=10)
        want, off = plain.attend(c, 0.1, 0, WEIGHTS if dtype == torch.bfloat16 else 0.0)
        assert float(((run(ops, c, 0.1) - want).abs() / off).max()) <= 1.0
