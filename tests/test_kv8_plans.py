"""What a step over the 8-bit cache is planned by, where there is no GPU: the entry points are recorded, not called."""
import types

import pytest
import torch

from allpaca_b200.ops import kv8

HEADS = (32, 8, 128, 16)          # query heads, KV heads, head size, page size


class Library:
    """Stands in for the kernels' library on a device of 148 SMs."""
    ap_attention_kv8_decode_takes = staticmethod(lambda P: 1)
    ap_attention_kv8_decode_scratch = staticmethod(lambda nh, nkv, ctas: 1024)
    ap_attention_kv8_decode_clusters = staticmethod(lambda nh, nkv, c: {1: 148, 2: 74, 4: 33, 8: 15, 16: 7}[c])
    ap_attention_kv8_tcgen05_takes = staticmethod(lambda nh, nkv, hd, P: 1)
    ap_attention_kv8_tcgen05_tokens = staticmethod(lambda nh, nkv: 128 // (nh // nkv))
    ap_attention_kv8_tcgen05_scratch = staticmethod(lambda tiles, nkv: tiles * nkv * (4 * 128 * HEADS[2] + 4))


@pytest.fixture
def step(monkeypatch):
    """step(seqs of (keys, rows), ...) -> [(entry point, how it is planned)]."""
    caches = [kv8._machine, kv8._single_rows_taken, kv8._portions_taken, kv8._scratch_bytes, kv8._row_by_row, kv8._portions_plan]
    for f in caches:
        f.cache_clear()
    calls, planned = [], []
    rows_cost, plan_portions = kv8._rows_cost, kv8.plan_portions

    def rows(pairs, longest, mean, *more):
        planned.append((longest * 64, mean * 64))
        return rows_cost(pairs, longest, mean, *more)

    def portions(lens, per_tile, nkv, keys, sms):
        planned.append((keys, plan_portions(lens, per_tile, nkv, keys, sms)))
        return planned[-1][1]
    monkeypatch.setattr(kv8, "library", types.SimpleNamespace(attention=lambda hd: Library))
    monkeypatch.setattr(kv8, "_sms", lambda device: 148)
    monkeypatch.setattr(kv8, "stream_handle", lambda: 0)
    monkeypatch.setattr(kv8, "call", lambda lib, name, *a: calls.append((name, planned[-1])))
    monkeypatch.setattr(kv8, "_rows_cost", rows)
    monkeypatch.setattr(kv8, "plan_portions", portions)
    monkeypatch.setattr(kv8, "_take_cache", lambda what, cache, nkv, hd, P, pos, seq, table: (
        -1, seq.shape[0], (0, cache.shape[0], cache.shape[1]), (0, table.shape[1], table.shape[0])))

    def run(seqs, **more):
        nh, nkv, hd, P = HEADS
        del calls[:], planned[:]
        for f in caches:                                   # (a plan that was made before is not made again)
            f.cache_clear()
        T, lens = sum(n for _, n in seqs), [n for _, n in seqs]
        ints = lambda n: torch.zeros(n, dtype=torch.int32)   # noqa: E731
        q = torch.zeros((T, nh * hd), dtype=torch.bfloat16)
        table = torch.zeros((len(seqs), max(-(-c // P) for c, _ in seqs)), dtype=torch.int32)
        kv8.attention_kv8(q, torch.zeros_like(q), torch.zeros((1, 16), dtype=torch.uint8), table, ints(T), ints(T), nh, nkv, hd, P, 0.1,
                          seq_start=ints(len(seqs) + 1), query_lens=lens, **more)
        return list(calls)
    yield run
    for f in caches:
        f.cache_clear()


PORTIONS, ROWS = "ap_attention_kv8_tcgen05", "ap_attention_kv8_decode"


def contexts(seqs):
    return [c for c, _ in seqs]


def test_a_one_row_sequence_behind_a_portion(step):
    """17 rows behind 30000 keys are far faster as portions; that the row behind them has ten keys changes nothing, whatever
    the caller says of the longest one-row sequence."""
    alone = step([(30017, 17)], max_context=30017)
    assert alone[0][0] == PORTIONS and alone[0][1][1][2] == 8
    seqs = [(30017, 17), (10, 1)]
    for more in ({}, {"contexts": contexts(seqs)}):
        (name, (keys, plan)), = step(seqs, max_context=10, mean_context=10, **more)
        assert name == PORTIONS and keys > 29000 and plan[2] == 8
    # more rows: their plan has key slices as well
    (name, (keys, plan)), = step([(30512, 512), (10, 1)], max_context=10, mean_context=10, contexts=[30512, 10])
    alone = step([(30512, 512)], max_context=30512)[0][1][1]
    assert name == PORTIONS and keys > 29000 and alone[2] > 1 and plan == (alone[0], alone[1] + 1, alone[2])   # (one CTA for the row behind)


def test_a_long_decoded_row_in_front_of_short_portions(step):
    """One row of 131072 keys: the portions behind it are planned by their own keys, not by the block table's width."""
    seqs = [(131072, 1), (317, 17)]
    got = step(seqs, max_context=131072, mean_context=131072, contexts=contexts(seqs))
    assert [name for name, _ in got] == [ROWS]                         # 17 rows behind 300 keys go row by row
    longest, mean = got[0][1]
    assert longest >= 131072 and mean < 8000                           # eighteen rows, one of them long
    seqs = [(131072, 1), (512, 512), (400, 400)]
    got = step(seqs, max_context=131072, mean_context=131072, contexts=contexts(seqs))
    assert [name for name, _ in got] == [PORTIONS, ROWS]
    assert got[0][1] == step(seqs[1:], max_context=512)[0][1]
    assert got[1][1] == step(seqs[:1], max_context=131072)[0][1]


def test_without_contexts(step):
    """Portions alone are planned by max_context, or by the block table's width."""
    assert step([(2512, 512)], max_context=2512) == step([(2512, 512)]) == step([(2512, 512)], contexts=[2512])
    (_, (keys, _)), = step([(2512, 512), (90000, 600)], max_context=2512)
    assert keys < 2512
    (_, (keys, _)), = step([(2512, 512), (90000, 1)], max_context=2512)
    assert keys > 80000


def test_contexts_that_do_not_fit(step):
    from allpaca_b200.ops import KernelError
    with pytest.raises(KernelError):
        step([(50, 2), (60, 1)], contexts=[50])


def test_the_engine_says_how_long_its_sequences_are(monkeypatch):
    """A step with portions names every sequence's keys; one of single rows leaves them out."""
    from allpaca_b200.engine.batch import StepBatch
    from allpaca_b200.parts import BuildEnv, LayerCache, PartSpec, Workspace, attention, build
    seen = []
    monkeypatch.setattr(attention.ops, "attention_kv8", lambda *a, **kw: seen.append(kw["contexts"]))
    env = BuildEnv(torch.bfloat16, torch.device("cpu"), Workspace(torch.device("cpu")), kv_dtype="fp8")
    mixer = build("mixer", PartSpec("gqa_attention", {"hidden_size": 64, "num_heads": 4, "num_kv_heads": 2, "head_dim": 16}), env)
    for firsts, lens, want in (([40, 0, 7], [1, 30, 5], [41, 30, 12]), ([40, 8], [1, 1], None)):
        T = sum(lens)
        none = torch.zeros(T, dtype=torch.int32)
        step = StepBatch(T, len(lens), 0, none, none, none, none, none, none, none, [none], host_first_position=firsts,
                         host_query_lens=lens, max_query_len=max(lens))
        mixer._attention(torch.zeros(T, 64, dtype=torch.bfloat16), T, step, LayerCache(group=0), env.workspace)
        assert seen.pop() == want


def wide_scratch(step, seqs, **more):
    """Bytes of scratch that a step's portions ask for."""
    asked = []

    def scratch(name, shape, dtype):
        if name == "attn.kv8_wide":
            asked.append(shape[0] * dtype.itemsize)
        return torch.empty(0, dtype=dtype)
    step(seqs, scratch=scratch, **more)
    return asked[0] if asked else 0


TOKEN = 2 * 8 * 128 * 2            # bytes of a token's keys and values, widened


def test_scratch_is_for_the_portions_own_keys(step):
    """Not for the widest block table of the step."""
    alone = wide_scratch(step, [(600, 512), (400, 400)], contexts=[600, 400])
    assert 2 * 600 * TOKEN <= alone <= 2 * 640 * TOKEN * 1.01
    seqs = [(131072, 1), (600, 512), (400, 400)]
    assert wide_scratch(step, seqs, contexts=contexts(seqs)) == alone


def test_twelve_prompts_beside_a_long_conversation_go_together(step):
    seqs = [(131072, 1)] + [(600 - i, 600 - i) for i in range(12)]
    assert [name for name, _ in step(seqs, contexts=contexts(seqs))] == [PORTIONS, ROWS]


def test_scratch_of_a_window(step):
    """512 rows behind 100000 keys see 512 + 1024 of them."""
    seqs = [(100512, 512)]
    assert wide_scratch(step, seqs, window=1024, contexts=contexts(seqs)) <= (512 + 1024 + 256) * TOKEN * 1.01
    assert wide_scratch(step, seqs, window=1024) <= (512 + 1024 + 256) * TOKEN * 1.01
    assert wide_scratch(step, seqs, contexts=contexts(seqs)) >= 100512 * TOKEN


def test_dense_tiles_hold_what_the_rows_see():
    for window in (1, 2, 64, 127, 128, 129, 500):
        for rows in (1, 2, 100, 128, 129):
            for keys in [k for k in (1, 2, 127, 128, 129, 700, 1000, 1023, 1024, 1025) if k >= rows]:
                first = max(keys - rows - window + 1, 0)
                assert (keys - 1) // 128 - first // 128 + 1 <= kv8.dense_tiles(rows, keys, window) <= -(-keys // 128)
                assert kv8.dense_tiles(rows, keys, 0) == -(-keys // 128)


def test_groups_of_portions():
    lens, keys = [100] * 5, [128, 1280, 128, 12800, 128]
    assert kv8.group_portions(lens, keys, 0, 10 ** 6) == [(0, 5, 100)]
    assert kv8.group_portions(lens, keys, 0, 30) == [(0, 3, 10), (3, 4, 100), (4, 5, 1)]
    assert kv8.group_portions(lens, keys, 0, 0) == [(i, i + 1, k // 128) for i, k in enumerate(keys)]
    assert kv8.group_portions([0, 3], [1, 3], 0, 10) == [(0, 2, 1)]


def test_the_most_scratch(step):
    """No step of an engine asks for more than portions_scratch_bytes."""
    import random
    r = random.Random(2)
    for i in range(60):
        window, n, tokens = r.choice((0, 0, 700)), r.randint(1, 24), r.choice((3000, 40000, 131072))
        seqs = []
        for _ in range(n):
            keys = r.randint(2, tokens)
            seqs.append((keys, min(keys, r.randint(2, 2048 // n))))
        most = kv8.portions_scratch_bytes(8, 128, tokens, 2048, 24, window)
        asked = wide_scratch(step, seqs, window=window, contexts=contexts(seqs))
        assert asked <= most <= max(131072 * TOKEN * 1.01, kv8.WIDE_SCRATCH)
    assert kv8.portions_scratch_bytes(8, 96, 131072, 2048, 24) == 0


def test_pages_leave_room_for_it(monkeypatch):
    """An engine that plans its pages by the free memory keeps what portions of the longest sequence need."""
    from allpaca_b200.config import EngineConfig
    from allpaca_b200.engine.runner import ModelRunner
    from allpaca_b200.models.decoder import CacheGroupPlan
    from allpaca_b200.parts import KV8Need, KVNeed
    free = 8 << 30
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (free, free))
    for need, kv_dtype, room in ((KV8Need(num_kv_heads=8, head_dim=128), "fp8", 2 * 131072 * TOKEN), (KVNeed(8, 128), "auto", 0),
                                 (KV8Need(num_kv_heads=8, head_dim=96), "fp8", 0)):
        plan = [CacheGroupPlan(need, [0])]
        runner = types.SimpleNamespace(
            engine=EngineConfig(dtype=torch.bfloat16, kv_dtype=kv_dtype, page_size=16, max_num_seqs=10 ** 6), max_model_len=131072,
            device=torch.device("meta"), model=types.SimpleNamespace(cache_plan=lambda: plan, state_bytes=lambda: [0],
                                                                     bind_caches=lambda *a: None))
        ModelRunner._setup_caches(runner)
        pages = runner.num_pages * need.page_bytes(16, torch.bfloat16)
        assert free * 0.85 - pages >= room and (room or free * 0.85 - pages < 1 << 20)


@pytest.mark.parametrize("hd", [64, 128, 80])
def test_block_tables_whose_keys_an_index_cannot_hold(hd):
    """The entry points refuse tables that name nearly 2^31 keys or more (checked before anything is launched: no rows here)."""
    from allpaca_b200.ops import library
    lib, nkv = library.attention(hd), 1
    entry = lib.ap_attention_kv8_rows
    for P, blocks, fine in ((16, 1 << 20, True), (1, 2 ** 31 - 1, False), (16, (1 << 27) - 1, False), (1, 2 ** 31 - 1 - 512, True),
                            (2 ** 30, 1, True), (2 ** 30, 2, False)):
        rc = entry(0, 0, 1, 0, 1, kv8.kv8_page_bytes(nkv, P, hd), 0, blocks, 1, 0, 0, 0, 2, nkv, hd, P, 0.1, 0, 0)
        assert (rc == 0) is fine, (P, blocks)
