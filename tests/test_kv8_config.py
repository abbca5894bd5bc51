"""The 8-bit cache where there is no GPU: its settings, its memory, its refusals."""
import pytest
import torch

import plain_kv8
from allpaca_b200 import ops
from allpaca_b200.config import EngineConfig
from allpaca_b200.config.model_config import ConfigError
from allpaca_b200.parts import BuildEnv, KV8Need, KVNeed, PartError, Workspace, build, PartSpec


def test_settings():
    cfg = EngineConfig()
    cfg.validate()
    assert cfg.kv_dtype == "auto"
    for name in ("fp8", "fp8_e4m3", torch.float8_e4m3fn):
        cfg = EngineConfig(kv_dtype=name)
        cfg.validate()
        assert cfg.kv_dtype == "fp8"
    with pytest.raises(ConfigError):
        EngineConfig(kv_dtype="int4").validate()


def test_pages():
    assert ops.kv8_page_bytes(8, 16, 128) == 2 * 8 * 16 * 129
    assert ops.kv8_page_bytes(1, 5, 16) == 176                     # 170 bytes, padded
    for nkv, P, hd in ((8, 16, 128), (1, 5, 16), (3, 4, 48), (1, 1, 256)):
        assert ops.kv8_page_bytes(nkv, P, hd) == plain_kv8.page_bytes(nkv, P, hd)
        need = KV8Need(num_kv_heads=nkv, head_dim=hd)
        assert need.page_shape(P) == (ops.kv8_page_bytes(nkv, P, hd),)
        assert need.page_bytes(P, torch.bfloat16) == ops.kv8_page_bytes(nkv, P, hd)
    assert KV8Need(num_kv_heads=2, head_dim=64) != KV8Need(num_kv_heads=2, head_dim=32)
    eight, sixteen = KV8Need(num_kv_heads=8, head_dim=128), KVNeed(8, 128)
    assert eight.page_bytes(16, torch.bfloat16) * 1.98 < sixteen.page_bytes(16, torch.bfloat16)


def test_the_mixer_asks_for_it():
    spec = PartSpec("gqa_attention", {"hidden_size": 64, "num_heads": 4, "num_kv_heads": 2, "head_dim": 16, "window": 32})
    for kv, kind in (("auto", False), ("fp8", True)):
        env = BuildEnv(torch.float32, torch.device("cpu"), Workspace(torch.device("cpu")), kv_dtype=kv)
        need = build("mixer", spec, env).cache_need()
        assert isinstance(need, KV8Need) is kind and need.window == 32


def test_head_sizes_that_no_kernel_takes():
    env = BuildEnv(torch.float32, torch.device("cpu"), Workspace(torch.device("cpu")), kv_dtype="fp8")
    for hd in (24, 272):
        with pytest.raises(PartError):
            build("mixer", PartSpec("gqa_attention", {"hidden_size": 64, "num_heads": 4, "num_kv_heads": 2, "head_dim": hd}), env)


def test_plans():
    """Work is cut into no more pieces than there are, and every sequence's rows find a CTA."""
    from allpaca_b200.ops import kv8
    fits = ((1, 148), (2, 74), (4, 33), (8, 15), (16, 7))
    for pairs in (1, 7, 8, 15, 16, 33, 74, 148, 149, 512, 4096):
        for longest in (1, 2, 5, 64, 1000):
            for mean in {1, max(1, longest // 3), longest}:
                ctas, cluster = kv8.plan_rows(pairs, longest, mean, 148, fits)
                assert 1 <= ctas and (ctas <= 148 if cluster == 0 else ctas == pairs * cluster and pairs <= dict(fits)[cluster])
    for lens in ([2], [1, 1, 5], [0, 7], [2048], [17] * 40, [600, 3], [31, 32, 33, 64, 65]):
        for per_tile in (1, 8, 32, 128):
            for keys in (0, 100, 5000, 100000):
                tiles, ctas, slices = kv8.plan_portions(lens, per_tile, 8, keys, 148)
                assert tiles in (1, 2) and slices in (1, 2, 4, 8) and ctas == sum(-(-n // (tiles * per_tile)) for n in lens)
                assert slices == 1 or ctas * 8 * slices <= 148


def test_no_cpu_branch():
    cache = torch.zeros((1, ops.kv8_page_bytes(2, 16, 64)), dtype=torch.uint8)
    one, table = torch.zeros(1, dtype=torch.int32), torch.zeros((1, 1), dtype=torch.int32)
    q = torch.zeros((1, 256))
    with pytest.raises(ops.KernelError):
        ops.rope_kv8_store(torch.zeros((1, 512)), q, cache, one, one, table, None, 0, 4, 2, 64, 16)
    with pytest.raises(ops.KernelError):
        ops.kv8_read(cache, one, one, table, q, q, 2, 64, 16)
    with pytest.raises(ops.KernelError):
        ops.attention_kv8(q, q, cache, table, one, one, 4, 2, 64, 16, 1.0)


def test_the_plain_numbers():
    """The plain quantiser against the definition, number by number."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(64, 32, generator=g) * torch.exp2(torch.randint(-50, 30, (64, 1), generator=g).float())
    kept, byte, _ = plain_kv8.quantise(x)
    scale = plain_kv8.power(byte.to(torch.int64) - 127)
    top = x.abs().amax(1).double()
    assert bool((top <= 448 * scale).all()) and bool((top > 448 * scale / 2).all())
    off = (kept - x.double()).abs()
    assert bool((off <= torch.maximum(x.double().abs() * 2.0 ** -4, scale[:, None] * 2.0 ** -10)).all())
