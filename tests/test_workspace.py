"""The named buffers of an engine: which replacements end a recorded step's life, and how buffers grow."""
import torch

from allpaca_b200.parts import Workspace


def test_only_buffers_that_a_recorded_step_holds_count():
    ws = Workspace(torch.device("cpu"))
    ws.get("a", (4,), torch.float32)
    ws.get("b", (4,), torch.float32)
    ws.get("a", (4,), torch.bfloat16)
    ws.recording = True
    ws.get("a", (2, 2), torch.float32)
    ws.get("a", (4,), torch.float32)                       # (the view that was handed out before)
    ws.recording = False
    before = ws.generation
    ws.get("b", (400,), torch.float32)                     # held by no graph
    ws.get("a", (400,), torch.bfloat16)                    # a buffer of its own
    ws.get("c", (7,), torch.float32)
    ws.get("a", (3,), torch.float32)                       # fits
    assert ws.generation == before
    ws.get("a", (5,), torch.float32)
    assert ws.generation > before
    # one that comes to be while a step is recorded
    ws.recording = True
    ws.get("d", (5,), torch.float32)
    ws.recording = False
    before = ws.generation
    ws.get("d", (6,), torch.float32)
    assert ws.generation > before


def test_a_buffer_that_grows_step_by_step():
    """64 requests, each a portion larger than the last, replace a few buffers and hold less than twice what is asked."""
    ws = Workspace(torch.device("meta"))
    held, replaced, asked = None, 0, 0
    for i in range(1, 65):
        n = i * 2 ** 20 + 64
        view = ws.grow("a", (n,), torch.bfloat16)
        assert view.shape == (n,)
        if ws._buffers["a:torch.bfloat16"] is not held:
            held, replaced, asked = ws._buffers["a:torch.bfloat16"], replaced + 1, asked + ws.bytes()
        assert ws.bytes() < 2 * 2 * n
    assert replaced <= 7 and asked < 2 * ws.bytes()
    assert ws.grow("a", (5, 3), torch.bfloat16).shape == (5, 3) and ws._buffers["a:torch.bfloat16"] is held
    # far more at once: as much as is asked
    ws.grow("a", (2 ** 30,), torch.bfloat16)
    assert ws.bytes() == 2 ** 31


def test_the_engines_long_prompt(monkeypatch):
    """A prompt of 32768 tokens in portions of 512 over the 8-bit cache: the mixer's buffer of widened keys is replaced a few times."""
    from allpaca_b200.engine.batch import StepBatch
    from allpaca_b200.parts import BuildEnv, LayerCache, PartSpec, attention, build
    env = BuildEnv(torch.bfloat16, torch.device("meta"), Workspace(torch.device("meta")), kv_dtype="fp8")
    mixer = build("mixer", PartSpec("gqa_attention", {"hidden_size": 64, "num_heads": 32, "num_kv_heads": 8, "head_dim": 128}), env)

    def kernel(*a, scratch, contexts, **kw):
        scratch("attn.kv8_wide", (contexts[0] * 2 * 8 * 128,), torch.bfloat16)
    monkeypatch.setattr(attention.ops, "attention_kv8", kernel)
    seen = []
    for at in range(0, 32768, 512):
        none = torch.zeros(512, dtype=torch.int32)
        step = StepBatch(512, 1, 0, none, none, none, none, none, none, none, [none], host_first_position=[at],
                         host_query_lens=[512], max_query_len=512)
        mixer._attention(torch.zeros(1), 512, step, LayerCache(group=0), env.workspace)
        buf = env.workspace._buffers["attn.kv8_wide:torch.bfloat16"]
        if not seen or seen[-1] is not buf:
            seen.append(buf)
    assert len(seen) <= 8
    assert sum(b.numel() for b in seen) <= 4 * 32768 * 2 * 8 * 128
