"""The engine with keys and values in 8 bits, against the plain decoder whose keys and values are rounded the same way.

Where the engine's key or value differs from the plain one by a part u of itself before it is rounded, it lands on the other
side of a border between two 8-bit numbers with probability u / h, and is then off by the step h, 2^-4 to 2^-3 of itself: on average
(root of the mean square) by sqrt(u h) = sqrt(u 2^-3.5) of itself at most.  In bfloat16 the plain decoder rounds what the engine
does not, and both round what comes before: u = 2^-8, so numbers of the cache differ by 2^-5.75 = 1.9 %, and logits, sums of many of
them, by as much of their usual size in each of up to three layers, 3.2 % together; the largest of some 500 logits' errors is about 3.1 times
the usual one, as the largest logit is among logits.  With the usual 3e-2 for everything else, in squares, sqrt(3.2^2 + 3^2) = 4.4 %; rows
differ by chance, some by 1.8 times: 8e-2.  (A wrong key, page or scale moves logits by tens of per cent.)  In 32 bits u is below 2^-20 and
sqrt(u h) 0.03 %, so by the same steps 1e-2 is ample."""
import numpy as np
import pytest
import torch

import helpers
import plain_kv8
import plain_llama

pytestmark = pytest.mark.gpu

TOL = {"float32": 1e-2, "bfloat16": 8e-2}
# head size 64 and widths that are multiples of 8: the kernels that serving uses
SERVING = {
    "architectures": ["LlamaForCausalLM"], "model_type": "llama", "hidden_act": "silu",
    "num_hidden_layers": 2, "hidden_size": 256, "num_attention_heads": 8, "num_key_value_heads": 2,
    "head_dim": 64, "intermediate_size": 384, "vocab_size": 311, "rope_theta": 10000.0,
    "rms_norm_eps": 1e-5, "max_position_embeddings": 1024, "tie_word_embeddings": False,
}
CONFIGS = {"A": helpers.TINY_A, "B": helpers.TINY_B, "C": helpers.TINY_C, "S": SERVING,
           "S128": dict(SERVING, head_dim=128, num_attention_heads=4, num_key_value_heads=4)}
LENGTH = {"A": 120, "B": 200, "C": 300, "S": 400, "S128": 300}


@pytest.fixture
def plain_logits(monkeypatch):
    attend = plain_llama.causal_attention

    def rounded(q, k, v, **kw):
        k, v = (plain_kv8.quantise(x.float().contiguous())[0].to(q.dtype) for x in (k, v))
        return attend(q, k, v, **kw)
    monkeypatch.setattr(plain_llama, "causal_attention", rounded)
    return helpers.plain_logits


def make_runner(model, dtype, pages=64, page_size=16, graphs=True, **more):
    from allpaca_b200.config import EngineConfig
    from allpaca_b200.engine.runner import ModelRunner
    return ModelRunner(model, EngineConfig(dtype=dtype, kv_dtype="fp8", page_size=page_size, num_pages=pages, max_num_seqs=4,
                                           max_num_batched_tokens=512, use_cuda_graphs=graphs, **more))


@pytest.mark.parametrize("name", sorted(CONFIGS))
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("page_size", [16, 8])
def test_logits(tmp_path, plain_logits, name, dtype, page_size):
    """Two requests: portions cut anywhere, portions beside decoded rows, decoded rows together (replayed as graphs), on pages that
    were full of NaN bytes."""
    from allpaca_b200 import ops
    from allpaca_b200.engine.batch import BatchEntry
    config, n = CONFIGS[name], LENGTH[name]
    model = helpers.make_model_folder(str(tmp_path / "m"), config, 3, dtype)
    runner = make_runner(model, dtype, pages=1024 // page_size, page_size=page_size)
    for storage in runner.storages:
        assert storage.pages.dtype == torch.uint8
        storage.pages.fill_(0x7f)
    a, b = helpers.random_tokens(n, config["vocab_size"], 1), helpers.random_tokens(n, config["vocab_size"], 2)
    want = {"a": plain_logits(model, a, dtype), "b": plain_logits(model, b, dtype)}

    def check(logits, rows):
        got = logits.double().cpu().numpy()
        for g, (rid, pos) in zip(got, rows):
            ref = want[rid][pos]
            assert abs(g - ref).max() <= TOL[dtype] * abs(ref).max(), (rid, pos)
    check(runner.step([BatchEntry("a", a[:70], [0, 33, 69])]), [("a", 0), ("a", 33), ("a", 69)])
    check(runner.step([BatchEntry("a", a[70:97], [0, 26])]), [("a", 70), ("a", 96)])
    check(runner.step([BatchEntry("a", a[97:98], [0]), BatchEntry("b", b[:80], [0, 79])]), [("a", 97), ("b", 0), ("b", 79)])
    for i in range(12):
        check(runner.step([BatchEntry("a", a[98 + i:99 + i], [0]), BatchEntry("b", b[80 + i:81 + i], [0])]),
              [("a", 98 + i), ("b", 80 + i)])
    assert runner.graph_replays > 0
    runner.finish("a")
    check(runner.step([BatchEntry("c", b[:n - 1], [n - 2])]), [("b", n - 2)])            # on the pages that a gave back
    check(runner.step([BatchEntry("c", b[n - 1:], [0])]), [("b", n - 1)])
    ops.check_kernel_status()


def test_graphs_give_the_same_bits(tmp_path):
    from allpaca_b200.engine.batch import BatchEntry
    model = helpers.make_model_folder(str(tmp_path / "m"), SERVING, 5, "bfloat16")
    tokens = helpers.random_tokens(120, SERVING["vocab_size"], 7)
    got = []
    for graphs in (False, True):
        runner = make_runner(model, "bfloat16", graphs=graphs)
        runner.step([BatchEntry("a", tokens[:100], [99])])
        got.append(np.stack([runner.step([BatchEntry("a", [t], [0])]).cpu().numpy()[0] for t in tokens[100:]]))
        assert (runner.graph_replays > 0) is graphs
    assert np.array_equal(got[0], got[1])


def test_half_the_memory(tmp_path):
    model = helpers.make_model_folder(str(tmp_path / "m"), SERVING, 5, "bfloat16")
    from allpaca_b200.config import EngineConfig
    from allpaca_b200.engine.runner import ModelRunner
    eight = make_runner(model, "bfloat16").memory_report()["cache_bytes"]
    sixteen = ModelRunner(model, EngineConfig(dtype="bfloat16", page_size=16, num_pages=64, max_num_seqs=4,
                                              max_num_batched_tokens=512)).memory_report()["cache_bytes"]
    assert eight * 128 == sixteen * 65                      # 64 numbers of 8 bits and a scale, not 64 of 16


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generation_with_preemption(tmp_path, plain_logits, dtype):
    """Requests that outgrow the pool are preempted and computed again; the tokens chosen are (near) maxima of the plain logits."""
    from allpaca_b200 import LLM, SamplingParams
    model = helpers.make_model_folder(str(tmp_path / "m"), SERVING, 9, dtype)
    llm = LLM(model=model, kv_dtype="fp8", page_size=16, num_pages=11, max_num_seqs=4, max_num_batched_tokens=128, prefill_chunk=40)
    prompts = [helpers.random_tokens(n, SERVING["vocab_size"], n) for n in (61, 17, 44)]
    outs = llm.generate(prompts, SamplingParams(temperature=0.0, max_tokens=30))
    assert llm.stats["preemptions"] > 0
    for p, o in zip(prompts, outs):
        assert len(o.token_ids) == 30
        logits = plain_logits(model, p + o.token_ids, dtype)
        for i, t in enumerate(o.token_ids):
            row = logits[len(p) + i - 1]
            assert row.max() - row[t] <= 2 * TOL[dtype] * abs(row).max()


def test_command_line_and_replay(tmp_path, plain_logits, capsys):
    import json
    from allpaca_b200.cli import main
    model = helpers.make_model_folder(str(tmp_path / "m"), helpers.TINY_A, 0, "float32")
    assert main(["generate", "--model", model, "--kv-dtype", "fp8", "--prompt-ids", "5 17 3", "--max-tokens", "4", "--temperature", "0",
                 "--json"]) == 0
    got = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert len(got["token_ids"]) == 4
    (tmp_path / "t.toml").write_text('[kv]\ndtype = "fp8"\n')
    assert main(["generate", "--model", model, "--config", str(tmp_path / "t.toml"), "--prompt-ids", "5 17 3", "--max-tokens", "4",
                 "--temperature", "0", "--json"]) == 0
    assert json.loads(capsys.readouterr().out.strip().splitlines()[-1]) == got
    tokens = [5, 17, 3, 9]
    out = helpers.run_trace(model, "float32", str(tmp_path / "o"), [{"step": 0, "entries": [{"id": "a", "tokens": tokens, "want": [3]}],
                                                                     "end": ["a"]}], 64, extra=["--kv-dtype", "fp8"])
    want = plain_logits(model, tokens, "float32")[3]
    assert abs(out[0][0] - want).max() <= TOL["float32"] * abs(want).max()


def test_models_that_keep_something_else_are_refused(tmp_path):
    from allpaca_b200.config import EngineConfig
    from allpaca_b200.config.model_config import ConfigError
    from allpaca_b200.engine.runner import ModelRunner
    import test_viresun_engine_gpu as viresun
    from viresun_configs import VIRESUN_A
    viresun.write_folder(tmp_path / "v", VIRESUN_A, 1, "float32")
    with pytest.raises(ConfigError):
        ModelRunner(str(tmp_path / "v"), EngineConfig(dtype="float32", kv_dtype="fp8", num_pages=8, max_num_seqs=2))
