"""Steps over the 8-bit cache in which one-row sequences stand before, between and behind portions, with their lengths named and without."""
import pytest
import torch

import plain_kv8 as plain
from test_kv8_gpu import WEIGHTS, ops, portions, run   # noqa: F401

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("portions")]

STEPS = [[(700, 17), (10, 1)], [(3000, 1), (317, 17)], [(3000, 1), (40, 1), (200, 150), (900, 1), (129, 5)], [(1, 1), (2, 2), (2000, 1)],
         [(2100, 300), (50, 50), (1, 1)], [(90, 0), (700, 1), (260, 130)]]


@pytest.mark.parametrize("nh,nkv,hd,P", [(8, 2, 128, 16), (4, 4, 64, 8), (6, 3, 48, 4)])
@pytest.mark.parametrize("seqs", STEPS, ids=[str(i) for i in range(len(STEPS))])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_with_and_without_contexts(ops, nh, nkv, hd, P, seqs, window, dtype):   # noqa: F811
    c = plain.case(seqs, nh, nkv, hd, P, dtype, seed=len(seqs) + hd)
    want, off = plain.attend(c, 0.09, window, WEIGHTS if dtype == torch.bfloat16 else 0.0)
    for more in ({}, {"contexts": [k for k, _ in seqs]}, {"contexts": [k + 77 for k, _ in seqs]}):
        got = run(ops, c, 0.09, window, **more)
        assert float(((got - want).abs() / off).max()) <= 1.0


def test_contexts_that_are_too_short_harm_no_other_sequence(ops):   # noqa: F811
    seqs = [(2100, 300), (300, 300), (900, 120)]
    for window in (0, 100):
        c = plain.case(seqs, 8, 2, 128, 16, torch.bfloat16, seed=3)
        want, off = plain.attend(c, 0.09, window, WEIGHTS)
        got = run(ops, c, 0.09, window, contexts=[5, 300, 900])
        assert float(((got - want).abs() / off)[300:].max()) <= 1.0


@pytest.mark.parametrize("kv_dtype", ["fp8", "auto"])
def test_a_prompt_in_portions_leaves_recorded_steps_alone(ops, tmp_path, kv_dtype):   # noqa: F811
    """Decoded rows between the portions of a growing prompt go on replaying their graph: no buffer of theirs is replaced."""
    import helpers
    from allpaca_b200.config import EngineConfig
    from allpaca_b200.engine.batch import BatchEntry
    from allpaca_b200.engine.runner import ModelRunner
    from test_kv8_engine_gpu import SERVING
    model = helpers.make_model_folder(str(tmp_path / "m"), SERVING, 3, "bfloat16")
    runner = ModelRunner(model, EngineConfig(dtype="bfloat16", kv_dtype=kv_dtype, page_size=16, num_pages=128, max_num_seqs=4,
                                             max_num_batched_tokens=512))
    long, short = helpers.random_tokens(960, 311, 1), helpers.random_tokens(120, 311, 2)
    runner.step([BatchEntry("long", long[:96], [])])
    runner.step([BatchEntry("short", short[:96], [])])     # (as many rows: every other buffer has its size)
    for t in short[96:100]:
        runner.step([BatchEntry("short", [t], [0])])
    assert runner.graph_replays == 1
    generation = runner.workspace.generation
    for i in range(1, 10):
        runner.step([BatchEntry("long", long[96 * i:96 * i + 96], [])])
        runner.step([BatchEntry("short", [short[99 + i]], [0])])
    assert runner.workspace.generation == generation
    assert runner.graph_replays == 10
    ops.check_kernel_status()
