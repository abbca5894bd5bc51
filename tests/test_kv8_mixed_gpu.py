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
