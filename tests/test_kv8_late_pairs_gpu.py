"""Single rows over the 8-bit cache, cut so that a CTA holds parts of two pairs that many CTAs share: it decides both at its end, often the
second while its warps have not seen the first one's decision yet."""
import pytest
import torch

import plain_kv8 as plain
from test_kv8_gpu import WEIGHTS, dev, ops   # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nh,nkv,hd,P", [(8, 2, 128, 16), (6, 3, 48, 8), (16, 1, 64, 64)])
@pytest.mark.parametrize("rows,keys,ctas", [(1, 9000, 13), (3, 9000, 31), (3, 5000, 100), (2, 9001, 148), (5, 2500, 61)])
def test_two_late_pairs_in_a_cta(ops, nh, nkv, hd, P, rows, keys, ctas, monkeypatch):   # noqa: F811
    from allpaca_b200.ops import kv8
    monkeypatch.setattr(kv8, "plan_rows", lambda *a: (ctas, 0))
    c = plain.case([(keys - 64 * i, 1) for i in range(rows)], nh, nkv, hd, P, torch.bfloat16, seed=ctas)
    want, off = plain.attend(c, 0.09, 0, WEIGHTS)
    q = dev(c["q"])
    args = (dev(c["pages"]), dev(c["table"]), dev(c["token_seq"]), dev(c["positions"]), nh, nkv, hd, P, 0.09)
    outs = [torch.full_like(q, float("nan")) for _ in range(60)]
    for out in outs:
        ops.attention_kv8(q, out, *args)
    ops.check_kernel_status()
    assert float(((outs[0].cpu().double() - want).abs() / off).max()) <= 1.0
    for out in outs:
        assert torch.equal(out, outs[0])
