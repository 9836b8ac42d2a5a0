"""GPU tests of the block with a gate and adapters at wider sizes than test_gpu_block_gate_adapters.py:
several tiles of every projection, adapter rows that the products split and share."""
import numpy as np
import pytest

import oracle as O
import test_gpu_block_gate_adapters as B
from moe_cases import REL_L2_TOL, rel_l2

pytestmark = pytest.mark.gpu
pytest.importorskip("torch")


@pytest.mark.parametrize("T", [1, 6, 40, 65, 200])
@pytest.mark.parametrize("wt", [O.Q4_0, O.Q8_0, O.F16])
@pytest.mark.parametrize("h,i", [(1024, 768), (2048, 320)])
def test_gate_and_adapters(orc, monkeypatch, h, i, wt, T):
    monkeypatch.setattr(B, "H", h)
    monkeypatch.setattr(B, "I", i)
    b = B.Block(orc, E=8, K=3, wt=wt, max_tokens=256)
    kw = dict(score="sigmoid", group=(4, 2), group_score="top2", norm=True, scale=1.5)
    bias = (np.random.default_rng(3).standard_normal(b.E) * 0.1).astype(np.float32)
    b.m.set_gate(B.gate_of(b.E, b.K, kw))
    b.m.set_balance_bias(0, bias)
    b.m.set_adapters(0, b.ad["gu"], b.ad["dn"])
    x, ids = b.x(T), B.ids_of(T)
    r = b.m.forward_host(0, x, debug=True, adapter_ids=ids)
    idx, w = B.check_gate(r, bias.astype(np.float64), b.K, **kw)
    assert rel_l2(r["out"], b.reference(x, idx, w, ids)) <= REL_L2_TOL
    plain = b.m.forward_host(0, x, debug=True)
    assert rel_l2(plain["out"], b.reference(x, idx, w)) <= REL_L2_TOL
    b.m.close()
