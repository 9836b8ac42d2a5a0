"""GPU tests of hymoe_route and of the block's gate where biases are as large or as low as a type
holds: the lowest finite value, a usual way to mask an expert, leaves it open (only -inf and NaN
close), and the sum of a group's two best can lie beyond fp32.  Selections against plain double
precision (gate_ref.py), in every form: a warp per token with experts in runs and spread, a thread
per token, the block.  The tolerances are those of test_gpu_gate.py."""
import numpy as np
import pytest

import gate_ref as R
import hymoe
from test_gpu_block_gate_adapters import Block, check_gate, gate_of
from test_gpu_gate import check_route, logits_of
from test_gpu_gate_rows import T_GROUPS

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

LOW, BIG = float(np.finfo(np.float32).min), float(np.finfo(np.float32).max)
INF = float("inf")


def biases(E, G):
    """name -> bias [E], group by group (E / G experts each, at least two)."""
    n = E // G

    def of(f):
        return torch.tensor([f(e // n, e % n) for e in range(E)], dtype=torch.float32)

    return {
        "one group unmasked": of(lambda g, i: 0.0 if g == 0 else LOW),
        "two experts unmasked": of(lambda g, i: 0.0 if g == 0 and i < 2 else LOW),
        "last group unmasked": of(lambda g, i: 0.01 * i if g == G - 1 else LOW),
        "every second expert masked": of(lambda g, i: LOW if i % 2 else 0.0),
        "one of each group unmasked": of(lambda g, i: 0.0 if i == g % n else LOW),
        "all masked": of(lambda g, i: LOW),
        "masked in steps": of(lambda g, i: LOW * (1.0 - g / 16) if g else 0.0),
        "lowest beside closed": of(lambda g, i: (-INF, LOW, 0.0, float("nan"))[(g + i) % 4]),
        "large sums": of(lambda g, i: (INF if i == 0 else 1e38) if g % 2 == 0 else BIG if i < 2 else 0.0),
        "large sums in steps": of(lambda g, i: 2e38 + 1e37 * g if i < 2 else -3e38),
        "both ends": of(lambda g, i: BIG if (g + i) % 2 else LOW),
        "large and ordinary": of(lambda g, i: 3e38 if g == 1 and i < 2 else LOW if g == 2 else 0.1 * i),
    }


NAMES = list(biases(16, 8))
GROUPS = [(16, 8, 3, 4), (16, 8, 3, 6), (16, 4, 1, 3), (64, 8, 3, 8), (72, 9, 4, 7), (96, 8, 8, 16), (128, 4, 2, 8), (256, 8, 4, 8)]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("E,G,kept,K", GROUPS, ids=lambda v: str(v))
def test_groups(E, G, kept, K, name):
    b = biases(E, G)[name]
    for score in ("sigmoid", "softmax"):
        for gs in ("top2", "max"):
            kw = dict(score=score, group=(G, kept), group_score=gs)
            gate = hymoe.Gate(E, K, **kw)
            for dtype in (torch.float32, torch.bfloat16):
                z = logits_of(12, E, dtype, seed=E + K)
                z[3] = 0.25  # every expert ties
                got = gate.route(z.cuda(), bias=b.cuda(), scores=dtype == torch.float32, counts=True)
                check_route(z, b, K, got, **kw)


@pytest.mark.parametrize("name", NAMES)
def test_without_groups(name):
    for E, K in ((16, 4), (64, 8), (72, 32), (256, 8)):
        b = biases(E, 8)[name]
        for score in ("sigmoid", "softmax"):
            z = logits_of(9, E, torch.float32, seed=E)
            check_route(z, b, K, hymoe.Gate(E, K, score=score).route(z.cuda(), bias=b.cuda()), score=score)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("E,G,kept,K", [(64, 8, 3, 8), (72, 9, 4, 7), (128, 4, 2, 3)], ids=lambda v: str(v))
def test_a_thread_per_token(E, G, kept, K, name):
    z = logits_of(T_GROUPS, E, torch.bfloat16, seed=E)
    z[3] = 0.25
    b = biases(E, G)[name]
    for gs in ("top2", "max"):
        kw = dict(score="sigmoid", group=(G, kept), group_score=gs)
        got = hymoe.Gate(E, K, **kw).route(z.cuda(), bias=b.cuda(), counts=True)
        n = 60
        check_route(z[:n], b, K, {k: got[k][:n] for k in ("idx", "weights")}, **kw)
        assert int(got["counts"].sum()) == int((got["idx"] >= 0).sum())


@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("name", NAMES)
def test_in_the_block(orc, T, name):
    b = Block(orc)
    kw = dict(score="sigmoid", group=(8, 3), group_score="top2", norm=True, scale=1.0)
    b.m.set_gate(gate_of(b.E, b.K, kw))
    bias = biases(b.E, 8)[name].numpy()
    b.m.set_balance_bias(0, bias)
    check_gate(b.m.forward_host(0, b.x(T), debug=True), bias.astype(np.float64), b.K, **kw)
    b.m.close()


def test_the_definition_keeps_masked_groups():
    """What the plain reference says of the simplest such token."""
    bias = np.array([0.0, 0.0] + [LOW] * 14)
    want = R.route(np.zeros((1, 16)), bias, 6, score="sigmoid", group=(8, 3), group_score="top2")
    np.testing.assert_array_equal(want["idx"], [[0, 1, 2, 3, 4, 5]])
