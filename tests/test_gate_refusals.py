"""CPU tests of hymoe_route and hymoe_route_backward: bad arguments are refused with a status and
a message, before the device is looked at."""
import ctypes as C

import pytest

import hymoe

F32, F16, BF16 = hymoe.TYPE_F32, hymoe.TYPE_F16, hymoe.TYPE_BF16
P = 1 << 20  # an address that is never read


def spec(score=0, ng=0, tg=0, gs=0, norm=1, scale=1.0):
    return hymoe.GateSpec(score, ng, tg, gs, norm, scale)


def route(g, m, T=4, E=64, K=8, bias=None, idx=P, w=2 * P, scores=None, counts=None):
    return hymoe.lib().hymoe_route(C.byref(g) if g else None, C.byref(m) if m else None, bias, T, E, K, idx, w,
                                   scores, counts, None)


def backward(g, m, d, T=4, E=64, K=8, idx=P, dw=2 * P, ds=None):
    return hymoe.lib().hymoe_route_backward(C.byref(g) if g else None, C.byref(m) if m else None, idx, dw, ds, T, E, K,
                                            C.byref(d) if d else None, None)


GOOD = hymoe.Mat(8 * P, F32, 64)


@pytest.mark.parametrize("g,E,K,word", [
    (None, 64, 8, b"gate"), (spec(score=2), 64, 8, b"score"), (spec(score=-1), 64, 8, b"score"),
    (spec(gs=2), 64, 8, b"group_score"), (spec(ng=33, tg=1), 66, 8, b"n_group"), (spec(ng=3, tg=1), 64, 8, b"n_group"),
    (spec(ng=4, tg=0), 64, 8, b"topk_group"), (spec(ng=4, tg=5), 64, 8, b"topk_group"),
    (spec(scale=float("nan")), 64, 8, b"finite"), (spec(scale=float("inf")), 64, 8, b"finite"),
    (spec(), 0, 1, b"n_experts"), (spec(), 513, 8, b"n_experts"), (spec(), 64, 0, b"topk"), (spec(), 64, 33, b"topk"),
    (spec(), 4, 5, b"topk")])
def test_bad_gates(g, E, K, word):
    m = hymoe.Mat(8 * P, F32, 1024)
    assert route(g, m, E=E, K=K) == 1 and word in hymoe.lib().hymoe_last_error(None)
    assert backward(g, m, hymoe.Mat(16 * P, F32, 1024), E=E, K=K) == 1
    assert word in hymoe.lib().hymoe_last_error(None)


@pytest.mark.parametrize("m", [None, hymoe.Mat(None, F32, 64), hymoe.Mat(8 * P, 7, 64), hymoe.Mat(8 * P, 8, 64),
                               hymoe.Mat(8 * P, F32, 63), hymoe.Mat(8 * P, F32, -64), hymoe.Mat(8 * P + 2, F32, 64),
                               hymoe.Mat(8 * P + 1, BF16, 64)])
def test_bad_matrices(m):
    assert route(spec(), m) == 1
    assert backward(spec(), m, GOOD) == 1
    assert backward(spec(), GOOD, m) == 1


def test_null_and_misaligned_outputs():
    assert route(spec(), GOOD, idx=None) == 1
    assert route(spec(), GOOD, w=None) == 1
    assert route(spec(), GOOD, w=2 * P + 2) == 1
    assert route(spec(), GOOD, bias=3 * P + 1) == 1
    assert route(spec(), GOOD, scores=3 * P + 2) == 1
    d = hymoe.Mat(16 * P, F32, 64)
    assert backward(spec(), GOOD, d, idx=None) == 1
    assert backward(spec(), GOOD, d, dw=None) == 1
    assert backward(spec(), GOOD, d, ds=3 * P + 2) == 1
    assert backward(spec(), GOOD, hymoe.Mat(16 * P, F16, 64)) == 1  # another type than the logits'


def test_overlaps():
    assert route(spec(), GOOD, idx=8 * P) == 1
    assert route(spec(), GOOD, idx=P, w=P + 64) == 1
    assert route(spec(), GOOD, scores=8 * P + 256) == 1
    assert backward(spec(), GOOD, hymoe.Mat(8 * P + 256, F32, 64)) == 1
    assert backward(spec(), GOOD, hymoe.Mat(P, F32, 64)) == 1
    assert b"overlap" in hymoe.lib().hymoe_last_error(None)


def test_no_tokens():
    assert backward(spec(), None, None, T=0) == 0


def test_python_checks():
    with pytest.raises(ValueError):
        hymoe.Gate(64, 8, score="linear")
    with pytest.raises(hymoe.HymoeError):
        hymoe.Gate(64, 65)
    torch = pytest.importorskip("torch")
    g = hymoe.Gate(64, 8)
    with pytest.raises(ValueError):
        g.route(torch.zeros(2, 64))  # host memory
    with pytest.raises(ValueError):
        g.route(torch.zeros(2, 63))
