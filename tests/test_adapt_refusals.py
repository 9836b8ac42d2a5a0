"""CPU tests of hymoe_adapt and hymoe_adapt_backward: bad arguments are refused with a status and a
message, before the device is looked at."""
import ctypes as C

import pytest

import hymoe

F32, F16, BF16 = hymoe.TYPE_F32, hymoe.TYPE_F16, hymoe.TYPE_BF16
P = 1 << 24  # addresses that are never read, 16 MiB apart


def spec(n=4, r=8, i=64, o=96, t=BF16, a=P, b=2 * P, scale=None):
    return hymoe.AdapterSpec(n, r, i, o, t, a, b, scale)


X, Y, DX = hymoe.Mat(3 * P, BF16, 64), hymoe.Mat(4 * P, BF16, 96), hymoe.Mat(5 * P, BF16, 64)
WS = 6 * P


def ref(m):
    return C.byref(m) if m is not None else None


def need(s, T, back):
    n = C.c_size_t()
    assert hymoe.lib().hymoe_adapt_workspace(C.byref(s), T, back, C.byref(n)) == 0
    return n.value


def fwd(s, x=X, base=None, out=Y, ids=None, T=300, ws=WS, ws_bytes=1 << 22):
    return hymoe.lib().hymoe_adapt(ref(s), ref(x), ids, T, ref(base), ref(out), ws, ws_bytes, None)


def bwd(s, x=X, dy=Y, base=None, dx=DX, ids=None, T=300, da=8 * P, db=9 * P, ws=WS, ws_bytes=1 << 22):
    return hymoe.lib().hymoe_adapt_backward(ref(s), ref(x), ref(dy), ids, T, ref(base), ref(dx), da, db, ws, ws_bytes, None)


@pytest.mark.parametrize("s,word", [
    (None, b"null"), (spec(n=0), b"n_adapters"), (spec(n=4097), b"n_adapters"), (spec(r=0), b"rank"),
    (spec(r=129), b"rank"), (spec(i=0), b"features"), (spec(o=0), b"features"), (spec(i=(1 << 20) + 1), b"features"),
    (spec(t=F32), b"F16 or BF16"), (spec(t=8), b"F16 or BF16")])
def test_bad_adapters(s, word):
    n = C.c_size_t()
    L = hymoe.lib()
    assert fwd(s) == 1 and word in L.hymoe_last_error(None)
    assert bwd(s) == 1 and word in L.hymoe_last_error(None)
    assert L.hymoe_adapt_workspace(ref(s), 1, 0, C.byref(n)) == 1 and word in L.hymoe_last_error(None)


def test_workspace_query():
    L, n = hymoe.lib(), C.c_size_t()
    assert L.hymoe_adapt_workspace(C.byref(spec()), 1, 0, None) == 1
    assert L.hymoe_adapt_workspace(C.byref(spec()), (1 << 24) + 1, 0, C.byref(n)) == 1
    assert need(spec(), 0, 0) >= 0
    # what n tokens need is enough for fewer
    last = {0: 0, 1: 0}
    for T in (1, 7, 63, 64, 65, 128, 300, 4096, 8192):
        for back in (0, 1):
            got = need(spec(r=33), T, back)
            assert got >= last[back]
            last[back] = got


@pytest.mark.parametrize("kw", [dict(a=None), dict(b=None), dict(a=P + 1), dict(b=2 * P + 1), dict(scale=7 * P + 2)])
def test_bad_weights(kw):
    assert fwd(spec(**kw)) == 1
    assert bwd(spec(**kw)) == 1


@pytest.mark.parametrize("m", [None, hymoe.Mat(None, BF16, 128), hymoe.Mat(10 * P, F16, 128), hymoe.Mat(10 * P, 8, 128),
                               hymoe.Mat(10 * P, BF16, 40), hymoe.Mat(10 * P + 1, BF16, 128), hymoe.Mat(10 * P + 2, F32, 128)])
def test_bad_matrices(m):
    s = spec()
    assert fwd(s, x=m) == 1
    assert fwd(s, out=m) == 1
    assert bwd(s, x=m) == 1
    assert bwd(s, dy=m) == 1
    if m is not None:
        assert fwd(s, base=m) == 1
        assert bwd(s, base=m) == 1
        assert bwd(s, dx=m) == 1


def test_types_that_do_not_go_together():
    assert fwd(spec(), base=hymoe.Mat(10 * P, F32, 96)) == 1           # base F32, out BF16
    assert bwd(spec(), dx=hymoe.Mat(10 * P, F32, 64)) == 1             # dx F32, x BF16
    assert bwd(spec(), base=hymoe.Mat(10 * P, BF16, 64), dx=None) == 1  # a base with nowhere to go


def test_workspace():
    s, T = spec(), 300
    for back, call in ((0, fwd), (1, bwd)):
        n = need(s, T, back)
        assert n > 0
        assert call(s, T=T, ws=None) == 1
        assert call(s, T=T, ws=WS + 16) == 1
        assert call(s, T=T, ws_bytes=n - 1) == 1
        assert b"workspace" in hymoe.lib().hymoe_last_error(None)


def test_overlaps():
    s = spec()
    near = hymoe.Mat(4 * P + 96, BF16, 96)
    assert fwd(s, base=near) == 1                        # not the same buffer, but overlapping
    assert fwd(s, base=hymoe.Mat(4 * P, BF16, 192)) == 1  # the same start, other rows
    assert fwd(s, out=hymoe.Mat(3 * P + 128, BF16, 96)) == 1
    assert fwd(s, out=hymoe.Mat(P, BF16, 96)) == 1
    assert fwd(s, ws=3 * P) == 1
    assert fwd(s, ws=4 * P) == 1
    assert bwd(s, dx=hymoe.Mat(3 * P, BF16, 64)) == 1
    assert bwd(s, da=9 * P + 64, db=9 * P) == 1
    assert bwd(s, da=4 * P) == 1
    assert bwd(s, ws=8 * P) == 1
    assert b"overlap" in hymoe.lib().hymoe_last_error(None)


def test_misaligned():
    assert fwd(spec(), ids=7 * P + 2) == 1
    assert bwd(spec(), ids=7 * P + 1) == 1
    assert bwd(spec(), da=8 * P + 2) == 1
    assert bwd(spec(), db=9 * P + 1) == 1


def test_too_many_tokens():
    assert fwd(spec(), T=(1 << 24) + 1) == 1
    assert bwd(spec(), T=(1 << 24) + 1) == 1


def test_no_tokens():
    assert fwd(spec(), x=None, out=None, T=0, ws=None, ws_bytes=0) == 0


def test_python_checks():
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError):
        hymoe.Adapters(torch.zeros(2, 8, 64), torch.zeros(2, 96, 8))
    with pytest.raises(ValueError):
        hymoe.Adapters(torch.zeros(2, 8, 64), torch.zeros(2, 96, 9))
