"""GPU tests of hymoe_adapt and of hymoe_adapt_backward's dx for infinite inputs: beside weights that
are not 0 a token's infinity comes out as the definition has it, whatever its batch, type and path; NaN
as NaN; the other tokens' rows keep their bits."""
import pytest

import hymoe

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

T16 = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
INF = float("inf")


def positive(g, shape, dtype):
    return (torch.rand(shape, generator=g, device="cuda") + 0.5).to(T16[dtype])


@pytest.mark.parametrize("order", ["run", "any"])
@pytest.mark.parametrize("types", [("bf16", "bf16", "bf16"), ("f16", "f16", "f16"), ("f16", "f16", "f32"), ("f32", "bf16", "f32"),
                                   ("f32", "f16", "f16"), ("bf16", "bf16", "f32")], ids="-".join)
@pytest.mark.parametrize("n_in,n_out,rank", [(128, 136, 1), (128, 136, 8), (96, 64, 40), (77, 65, 3), (264, 72, 128), (2048, 64, 16)])
@pytest.mark.parametrize("T", [4, 70, 128, 300])
def test_infinities_as_defined(T, n_in, n_out, rank, types, order):
    x, w, y = types
    g = torch.Generator(device="cuda")
    g.manual_seed(T + rank)
    a, b = positive(g, (1, rank, n_in), w), positive(g, (1, n_out, rank), w)
    ad = hymoe.Adapters(a / 64, b / 64)
    ids = torch.zeros((T,), dtype=torch.int32, device="cuda")
    if order == "any":
        ids[2::5] = -1
    v, dy = positive(g, (T, n_in), x), positive(g, (T, n_out), y)
    base = positive(g, (T, n_out), y)
    out = ad.apply(v, ids, base=base)
    dx = ad.backward(v, dy, ids, want=("dx",))["dx"]
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(dx).all())
    at = {0: INF, 1: -INF, T - 1: float("nan")}
    for t, bad in at.items():
        v[t, t % n_in], dy[t, t % n_out] = bad, bad
    got, back = ad.apply(v, ids, base=base), ad.backward(v, dy, ids, want=("dx",))["dx"]
    rest = [t for t in range(T) if t not in at]
    assert torch.equal(got[rest], out[rest]) and torch.equal(back[rest], dx[rest])
    for r in (got, back):
        assert bool((r[0] == INF).all()) and bool((r[1] == -INF).all()), "an infinity became something else"
        if int(ids[T - 1]) == 0:
            assert bool(r[T - 1].isnan().all())
