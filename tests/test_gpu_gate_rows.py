"""GPU tests of hymoe_route for many tokens, which threads take one each: against plain double
precision (gate_ref.py), with the tolerances of test_gpu_gate.py, and against the same tokens in
short calls, which warps take one each."""
import numpy as np
import pytest

import gate_ref as R
import hymoe
from test_gpu_gate import EPS, bias_of, check_route, logits_of, span_of

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

T0, T_GROUPS = 16384 + 77, 65536 + 77  # tokens enough for that form, and with groups

CASES = [  # E, K, score, bias, group, group_score, norm, scale
    (8, 8, "softmax", False, None, "max", True, 1.0),
    (8, 1, "sigmoid", True, None, "max", False, 1.0),
    (40, 5, "softmax", False, None, "max", False, 16.0),
    (64, 8, "sigmoid", True, (8, 3), "top2", True, 2.5),
    (72, 7, "sigmoid", False, (9, 4), "top2", True, 1.0),
    (128, 6, "sigmoid", True, None, "max", True, 1.0),
    (160, 6, "softmax", False, (20, 3), "max", False, 16.0),
    (256, 8, "sigmoid", True, (8, 4), "top2", True, 2.5),
    (256, 2, "sigmoid", False, (32, 5), "max", False, 1.0),
    (512, 8, "softmax", False, None, "max", True, 1.0),
    (504, 8, "sigmoid", True, (1, 1), "max", True, 1.0),
]
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def strange(z, E):
    """Rows of every kind among ordinary ones."""
    z = z.float()
    z[0], z[1], z[2, 5:] = float("-inf"), float("nan"), float("-inf")
    z[3, ::2], z[4, E // 2], z[5, [1, E - 1]] = float("nan"), float("inf"), float("inf")
    z[6], z[7], z[8], z[9] = -6e4, float("inf"), 0.0, -80.0
    z[10, 1:], z[11], z[12] = float("-inf"), 30.0, -0.0
    z[13:40] = z[13:40].masked_fill(torch.rand(27, E, generator=torch.Generator().manual_seed(9)) < 0.7, float("-inf"))
    return z


@pytest.mark.parametrize("case", CASES, ids=["-".join(map(str, c[:6])) for c in CASES])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rows(case, dtype):
    E, K, score, biased, group, gs, norm, scale = case
    T = T_GROUPS if group else T0
    z = strange(logits_of(T, E, dtype, seed=E), E).to(dtype)
    b = bias_of(E) if biased else None
    if biased and E > 8:
        b[3], b[5], b[7] = float("-inf"), float("nan"), 5.0
    gate = hymoe.Gate(E, K, score=score, group=group, group_score=gs, norm_topk_prob=norm, scale=scale)
    d, db = z.cuda(), None if b is None else b.cuda()
    got = gate.route(d, bias=db, counts=True)
    n = 300  # these against double precision, the others against calls of a few tokens
    zz = z[:n].double().numpy()
    want = R.route(zz, None if b is None else b.double().numpy(), K, score=score, group=group, group_score=gs, norm=norm, scale=scale)
    np.testing.assert_array_equal(got["idx"][:n].cpu().numpy(), want["idx"])
    tol = (min(span_of(zz), 208.0) + 16) * EPS  # beyond e^-104 an exponential is 0
    np.testing.assert_allclose(got["weights"][:n].double().cpu().numpy(), want["weights"], rtol=tol, atol=2.0 ** -120)
    parts = [gate.route(d[t:t + 1500], bias=db, counts=True) for t in range(0, T, 1500)]
    assert torch.equal(got["idx"], torch.cat([p["idx"] for p in parts]))
    assert torch.equal(got["counts"], sum(p["counts"] for p in parts))
    torch.testing.assert_close(got["weights"], torch.cat([p["weights"] for p in parts]), rtol=64 * EPS, atol=2.0 ** -120)


@pytest.mark.parametrize("T", [16384, 16385, 16415, 80000])
def test_row_counts_and_rows_behind_the_last_token(T):
    E, K = 64, 4
    z = logits_of(T, E, torch.bfloat16).cuda()
    gate = hymoe.Gate(E, K, score="sigmoid")
    r = gate.route(z, counts=True)
    one = gate.route(z[-3:])
    assert torch.equal(r["idx"][-3:], one["idx"]) and int(r["counts"].sum()) == T * K
    idx = torch.full((T + 9, K), 77, dtype=torch.int32, device="cuda")
    w = torch.full((T + 9, K), 5.0, device="cuda")
    m = hymoe.Mat(z.data_ptr(), 30, E)
    assert gate.L.hymoe_route(gate._spec, m, None, T, E, K, idx.data_ptr(), w.data_ptr(), None, None, None) == 0
    torch.cuda.synchronize()
    assert torch.equal(idx[:T], r["idx"]) and bool((idx[T:] == 77).all()) and bool((w[T:] == 5.0).all())


def test_selection_hangs_on_last_bits():
    """Choice values that only differ far below fp32, in every lane of a warp and here and there."""
    E, K = 64, 8
    g = torch.Generator().manual_seed(5)
    z = torch.randn(T_GROUPS, E, generator=g)
    b = torch.from_numpy((1.0 - 1.0 / (1.0 + np.exp(-z[0].double().numpy()))).astype(np.float32))
    z[1:128] = z[0] + torch.randn(127, E, generator=g) * 1e-7
    z[200:2000:9] = z[0] + torch.randn(200, E, generator=g) * 1e-7
    for kw in (dict(), dict(group=(8, 4), group_score="top2")):
        gate = hymoe.Gate(E, K, score="sigmoid", **kw)
        got = gate.route(z.cuda(), bias=b.cuda())
        rows = list(range(140)) + list(range(200, 2000, 9))
        check_route(z[rows], b, K, {k: v[rows] for k, v in got.items()}, score="sigmoid", **kw)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_ties_and_zeros_of_both_signs(dtype):
    E, K = 128, 8
    g = torch.Generator().manual_seed(11)
    z = torch.where(torch.rand(T0, E, generator=g) < 0.5, 0.0, -0.0)
    z[100:200] = 1.0 + torch.randint(0, 3, (100, E), generator=g) * torch.finfo(dtype).eps
    z[200:300] = -(3.0 + torch.randint(0, 9, (100, E), generator=g) * 2 * torch.finfo(dtype).eps)
    z = z.to(dtype)
    for b in (None, torch.full((E,), 0.25)):
        gate = hymoe.Gate(E, K, score="sigmoid")
        got = gate.route(z.cuda(), bias=None if b is None else b.cuda())
        check_route(z[:320], b, K, {k: v[:320] for k, v in got.items()}, score="sigmoid")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("off,ld", [(0, 72), (8, 64), (1, 65), (4, 68)])
def test_strides_and_alignment(dtype, off, ld):
    E, K = 64, 6
    flat = logits_of(T0, ld, dtype, seed=8).reshape(-1)
    flat = torch.cat([torch.zeros(off, dtype=dtype), flat]).cuda()
    z = flat.as_strided((T0, E), (ld, 1), off)
    gate = hymoe.Gate(E, K, score="sigmoid")
    got = gate.route(z, counts=True)
    want = gate.route(z.contiguous(), counts=True)
    assert all(torch.equal(got[k], want[k]) for k in ("idx", "counts"))
    check_route(z[:200].cpu(), None, K, {k: got[k][:200] for k in ("idx", "weights")}, score="sigmoid")


def test_graph_and_streams():
    E, K = 128, 6
    gate = hymoe.Gate(E, K, score="sigmoid")
    b = bias_of(E).cuda()
    zs = [logits_of(T0, E, torch.bfloat16, seed=s).cuda() for s in (1, 2)]
    live = [z.clone() for z in zs]
    graphs, outs = [], []
    for v in live:
        gate.route(v, bias=b, counts=True)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(gate.route(v, bias=b, counts=True))
        graphs.append(graph)
    for turn in range(3):
        for z, v in zip(zs, live):
            v.copy_(z.roll(turn, 0))
        torch.cuda.synchronize()
        for graph in graphs:
            with torch.cuda.stream(torch.cuda.Stream()):
                graph.replay()
        eager = []
        for z in zs:
            with torch.cuda.stream(torch.cuda.Stream()):
                eager.append(gate.route(z.roll(turn, 0), bias=b, counts=True))
        torch.cuda.synchronize()
        assert all(torch.equal(o[k], e[k]) for o, e in zip(outs, eager) for k in o)
