"""GPU tests of hymoe_route and hymoe_route_backward against plain double precision (gate_ref.py).

Tolerances.  Selections are exact.  A score or weight in fp32 may be off by: the subtraction of
the row's maximum inside an exponential, half a step of a number of at most `span` (the row's range
of logits), so span * 2^-24 relative; the exponential, the sum and the quotient, 16 more half
steps.  Gradients are a few products of such numbers: the same bound on the sum of their terms'
magnitudes, and the rounding to the logits' type, half a step."""
import numpy as np
import pytest

import gate_ref as R
import hymoe

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

EPS = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}


def logits_of(T, E, dtype, seed=0, std=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, E, generator=g) * std + torch.randn(1, E, generator=g)).to(dtype)


def bias_of(E, seed=1, std=0.1):
    return torch.randn(E, generator=torch.Generator().manual_seed(seed)) * std


def span_of(z):
    z = R.clean(z)
    fin = np.where(np.isfinite(z) & (np.abs(z) < 1e30), np.abs(z), 0.0)
    return 2.0 * float(fin.max(initial=0.0))


def check_route(z, bias, K, got, **kw):
    """z: the logits as a CPU tensor."""
    zz = z.double().numpy()
    want = R.route(zz, None if bias is None else bias.double().numpy(), K, **kw)
    tol = (span_of(zz) + 16) * EPS
    np.testing.assert_array_equal(got["idx"].cpu().numpy(), want["idx"])
    np.testing.assert_allclose(got["weights"].double().cpu().numpy(), want["weights"], rtol=tol, atol=2.0 ** -120)
    if "counts" in got:
        np.testing.assert_array_equal(got["counts"].cpu().numpy(), want["counts"])
    if "scores" in got:
        np.testing.assert_allclose(got["scores"].double().cpu().numpy(), want["scores"], rtol=tol, atol=2.0 ** -120)


def check_grad(z, idx, dw, ds, got, score, norm, scale):
    zz, tol = z.double().numpy(), (span_of(z.double().numpy()) + 32) * EPS
    for t in range(z.shape[0]):
        want, mag = R.grad_row(zz[t], idx[t].numpy(), dw[t].double().numpy(),
                               None if ds is None else ds[t].double().numpy(), score, norm, scale)
        lim = tol * mag + (HALF_STEP[got.dtype]) * np.abs(want) * 1.01 + SMALLEST[got.dtype]
        err = np.abs(got[t].double().cpu().numpy() - want)
        assert (err <= lim).all(), (t, float((err / lim).max()))


CASES = [  # T, E, K, dtype, score, bias, group, group_score, norm, scale
    (1, 1, 1, torch.float32, "softmax", False, None, "max", True, 1.0),
    (1, 2, 2, torch.float32, "sigmoid", True, (2, 1), "top2", True, 1.0),
    (7, 8, 3, torch.float16, "softmax", True, (4, 2), "top2", False, 2.5),
    (16, 31, 5, torch.bfloat16, "sigmoid", False, None, "max", True, 1.0),
    (17, 32, 32, torch.float32, "softmax", True, None, "max", True, 16.0),
    (33, 33, 9, torch.float16, "sigmoid", True, (11, 4), "max", True, 1.0),
    (64, 64, 8, torch.float32, "softmax", False, (8, 3), "max", True, 1.0),
    (100, 64, 6, torch.bfloat16, "sigmoid", True, (32, 8), "top2", True, 2.5),
    (129, 72, 8, torch.float32, "sigmoid", False, (8, 4), "top2", False, 1.0),
    (65, 128, 1, torch.bfloat16, "softmax", False, None, "max", False, 1.0),
    (50, 160, 6, torch.float32, "softmax", True, (8, 3), "max", False, 16.0),
    (40, 255, 16, torch.float16, "sigmoid", False, (5, 5), "top2", True, 1.0),
    (300, 256, 8, torch.bfloat16, "sigmoid", True, (8, 4), "top2", True, 2.5),
    (25, 384, 8, torch.float32, "sigmoid", True, (1, 1), "top2", True, 1.0),
    (19, 511, 12, torch.float32, "softmax", True, None, "max", True, 1.0),
    (20, 512, 32, torch.bfloat16, "sigmoid", True, (16, 2), "max", True, 1.0),
]
NAMES = ["-".join(str(v).replace("torch.", "") for v in c[:6]) for c in CASES]


@pytest.mark.parametrize("case", CASES, ids=NAMES)
def test_route(case):
    T, E, K, dtype, score, biased, group, gs, norm, scale = case
    z = logits_of(T, E, dtype)
    b = bias_of(E) if biased else None
    g = hymoe.Gate(E, K, score=score, group=group, group_score=gs, norm_topk_prob=norm, scale=scale)
    got = g.route(z.cuda(), bias=None if b is None else b.cuda(), scores=True, counts=True)
    check_route(z, b, K, got, score=score, group=group, group_score=gs, norm=norm, scale=scale)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_closed_experts_and_strange_logits(score, biased, dtype):
    """-inf, NaN, +inf and the type's lowest value in rows, and rows that leave nothing open."""
    T, E, K = 24, 64, 8
    z = logits_of(T, E, dtype, seed=3).float()
    low = torch.finfo(dtype).min
    z[0] = float("-inf")
    z[1] = float("nan")
    z[2, 5:] = float("-inf")          # fewer open than K
    z[3, ::2] = float("nan")
    z[4, 7] = float("inf")
    z[5, [7, 40]] = float("inf")
    z[6] = low
    z[7, :60] = low
    z[8, 1:] = float("-inf")
    z[9] = float("inf")
    z[10] = 0.0                       # every expert ties
    z[11] = -80.0                     # tiny sigmoids
    z[12, :] = 30.0
    z[13] = torch.tensor([-60.0, -61.0] * 32)
    z = z.to(dtype)
    b = bias_of(E, std=0.3) if biased else None
    if biased:
        b[3], b[9], b[11] = float("-inf"), float("nan"), 5.0
    for group, gs in ((None, "max"), ((8, 2), "max"), ((8, 2), "top2")):
        g = hymoe.Gate(E, K, score=score, group=group, group_score=gs)
        got = g.route(z.cuda(), bias=None if b is None else b.cuda(), scores=True, counts=True)
        zz = z.double().numpy()
        want = R.route(zz, None if b is None else b.double().numpy(), K, score=score, group=group, group_score=gs)
        np.testing.assert_array_equal(got["idx"].cpu().numpy(), want["idx"])
        np.testing.assert_array_equal(got["counts"].cpu().numpy(), want["counts"])
        tol = (2 * 80 + 16) * EPS
        np.testing.assert_allclose(got["weights"].double().cpu().numpy(), want["weights"], rtol=tol, atol=2.0 ** -120)
        np.testing.assert_allclose(got["scores"].double().cpu().numpy(), want["scores"], rtol=tol, atol=2.0 ** -120)


def test_selection_hangs_on_last_bits():
    """Scores plus biases that only differ far below fp32: the order of double precision."""
    E, K, T = 64, 8, 256
    g = torch.Generator().manual_seed(5)
    z = torch.randn(T, E, generator=g)
    # biases that put every expert's choice value of row 0 at almost the same number
    s0 = 1.0 / (1.0 + np.exp(-z[0].double().numpy()))
    b = torch.from_numpy((1.0 - s0).astype(np.float32))
    z[1:128] = z[0] + torch.randn(127, E, generator=g) * 1e-7
    for score in ("sigmoid", "softmax"):
        gate = hymoe.Gate(E, K, score=score, group=(8, 4), group_score="top2")
        got = gate.route(z.cuda(), bias=b.cuda(), counts=True)
        check_route(z, b, K, got, score=score, group=(8, 4), group_score="top2")
        gate = hymoe.Gate(E, K, score=score)
        got = gate.route(z.cuda(), bias=b.cuda(), counts=True)
        check_route(z, b, K, got, score=score)


def test_ties_with_equal_biases():
    """bf16 logits repeat: equal scores go to the lower expert, with and without a bias."""
    T, E, K = 200, 256, 8
    z = logits_of(T, E, torch.bfloat16, std=0.5)
    for b in (None, torch.zeros(E), torch.full((E,), 0.25)):
        for score in ("softmax", "sigmoid"):
            for group, gs in ((None, "max"), ((16, 3), "top2")):
                gate = hymoe.Gate(E, K, score=score, group=group, group_score=gs)
                got = gate.route(z.cuda(), bias=None if b is None else b.cuda())
                check_route(z, b, K, got, score=score, group=group, group_score=gs)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("E", [40, 64, 512])
def test_zeros_of_both_signs_and_neighbours(dtype, E):
    """-0 ties with 0; neighbouring numbers of the type do not tie."""
    g = torch.Generator().manual_seed(11)
    z = torch.where(torch.rand(30, E, generator=g) < 0.5, 0.0, -0.0)
    z[10:20] = 1.0 + torch.randint(0, 3, (10, E), generator=g) * torch.finfo(dtype).eps
    z[20:] = -(3.0 + torch.randint(0, 9, (10, E), generator=g) * 2 * torch.finfo(dtype).eps)
    z = z.to(dtype)
    for score in ("softmax", "sigmoid"):
        for group in (None, (4, 2)):
            gate = hymoe.Gate(E, 8, score=score, group=group)
            check_route(z, None, 8, gate.route(z.cuda(), counts=True), score=score, group=group)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E,off,ld", [(64, 0, 64), (64, 1, 65), (64, 8, 96), (256, 3, 300), (60, 0, 60), (48, 4, 52)])
def test_strides_and_alignment(dtype, E, off, ld):
    T, K = 37, 6
    buf = logits_of(T, ld + off, dtype, seed=8).cuda()
    flat = torch.empty(T * ld + off, dtype=dtype, device="cuda").copy_(buf.reshape(-1)[:T * ld + off])
    z = flat.as_strided((T, E), (ld, 1), off)
    gate = hymoe.Gate(E, K, score="sigmoid")
    check_route(z.cpu(), None, K, gate.route(z, counts=True, scores=True), score="sigmoid")
    idx = gate.route(z)["idx"]
    dw = torch.randn(T, K, generator=torch.Generator().manual_seed(1))
    check_grad(z.cpu(), idx.cpu(), dw, None, gate.backward(z, idx, dw.cuda()), "sigmoid", True, 1.0)


def test_no_tokens_clears_the_counts():
    gate = hymoe.Gate(64, 8)
    r = gate.route(torch.empty(0, 64, device="cuda"), counts=True, scores=True)
    assert r["idx"].shape == (0, 8) and int(r["counts"].abs().sum()) == 0
    assert gate.backward(torch.empty(0, 64, device="cuda"), r["idx"], r["weights"]).shape == (0, 64)


def test_many_tokens_and_large_offsets():
    """More than 2^31 elements of logits: the last rows are routed like the first."""
    E, K, T = 512, 8, (1 << 22) + 33
    z = torch.empty(T, E, dtype=torch.bfloat16, device="cuda")
    part = logits_of(2048, E, torch.bfloat16)
    z.view(-1)[:].zero_()
    z[:2048], z[-2048:] = part.cuda(), part.cuda()
    gate = hymoe.Gate(E, K, score="sigmoid")
    r = gate.route(z, counts=True)
    check_route(part, None, K, {"idx": r["idx"][:2048], "weights": r["weights"][:2048]}, score="sigmoid")
    assert torch.equal(r["idx"][:2048], r["idx"][-2048:]) and torch.equal(r["weights"][:2048], r["weights"][-2048:])
    assert int(r["counts"].sum()) == T * K
    dw = torch.ones(T, K, device="cuda")
    d = gate.backward(z, r["idx"], dw)
    assert torch.equal(d[:2048], d[-2048:])


@pytest.mark.parametrize("case", CASES, ids=NAMES)
@pytest.mark.parametrize("with_ds", [False, True])
def test_gradient_formula(case, with_ds):
    T, E, K, dtype, score, biased, group, gs, norm, scale = case
    z = logits_of(T, E, dtype, seed=9)
    if T > 4 and E > 4:
        z[0] = float("-inf")
        z[1, ::3] = float("-inf")
        z[2, 1] = float("nan")
        z[3, 0] = float("inf")
    b = bias_of(E) if biased else None
    gate = hymoe.Gate(E, K, score=score, group=group, group_score=gs, norm_topk_prob=norm, scale=scale)
    idx = gate.route(z.cuda(), bias=None if b is None else b.cuda())["idx"]
    g = torch.Generator().manual_seed(2)
    dw, ds = torch.randn(T, K, generator=g), torch.randn(T, E, generator=g) if with_ds else None
    got = gate.backward(z.cuda(), idx, dw.cuda(), d_scores=None if ds is None else ds.cuda())
    assert got.dtype == dtype
    check_grad(z, idx.cpu(), dw, ds, got, score, norm, scale)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("norm", [True, False])
def test_gradient_against_differences(score, norm):
    """Central differences of the weights' definition in double precision, h = 1e-5: their own
    error is about h^2 plus 1e-16 / h, both below 1e-9 of the loss's size."""
    T, E, K, scale, h = 6, 24, 5, 2.5, 1e-5
    z = logits_of(T, E, torch.float32, seed=4)
    gate = hymoe.Gate(E, K, score=score, norm_topk_prob=norm, scale=scale)
    idx = gate.route(z.cuda())["idx"]
    g = torch.Generator().manual_seed(2)
    dw, ds = torch.randn(T, K, generator=g), torch.randn(T, E, generator=g)
    got = gate.backward(z.cuda(), idx, dw.cuda(), d_scores=ds.cuda()).double().cpu().numpy()
    for t in range(T):
        row, i = z[t].double().numpy(), idx[t].cpu().numpy()
        _, mag = R.grad_row(row, i, dw[t].double().numpy(), ds[t].double().numpy(), score, norm, scale)
        for e in range(E):
            up, dn = row.copy(), row.copy()
            up[e] += h
            dn[e] -= h
            args = (i, dw[t].double().numpy(), ds[t].double().numpy(), score, norm, scale)
            d = (R.loss(up, *args) - R.loss(dn, *args)) / (2 * h)
            assert abs(d - got[t, e]) <= (span_of(row) + 32) * EPS * mag[e] + 1e-8, (t, e)


def test_gradient_of_repeated_and_foreign_indices():
    """The same expert twice, indices outside the range and indices of closed experts."""
    T, E, K = 5, 40, 4
    z = logits_of(T, E, torch.float32, seed=6)
    z[1, 7] = float("-inf")
    idx = torch.tensor([[3, 3, 5, 3], [7, 2, -1, 40], [-5, 1000, -1, -1], [0, 39, 0, 39], [1, 2, 3, 4]], dtype=torch.int32)
    dw = torch.randn(T, K, generator=torch.Generator().manual_seed(3))
    for score in ("softmax", "sigmoid"):
        for norm in (True, False):
            gate = hymoe.Gate(E, K, score=score, norm_topk_prob=norm)
            got = gate.backward(z.cuda(), idx.cuda(), dw.cuda())
            check_grad(z, idx, dw, None, got, score, norm, 1.0)


def test_gradient_in_place():
    import ctypes as C
    T, E, K = 50, 96, 6
    z = logits_of(T, E, torch.bfloat16).cuda()
    gate = hymoe.Gate(E, K)
    idx = gate.route(z)["idx"]
    dw = torch.randn(T, K, device="cuda")
    want = gate.backward(z, idx, dw)
    m = hymoe.Mat(z.data_ptr(), hymoe.TYPE_BF16, E)
    st = hymoe.lib().hymoe_route_backward(C.byref(gate.spec), C.byref(m), idx.data_ptr(), dw.data_ptr(), None, T, E, K,
                                          C.byref(m), torch.cuda.current_stream().cuda_stream)
    assert st == 0 and torch.equal(z, want)


def test_rows_between_are_left():
    """Strided gradient rows: the columns behind n_experts stay as they were."""
    import ctypes as C
    T, E, K, ld = 9, 50, 4, 64
    z = logits_of(T, E, torch.float32).cuda()
    gate = hymoe.Gate(E, K)
    idx = gate.route(z)["idx"]
    dw = torch.randn(T, K, device="cuda")
    out = torch.full((T, ld), 7.0, device="cuda")
    st = hymoe.lib().hymoe_route_backward(C.byref(gate.spec), C.byref(hymoe.Mat(z.data_ptr(), 0, E)), idx.data_ptr(),
                                          dw.data_ptr(), None, T, E, K, C.byref(hymoe.Mat(out.data_ptr(), 0, ld)),
                                          torch.cuda.current_stream().cuda_stream)
    assert st == 0
    assert torch.equal(out[:, :E], gate.backward(z, idx, dw)) and bool((out[:, E:] == 7.0).all())


def test_graph_capture_and_streams():
    """A captured call replays on changed inputs; calls on two streams at once share nothing."""
    T, E, K = 512, 128, 6
    z = [logits_of(T, E, torch.bfloat16, seed=s) for s in range(3)]
    b = bias_of(E)
    gate = hymoe.Gate(E, K, score="sigmoid")
    zd, bd, dw = z[0].cuda(), b.cuda(), torch.randn(T, K, device="cuda")
    gate.route(zd, bias=bd, counts=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = gate.route(zd, bias=bd, counts=True, scores=True)
        d = gate.backward(zd, r["idx"], dw)
    for s in (1, 2):
        zd.copy_(z[s])
        graph.replay()
        torch.cuda.synchronize()
        check_route(z[s], b, K, r, score="sigmoid")
        check_grad(z[s], r["idx"].cpu(), dw.cpu(), None, d, "sigmoid", True, 1.0)
    streams = [torch.cuda.Stream() for _ in range(2)]
    zs, outs = [z[1].cuda(), z[2].cuda()], []
    torch.cuda.synchronize()
    for _ in range(8):
        for s, zz in zip(streams, zs):
            with torch.cuda.stream(s):
                outs.append(gate.route(zz, bias=bd, counts=True))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        check_route(z[1 + i % 2], b, K, o, score="sigmoid")


def test_refuses_host_memory():
    import ctypes as C
    gate = hymoe.Gate(64, 8)
    z = torch.zeros(4, 64, device="cuda")
    host = torch.zeros(4, 64)
    idx, w = torch.zeros(4, 8, dtype=torch.int32, device="cuda"), torch.zeros(4, 8, device="cuda")
    L = hymoe.lib()
    args = (None, 4, 64, 8, idx.data_ptr(), w.data_ptr(), None, None, None)
    assert L.hymoe_route(C.byref(gate.spec), C.byref(hymoe.Mat(host.data_ptr(), 0, 64)), *args) == 1
    assert L.hymoe_route(C.byref(gate.spec), C.byref(hymoe.Mat(z.data_ptr(), 0, 64)), *args) == 0
    with pytest.raises(ValueError):
        gate.route(z, bias=torch.zeros(64))
    with pytest.raises(ValueError):
        gate.route(z.t())
