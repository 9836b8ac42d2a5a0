"""GPU tests of the block with a gate and with adapters (hymoe_set_gate, hymoe_set_balance_bias,
hymoe_set_adapters, hymoe_forward_adapted), alone and together, against the definition in double
precision: the gate of gate_ref.py on the call's own router logits, the experts' and the adapters'
products in numpy.  Selections are exact; outputs within the block's tolerance (fp16 operands)."""
import ctypes as C

import numpy as np
import pytest

import gate_ref as R
import hymoe
import oracle as O
from moe_cases import REL_L2_TOL, host_layer, rel_l2

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

H, I = 256, 128


class Block:
    def __init__(self, orc, E=16, K=4, wt=O.Q4_0, max_tokens=512, layers=1, seed=5):
        self.E, self.K, self.orc = E, K, orc
        self.lay = host_layer(orc, seed, 0, H, I, E, wt)
        self.m = hymoe.MoE(H, I, E, K, layers, max(16, max_tokens))
        for layer in range(layers):
            self.load(layer, wt)
        g = torch.Generator().manual_seed(seed)
        n, r = 3, 12
        self.raw = {}
        for name, (i, o) in {"gu": (H, 2 * I), "dn": (I, H)}.items():
            a = (torch.randn(n, r, i, generator=g) * i ** -0.5).half()
            b = (torch.randn(n, o, r, generator=g) * 0.1).half()
            s = torch.rand(n, generator=g) + 0.5
            self.raw[name] = (a, b, s)
        self.ad = {k: hymoe.Adapters(a.cuda(), b.cuda(), s.cuda()) for k, (a, b, s) in self.raw.items()}

    def load(self, layer, wt):
        lay = self.lay
        self.m.load_layer(layer, lay["router"], lay["sgu"], lay["sdn"], lay["egu"], lay["edn"], wt)

    def delta(self, name, x, ids):
        a, b, s = (t.double().numpy() for t in self.raw[name])
        out = np.zeros((len(x), b.shape[1]))
        for k in range(len(s)):
            rows = ids == k
            out[rows] = s[k] * (x[rows] @ a[k].T) @ b[k].T
        return out

    @staticmethod
    def swiglu(z):
        g, u = z[:, :I], z[:, I:]
        return g / (1.0 + np.exp(-g)) * u

    def reference(self, x, idx, w, ids=None, use=("gu", "dn")):
        x = x.astype(np.float64)
        z = x @ self.lay["sgu_f"].reshape(2 * I, H).astype(np.float64).T
        if ids is not None and "gu" in use:
            z = z + self.delta("gu", x, ids)
        h = self.swiglu(z)
        out = h @ self.lay["sdn_f"].reshape(H, I).astype(np.float64).T
        if ids is not None and "dn" in use:
            out = out + self.delta("dn", h, ids)
        for e in range(self.E):
            rows, ks = np.nonzero(idx == e)
            if len(rows):
                y = self.swiglu(x[rows] @ self.lay["egu_f"][e].reshape(2 * I, H).astype(np.float64).T)
                y = y @ self.lay["edn_f"][e].reshape(H, I).astype(np.float64).T
                np.add.at(out, rows, w[rows, ks][:, None] * y)
        return out

    def x(self, T, seed=1):
        return O.synth_x(self.orc, seed, T, H)


def ids_of(T, seed=2):
    return np.random.default_rng(seed).integers(-1, 3, T).astype(np.int32)


def check_gate(r, bias, K, **kw):
    """The call's routing against the definition on its own logits; returns (idx, w)."""
    want = R.route(r["logits"].astype(np.float64), bias, K, **kw)
    np.testing.assert_array_equal(r["idx"], want["idx"])
    z = r["logits"][np.isfinite(r["logits"])]
    tol = (2 * float(np.abs(z).max(initial=0)) + 16) * 2.0 ** -24
    np.testing.assert_allclose(r["w"], want["weights"], rtol=tol, atol=2.0 ** -120)
    np.testing.assert_allclose(r["probs"], want["scores"], rtol=tol, atol=2.0 ** -120)
    return want["idx"], want["weights"]


GATES = [dict(score="sigmoid", norm=True, scale=2.5), dict(score="softmax", norm=False, scale=1.0),
         dict(score="sigmoid", group=(8, 3), group_score="top2", norm=True, scale=1.0)]


def gate_of(E, K, kw):
    return hymoe.Gate(E, K, score=kw["score"], group=kw.get("group"), group_score=kw.get("group_score", "max"),
                      norm_topk_prob=kw["norm"], scale=kw["scale"])


@pytest.mark.parametrize("T", [1, 4, 8, 16, 17, 64, 65, 300])
@pytest.mark.parametrize("kw", GATES, ids=["sigmoid", "softmax", "groups"])
def test_gated_block(orc, T, kw):
    b = Block(orc)
    bias = (np.random.default_rng(3).standard_normal(b.E) * 0.1).astype(np.float32)
    b.m.set_gate(gate_of(b.E, b.K, kw))
    for use in (None, bias):
        b.m.set_balance_bias(0, use)
        x = b.x(T)
        r = b.m.forward_host(0, x, debug=True)
        idx, w = check_gate(r, None if use is None else use.astype(np.float64), b.K, **kw)
        assert rel_l2(r["out"], b.reference(x, idx, w)) <= REL_L2_TOL
    b.m.close()


def test_gate_of_64_experts_and_placement(orc):
    """The full expert count (vector path), with the experts moved to other slots."""
    b = Block(orc, E=64, K=8)
    bias = (np.random.default_rng(4).standard_normal(64) * 0.05).astype(np.float32)
    kw = dict(score="sigmoid", group=(8, 4), group_score="top2", norm=True, scale=1.0)
    b.m.set_gate(gate_of(64, 8, kw))
    b.m.set_balance_bias(0, bias)
    for T in (5, 130):
        r = b.m.forward_host(0, b.x(T), debug=True)
        idx, w = check_gate(r, bias.astype(np.float64), 8, **kw)
        assert rel_l2(r["out"], b.reference(b.x(T), idx, w)) <= REL_L2_TOL
        b.m.set_placement(0, np.random.default_rng(5).permutation(64).tolist())
        b.load(0, O.Q4_0)
        moved = b.m.forward_host(0, b.x(T), debug=True)
        np.testing.assert_array_equal(moved["idx"], r["idx"])
        assert rel_l2(moved["out"], b.reference(b.x(T), idx, w)) <= REL_L2_TOL
    b.m.close()


@pytest.mark.parametrize("T", [3, 20, 100])
def test_closed_experts_in_the_block(orc, T):
    """A router bias of -inf closes experts; with too few open ones entries stay empty."""
    b = Block(orc)
    kw = dict(score="softmax", norm=True, scale=1.0)
    b.m.set_gate(gate_of(b.E, b.K, kw))
    rb = np.zeros(b.E, np.float32)
    rb[3:] = -np.inf
    r = b.m.forward_host(0, b.x(T), bias=rb, debug=True)
    idx, w = check_gate(r, None, b.K, **kw)
    assert (idx[:, 3:] == -1).all()
    assert rel_l2(r["out"], b.reference(b.x(T), idx, w)) <= REL_L2_TOL
    b.m.set_placement(0, np.random.default_rng(5).permutation(b.E).tolist())
    b.load(0, O.Q4_0)
    moved = b.m.forward_host(0, b.x(T), bias=rb, debug=True)
    np.testing.assert_array_equal(moved["idx"], idx)
    b.m.set_placement(0, None)
    b.load(0, O.Q4_0)
    rb[:] = -np.inf  # nothing open: the shared expert alone
    r = b.m.forward_host(0, b.x(T), bias=rb, debug=True)
    assert (r["idx"] == -1).all() and (r["w"] == 0).all()
    assert rel_l2(r["out"], b.reference(b.x(T), r["idx"], r["w"])) <= REL_L2_TOL
    b.m.close()


def test_default_routing_comes_back(orc):
    b = Block(orc)
    x = b.x(70)
    first = b.m.forward_host(0, x, debug=True)
    b.m.set_gate(gate_of(b.E, b.K, GATES[0]))
    assert not np.array_equal(b.m.forward_host(0, x)["out"], first["out"])
    b.m.set_gate(None)
    assert np.array_equal(b.m.forward_host(0, x)["out"], first["out"])
    b.m.set_gate(gate_of(b.E, b.K, GATES[0]))
    b.m.set_routing(plain=True)  # the other routing call replaces the gate
    assert np.array_equal(b.m.forward_host(0, x)["out"], first["out"])
    # the softmax gate with renormalised weights is moe_forward_cpu's routing
    b.m.set_gate(hymoe.Gate(b.E, b.K))
    r = b.m.forward_host(0, x, debug=True)
    np.testing.assert_array_equal(r["idx"], first["idx"])
    np.testing.assert_allclose(r["w"], first["w"], rtol=2e-6)
    b.m.close()


@pytest.mark.parametrize("wt", [O.Q4_0, O.Q8_0, O.F16])
@pytest.mark.parametrize("T", [1, 2, 6, 8, 9, 33, 64, 65, 300])
def test_adapted_block(orc, wt, T):
    """Both projections, then each alone; every weight path (streaming, weight-block and
    tensor-core kernels)."""
    b = Block(orc, wt=wt)
    x, ids = b.x(T), ids_of(T)
    base = b.m.forward_host(0, x, debug=True)
    for use in (("gu", "dn"), ("gu",), ("dn",)):
        b.m.set_adapters(0, b.ad["gu"] if "gu" in use else None, b.ad["dn"] if "dn" in use else None)
        r = b.m.forward_host(0, x, debug=True, adapter_ids=ids)
        np.testing.assert_array_equal(r["idx"], base["idx"])
        want = b.reference(x, base["idx"].astype(np.int64), base["w"].astype(np.float64), ids, use)
        assert rel_l2(r["out"], want) <= REL_L2_TOL
        if (ids >= 0).any():
            assert rel_l2(base["out"], want) > 10 * REL_L2_TOL  # the adapters are a visible part
        none = ids < 0
        np.testing.assert_array_equal(b.m.forward_host(0, x)["out"], base["out"])  # left out by hymoe_forward
        if none.any():
            assert rel_l2(r["out"][none], base["out"][none]) <= REL_L2_TOL
    b.m.close()


def test_gate_and_adapters_together(orc):
    """As a serving layer uses them: RMSNorm, gate with bias and adapters in one call, host and
    device pointers, a replayed graph, chunked host copies."""
    T = 2100
    b = Block(orc, max_tokens=T)
    kw = GATES[2]
    bias = (np.random.default_rng(3).standard_normal(b.E) * 0.1).astype(np.float32)
    nw = (1.0 + 0.1 * np.random.default_rng(7).standard_normal(H)).astype(np.float32)
    b.m.set_gate(gate_of(b.E, b.K, kw))
    b.m.set_balance_bias(0, bias)
    b.m.set_adapters(0, b.ad["gu"], b.ad["dn"])
    b.m.set_norm(0, nw, 1e-5)
    for n in (7, 500, T):
        x, ids = b.x(n), ids_of(n)
        xn = b.orc.rms_norm(x, nw, 1e-5)
        r = b.m.forward_host(0, x, resid="x", debug=True, pre_norm=True, adapter_ids=ids)
        idx, w = check_gate(r, bias.astype(np.float64), b.K, **kw)
        want = x + b.reference(xn, idx, w, ids)
        assert rel_l2(r["out"], want) <= REL_L2_TOL
        plain = b.m.forward_host(0, x, resid="x", pre_norm=True, adapter_ids=ids)  # no debug: chunked where long
        assert rel_l2(plain["out"], want) <= REL_L2_TOL
        xd, idd = torch.from_numpy(x).cuda(), torch.from_numpy(ids).cuda()
        outs = [torch.zeros_like(xd) for _ in range(2)]
        torch.cuda.synchronize()
        for graph, o in ((False, outs[0]), (True, outs[1]), (True, outs[1])):
            b.m.forward_device(0, xd.data_ptr(), o.data_ptr(), n, resid_ptr=xd.data_ptr(), graph=graph, pre_norm=True,
                               adapter_ids_ptr=idd.data_ptr())
        b.m.synchronize()
        assert np.array_equal(outs[0].cpu().numpy(), r["out"]) and torch.equal(outs[0], outs[1])
        idd.copy_(torch.from_numpy(ids[::-1].copy()))  # the replay reads the ids of the moment
        torch.cuda.synchronize()
        b.m.forward_device(0, xd.data_ptr(), outs[1].data_ptr(), n, resid_ptr=xd.data_ptr(), graph=True, pre_norm=True,
                           adapter_ids_ptr=idd.data_ptr())
        b.m.synchronize()
        assert rel_l2(outs[1].cpu().numpy(), x + b.reference(xn, idx, w, ids[::-1])) <= REL_L2_TOL
    b.m.close()


def test_layers_keep_their_own(orc):
    b = Block(orc, layers=2)
    b.m.set_gate(gate_of(b.E, b.K, GATES[0]))
    bias = np.linspace(-0.3, 0.3, b.E).astype(np.float32)
    b.m.set_balance_bias(1, bias)
    b.m.set_adapters(1, None, b.ad["dn"])
    x, ids = b.x(30), ids_of(30)
    r0 = b.m.forward_host(0, x, debug=True)
    idx, w = check_gate(r0, None, b.K, **GATES[0])
    r1 = b.m.forward_host(1, x, debug=True, adapter_ids=ids)
    idx1, w1 = check_gate(r1, bias.astype(np.float64), b.K, **GATES[0])
    assert rel_l2(r1["out"], b.reference(x, idx1, w1, ids, ("dn",))) <= REL_L2_TOL
    with pytest.raises(hymoe.HymoeError):
        b.m.forward_host(0, x, adapter_ids=ids)  # layer 0 has no adapters
    b.m.set_adapters(1)
    with pytest.raises(hymoe.HymoeError):
        b.m.forward_host(1, x, adapter_ids=ids)
    b.m.close()


def test_operators_agree_with_the_block(orc):
    """hymoe_route on the block's logits, then the experts by a one-hot default routing: the same
    choices; hymoe_adapt beside the block gives what the block adds."""
    b = Block(orc)
    x, ids = b.x(90), ids_of(90)
    b.m.set_gate(gate_of(b.E, b.K, GATES[0]))
    r = b.m.forward_host(0, x, debug=True)
    got = gate_of(b.E, b.K, GATES[0]).route(torch.from_numpy(r["logits"]).cuda(), scores=True, counts=True)
    np.testing.assert_array_equal(got["idx"].cpu().numpy(), r["idx"])
    np.testing.assert_array_equal(got["weights"].cpu().numpy(), r["w"])
    np.testing.assert_array_equal(got["counts"].cpu().numpy(), np.bincount(r["idx"].ravel(), minlength=b.E))
    b.m.set_adapters(0, b.ad["gu"], None)
    assert rel_l2(b.m.forward_host(0, x, adapter_ids=np.full(90, -1, np.int32))["out"], r["out"]) <= 1e-6
    z = torch.from_numpy(x).cuda().half()
    delta = b.ad["gu"].apply(z, torch.from_numpy(ids).cuda(), base=torch.zeros(90, 2 * I, device="cuda"))
    assert rel_l2(delta.cpu().numpy(), b.delta("gu", z.double().cpu().numpy(), ids)) <= 1e-5
    b.m.close()


def test_refusals(orc):
    b = Block(orc)
    L, h = hymoe.lib(), b.m.h
    with pytest.raises(ValueError):
        b.m.set_gate(hymoe.Gate(b.E, b.K + 1))
    bad = hymoe.GateSpec(7, 0, 0, 0, 1, 1.0)
    assert L.hymoe_set_gate(h, C.byref(bad)) == 1
    assert L.hymoe_set_balance_bias(h, 9, None, 1) == 1
    assert L.hymoe_set_adapters(h, 9, None, None) == 1
    bf = hymoe.Adapters(torch.zeros(1, 8, H, device="cuda", dtype=torch.bfloat16), torch.zeros(1, 2 * I, 8, device="cuda", dtype=torch.bfloat16))
    assert L.hymoe_set_adapters(h, 0, C.byref(bf.spec), None) == 4
    assert L.hymoe_set_adapters(h, 0, C.byref(b.ad["dn"].spec), None) == 1  # the other projection's sizes
    assert L.hymoe_forward_adapted(h, 9, None, None, None, 0, None, None, None, 0) == 1
    assert L.hymoe_forward_adapted(h, 0, None, None, None, 0, None, None, None, 0) == 7
    b.m.close()
