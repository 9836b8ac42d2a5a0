"""GPU tests of a layer's small parameters set from device memory (hymoe_set_balance_bias,
hymoe_set_norm): the copy has landed when the call returns, whatever is queued on other streams, and
follows what the caller queued on the default stream."""
import numpy as np
import pytest

import hymoe
from test_gpu_block_gate_adapters import GATES, Block, check_gate, gate_of

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

BUSY = 200_000_000  # cycles: about a tenth of a second of the default stream


def forward(b, x, **kw):
    """A device-pointer call on the context's own stream, right away."""
    xd = torch.from_numpy(x).cuda()
    out, logits = torch.zeros_like(xd), torch.zeros(len(x), b.E, device="cuda")
    idx, w = torch.zeros(len(x), b.K, dtype=torch.int32, device="cuda"), torch.zeros(len(x), b.K, device="cuda")
    probs = torch.zeros(len(x), b.E, device="cuda")
    torch.cuda.synchronize()
    dbg = hymoe.Debug(logits.data_ptr(), probs.data_ptr(), w.data_ptr(), idx.data_ptr())

    def run(before):
        before()
        b.m.forward_device(0, xd.data_ptr(), out.data_ptr(), len(x), dbg=dbg, **kw)
        b.m.synchronize()
        torch.cuda.synchronize()
        return {"out": out.cpu().numpy(), "logits": logits.cpu().numpy(), "probs": probs.cpu().numpy(),
                "idx": idx.cpu().numpy(), "w": w.cpu().numpy()}

    return run


@pytest.mark.parametrize("source", ["device", "host"])
def test_balance_bias_has_landed(orc, source):
    b = Block(orc)
    b.m.set_gate(gate_of(b.E, b.K, GATES[0]))
    run = forward(b, b.x(20))
    g = np.random.default_rng(11)
    for turn in range(4):  # the first call allocates the layer's bias, the others replace it
        bias = g.standard_normal(b.E).astype(np.float32)
        src = torch.from_numpy(bias).cuda() if source == "device" else bias.copy()
        torch.cuda.synchronize()

        def before():
            torch.cuda._sleep(BUSY)
            if source == "device":
                assert hymoe.lib().hymoe_set_balance_bias(b.m.h, 0, src.data_ptr(), 0) == 0
                with torch.cuda.stream(torch.cuda.Stream()):
                    src.fill_(float("nan"))  # it was copied
            else:
                b.m.set_balance_bias(0, src)
                src[:] = np.nan

        check_gate(run(before), bias.astype(np.float64), b.K, **GATES[0])
    b.m.close()


def test_balance_bias_follows_the_default_stream(orc):
    b = Block(orc)
    b.m.set_gate(gate_of(b.E, b.K, GATES[0]))
    run = forward(b, b.x(20))
    bias = np.random.default_rng(12).standard_normal(b.E).astype(np.float32)
    src, value = torch.zeros(b.E, device="cuda"), torch.from_numpy(bias).cuda()
    torch.cuda.synchronize()

    def before():
        torch.cuda._sleep(BUSY)
        src.copy_(value)
        assert hymoe.lib().hymoe_set_balance_bias(b.m.h, 0, src.data_ptr(), 0) == 0

    check_gate(run(before), bias.astype(np.float64), b.K, **GATES[0])
    b.m.close()


def test_norm_has_landed(orc):
    b = Block(orc)
    x = b.x(20)
    g = np.random.default_rng(13)
    run = forward(b, x, pre_norm=True)
    for turn in range(3):
        nw = (1.0 + 0.5 * g.standard_normal(x.shape[1])).astype(np.float32)
        b.m.set_norm(0, nw, 1e-5)
        torch.cuda.synchronize()
        want = b.m.forward_host(0, x, pre_norm=True)["out"]
        b.m.set_norm(0, np.ones_like(nw), 1e-5)
        src = torch.from_numpy(nw).cuda()
        torch.cuda.synchronize()

        def before():
            torch.cuda._sleep(BUSY)
            assert hymoe.lib().hymoe_set_norm(b.m.h, 0, src.data_ptr(), 1e-5, 0) == 0

        np.testing.assert_array_equal(run(before)["out"], want)
    b.m.close()


def test_balance_bias_of_the_wrong_memory_is_refused(orc):
    """A host pointer given as device memory: refused, and the layer has no bias (or the one it had)."""
    b = Block(orc)
    b.m.set_gate(gate_of(b.E, b.K, GATES[0]))
    L, wrong = hymoe.lib(), np.full(b.E, 7.0, np.float32)
    wrong[::2] = -7.0
    x, bias = b.x(20), np.random.default_rng(14).standard_normal(b.E).astype(np.float32)
    for use in (None, bias):
        b.m.set_balance_bias(0, use)
        assert L.hymoe_set_balance_bias(b.m.h, 0, wrong.ctypes.data, 0) == 1
        assert "device" in L.hymoe_last_error(b.m.h).decode()
        check_gate(b.m.forward_host(0, x, debug=True), None if use is None else use.astype(np.float64), b.K, **GATES[0])
    b.m.close()
