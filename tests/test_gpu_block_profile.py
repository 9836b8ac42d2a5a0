"""GPU test of hymoe_profile for calls with adapters: their launches and time count in the phase of the
projection that they join."""
import numpy as np
import pytest

import hymoe
from test_gpu_block_gate_adapters import H, I, Block, ids_of

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("T,launches", [(6, 1), (32, 1), (65, 3), (400, 3)])
def test_adapters_are_in_their_phases(orc, T, launches):
    b = Block(orc)
    g = torch.Generator().manual_seed(1)
    wide = {k: hymoe.Adapters(torch.randn(3, 128, i, generator=g).half().cuda(), (torch.randn(3, o, 128, generator=g) * 0.01).half().cuda())
            for k, (i, o) in {"gu": (H, 2 * I), "dn": (I, H)}.items()}
    x, ids = b.x(T), ids_of(T)

    def phases(use):
        if use:
            b.m.set_adapters(0, wide["gu"] if "gu" in use else None, wide["dn"] if "dn" in use else None)
        kw = {"adapter_ids": ids} if use else {}
        b.m.forward_host(0, x, **kw)
        b.m.profile(True)
        for _ in range(20):
            b.m.forward_host(0, x, **kw)
        b.m.profile(False)
        return b.m.profile_read()

    plain = phases(())
    for use in (("gu",), ("dn",), ("gu", "dn")):
        got = phases(use)
        for phase, name in (("gate_up", "gu"), ("down", "dn")):
            more = 20 * launches if name in use else 0
            # (without adapters 4 to 8 tokens run the shared expert apart, which is a launch of its own)
            (ms, n), (ms0, n0) = got[phase], plain[phase]
            assert n - more <= n0 and n >= 20 + more
            assert ms > 0
    assert np.isfinite([ms for ms, n in got.values()]).all()
    b.m.close()
