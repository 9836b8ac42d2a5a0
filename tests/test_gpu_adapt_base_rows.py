"""GPU test of hymoe_adapt for tokens without an adapter: their rows are the base's, bit for bit (signs
of zeros, NaN and infinities as they are), however few tokens the call has."""
import pytest

import hymoe

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"bf16": (torch.bfloat16, torch.int16), "f16": (torch.float16, torch.int16), "f32": (torch.float32, torch.int32)}


@pytest.mark.parametrize("w,y", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("n_in,n_out", [(128, 136), (63, 33)])
@pytest.mark.parametrize("T", [1, 5, 40, 100, 300])
def test_rows_without_an_adapter(T, n_in, n_out, w, y):
    g = torch.Generator(device="cuda")
    g.manual_seed(T)
    x = torch.randn((T, n_in), generator=g, device="cuda").to(TYPES[w][0])
    a = torch.randn((2, 8, n_in), generator=g, device="cuda").to(TYPES[w][0])
    b = torch.randn((2, n_out, 8), generator=g, device="cuda").to(TYPES[w][0])
    base = torch.randn((T, n_out), generator=g, device="cuda")
    special = torch.tensor([0.0, -0.0, float("inf"), float("-inf"), 1e-40, -1e-7], device="cuda")
    base[:, :30] = special.repeat(5)
    base = base.to(TYPES[y][0])
    bits = base.view(TYPES[y][1])
    bits[:, 31] = (0x7F800000 | 0x155555) if y == "f32" else 0x7FD5 if y == "bf16" else 0x7F55  # a NaN of its own
    ids = torch.full((T,), -1, dtype=torch.int32, device="cuda")
    ids[1::3] = 1
    out = torch.zeros_like(base)
    hymoe.Adapters(a, b).apply(x, ids, base=base, out=out)
    rows = ids < 0
    assert torch.equal(out.view(TYPES[y][1])[rows], bits[rows])
    none = hymoe.Adapters(a, b).apply(x, ids, out=torch.full_like(base, 5.0))
    assert not bool(none.view(TYPES[y][1])[rows].any())
