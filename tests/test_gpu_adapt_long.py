"""GPU tests of hymoe_adapt and hymoe_adapt_backward for long batches of rows on 16-byte boundaries,
whose products run on the 5th-generation tensor cores: tiles of consecutive tokens, of scattered ones
and without an adapter beside one another, widths that end inside a tile, gradients of long adapters
in pieces.  The tolerances are those of test_gpu_adapt.py."""
import pytest

import hymoe
from test_gpu_adapt import Problem, check, near

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def runs(*parts):
    """(length, adapters in turn) ..."""
    return torch.cat([torch.tensor(who, dtype=torch.int32).repeat(-(-n // len(who)))[:n] for n, who in parts]).cuda()


MIXES = {
    "runs": [(200, [2]), (130, [0]), (333, [3]), (1, [1])],
    "scattered": [(777, [3, 0, 1, 2, 0])],
    "both": [(200, [2]), (301, [0, 1]), (150, [-1]), (333, [3]), (64, [2])],
    "gaps": [(129, [-1]), (128, [1]), (3, [-1]), (400, [0, -1])],
    "one_of_four": [(700, [3])],
}


def with_ids(ids, *shape, **kw):
    p = Problem(len(ids), *shape, **kw)
    p.ids = ids
    return p


@pytest.mark.parametrize("mix", MIXES)
@pytest.mark.parametrize("n_in,n_out,rank", [(64, 72, 8), (72, 264, 24), (520, 1000, 16), (320, 136, 128), (1032, 64, 64)])
@pytest.mark.parametrize("types", [("bf16", "bf16", "bf16"), ("f16", "f16", "f16"), ("f16", "f16", "f32")], ids="-".join)
def test_mixes(mix, n_in, n_out, rank, types):
    x, w, y = types
    p = with_ids(runs(*MIXES[mix]), n_in, n_out, rank, 4, x=x, w=w, y=y)
    check(p)
    p.base = p.base_x = None
    out = check(p)
    free = (p.ids < 0).nonzero().flatten()
    assert not bool(out[free].any())


@pytest.mark.parametrize("mix", ["both", "gaps"])
@pytest.mark.parametrize("y", ["bf16", "f32"])
def test_in_place(mix, y):
    p = with_ids(runs(*MIXES[mix]), 256, 392, 32, 4, y=y)
    want = p.adapters.apply(p.x, p.ids, base=p.base)
    got = p.base.clone()
    p.adapters.apply(p.x, p.ids, base=got, out=got)
    assert torch.equal(got, want)
    free = (p.ids < 0).nonzero().flatten()
    assert torch.equal(got[free], p.base[free])


@pytest.mark.parametrize("w", ["bf16", "f16"])
@pytest.mark.parametrize("T,n", [(1300, 1), (2048, 2), (5000, 7), (4097, 300)])
def test_thousands_of_tokens(T, n, w):
    check(Problem(T, 264, 512, 16, n, ids="one" if n == 1 else "requests", x=w, w=w, y=w))
    ids = torch.full((T,), n - 1, dtype=torch.int32, device="cuda")
    ids[::50] = 0  # one long adapter in pieces, one short, the others without tokens
    check(with_ids(ids, 264, 512, 16, n, x=w, w=w, y=w))


@pytest.mark.parametrize("T", [300, 700])
@pytest.mark.parametrize("ids", ["mixed", "requests"])
@pytest.mark.parametrize("w", ["bf16", "f16"])
def test_infinities_stay_in_their_rows_and_adapters(T, ids, w):
    p = Problem(T, 200, 136, 16, 3, ids=ids, x=w, w=w, y=w)
    want, g = p.adapters.apply(p.x, p.ids, base=p.base), p.adapters.backward(p.x, p.dy, p.ids, base=p.base_x)
    at = [t for t in (p.ids == 1).nonzero().flatten().tolist()][3:9:5]
    p.x[at[0], 5], p.x[at[1], 0] = float("inf"), float("nan")
    p.dy[at[0], 7] = float("-inf")
    got, bad = p.adapters.apply(p.x, p.ids, base=p.base), p.adapters.backward(p.x, p.dy, p.ids, base=p.base_x)
    rest = [t for t in range(T) if t not in at]
    assert torch.equal(got[rest], want[rest]) and not bool(torch.isfinite(got[at]).any())
    rest = [t for t in range(T) if t != at[0]]
    assert torch.equal(bad["dx"][rest], g["dx"][rest]) and not bool(torch.isfinite(bad["dx"][at[0]]).any())
    for k in (0, 2):
        assert torch.equal(bad["da"][k], g["da"][k]) and torch.equal(bad["db"][k], g["db"][k])
    assert not bool(torch.isfinite(bad["da"][1]).any()) and not bool(torch.isfinite(bad["db"][1]).any())
    # without an adapter the same inputs do not matter
    p.ids[at] = -1
    got, g = p.adapters.apply(p.x, p.ids, base=p.base), p.adapters.backward(p.x, p.dy, p.ids)
    assert torch.equal(got[at], p.base[at])
    assert all(bool(torch.isfinite(v).all()) for v in g.values())


def test_strides():
    """Aligned rows inside wider buffers; what lies between stays as it was."""
    for off, pad in ((0, 8), (8, 24), (64, 64)):
        p = with_ids(runs(*MIXES["both"]), 128, 200, 16, 4)

        def wide(t):
            ld = t.shape[1] + pad
            buf = torch.full((t.shape[0] * ld + off,), 3.0, dtype=t.dtype, device="cuda")
            v = buf.as_strided(t.shape, (ld, 1), off)
            v.copy_(t)
            return v, buf

        p.x, p.dy, p.base, p.base_x = (wide(t)[0] for t in (p.x, p.dy, p.base, p.base_x))
        out, buf = wide(torch.zeros(p.T, 200, dtype=torch.bfloat16, device="cuda"))
        before = buf.clone()
        check(p, out=out)
        mask = torch.ones_like(buf, dtype=torch.bool)
        mask.as_strided(out.shape, out.stride(), off).fill_(False)
        assert torch.equal(buf[mask], before[mask])


@pytest.mark.parametrize("std", [1e4, 1e-6])
def test_large_and_tiny_values(std):
    """fp16 gradients of intermediates beyond fp16's range either way keep their digits."""
    p = Problem(400, 256, 128, 16, 3, x="f16", w="f16", y="f32")
    p.x = (p.x.float() * std).clamp(-6e4, 6e4).half()
    check(p)
    p = Problem(400, 256, 128, 16, 3, x="f16", w="f16", y="f16", base=False)
    p.base_x = None
    p.dy = (p.dy.float() * std).clamp(-6e4, 6e4).half()
    p.x = (p.x.float() / std).clamp(-6e4, 6e4).half()
    got = p.adapters.backward(p.x, p.dy, p.ids, want=("da", "db"))
    want, mag = p.gradients(), p.gradients(True)
    near(got["da"], want["da"], mag["da"], None, p.n_out + p.T)
    near(got["db"], want["db"], mag["db"], None, p.n_in + p.T)


def test_gradients_one_by_one_and_empty_adapters():
    ids = runs((300, [0]), (700, [1, 3, 3]), (40, [-1]))
    p = with_ids(ids, 136, 264, 24, 6)
    both = p.adapters.backward(p.x, p.dy, p.ids, base=p.base_x)
    for k in (2, 4, 5):
        assert not bool(both["da"][k].any()) and not bool(both["db"][k].any())
    for name in ("dx", "da", "db"):
        one = p.adapters.backward(p.x, p.dy, p.ids, base=p.base_x if name == "dx" else None, want=(name,))
        assert list(one) == [name] and torch.equal(one[name], both[name])


def test_same_bits_every_time():
    for w in ("bf16", "f16"):
        p = with_ids(runs(*MIXES["both"], (900, [1])), 264, 520, 32, 4, x=w, w=w, y=w)
        out, g = p.adapters.apply(p.x, p.ids, base=p.base), p.adapters.backward(p.x, p.dy, p.ids, base=p.base_x)
        for _ in range(5):
            assert torch.equal(p.adapters.apply(p.x, p.ids, base=p.base), out)
            again = p.adapters.backward(p.x, p.dy, p.ids, base=p.base_x)
            assert all(torch.equal(g[k], again[k]) for k in g)


def test_other_types_beside_the_weights():
    """fp32 rows on one side only: each product takes its own path over one plan."""
    for x, y in (("f32", "bf16"), ("bf16", "f32")):
        p = with_ids(runs(*MIXES["both"]), 256, 264, 16, 4, x=x, y=y)
        check(p)


@pytest.mark.parametrize("T", [100, 300])
def test_workspace_as_it_comes(T):
    """Whatever the workspace holds before the call; its first word says afterwards that no wait expired."""
    p = Problem(T, 256, 264, 16, 4)
    ad = p.adapters
    want, grads = ad.apply(p.x, p.ids, base=p.base), ad.backward(p.x, p.dy, p.ids, base=p.base_x)
    mat = lambda t: hymoe.Mat(t.data_ptr(), 30, t.shape[1])
    for fill in (0, 0xFF, 0x7F):
        ws = torch.full((ad._workspace_bytes(T, True),), fill, dtype=torch.uint8, device="cuda")
        out = torch.full_like(want, float("nan"))
        n = ad._workspace_bytes(T, False)
        stream = torch.cuda.current_stream().cuda_stream
        assert ad.L.hymoe_adapt(ad._spec, mat(p.x), p.ids.data_ptr(), T, mat(p.base), mat(out), ws.data_ptr(), n, stream) == 0
        torch.cuda.synchronize()
        assert torch.equal(out, want) and not bool(ws[:4].any()) and bool((ws[n:] == fill).all())
        ws.fill_(fill)
        dx, da, db = (torch.full_like(grads[k], float("nan")) for k in ("dx", "da", "db"))
        assert ad.L.hymoe_adapt_backward(ad._spec, mat(p.x), mat(p.dy), p.ids.data_ptr(), T, mat(p.base_x), mat(dx), da.data_ptr(),
                                         db.data_ptr(), ws.data_ptr(), ws.numel(), stream) == 0
        torch.cuda.synchronize()
        assert not bool(ws[:4].any())
        assert all(torch.equal(a, grads[k]) for k, a in (("dx", dx), ("da", da), ("db", db)))


@pytest.mark.parametrize("shape,kw", [
    ((5000, 72, 64, 8, 4096), {}),                                        # most adapters, about a token each
    ((200, 128, 136, 128, 4096), dict(x="f16", w="f16", y="f32")),        # fewer tokens than adapters
    ((130, 1 << 20, 64, 8, 2), {}),                                       # the longest rows to read
    ((130, 64, 1 << 20, 8, 2), dict(x="f16", w="f16", y="f16")),          # and to write
    ((90, 1 << 20, 72, 1, 1), dict(ids="one")),
    ((33000, 64, 72, 16, 2), dict(ids="requests")),                       # long sums
    ((70001, 64, 64, 8, 9), dict(x="f32", y="f32"))])
def test_largest_sizes(shape, kw):
    check(Problem(*shape, **kw))
