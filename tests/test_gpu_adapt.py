"""GPU tests of hymoe_adapt and hymoe_adapt_backward against double precision.

Tolerances.  With m the sum of a result's terms' magnitudes and n the length of its sums, fp32
sums that lose at most 2^-23 of the running sum in each of n / 16 + 32 steps are off by at most
(n / 16 + 32) 2^-23 m in every element.  In the 2-norm the running sum of n random terms is about
sqrt(k) after k terms, which makes 2/3 of that of the last one, over n / 16 steps: n / 24 steps of
2^-23 of the result, and 24 more for the other roundings.  A 16-bit result is rounded once (half a
step) from an intermediate that may be held in two 16-bit parts (2^-16); an fp32 result's
intermediate is held to 2^-21."""
import pytest

import hymoe

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
PARTS = {torch.float32: 2.0 ** -21, torch.float16: 2.0 ** -16, torch.bfloat16: 2.0 ** -16}
SMALLEST = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}
T16 = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


class Problem:
    def __init__(self, T, n_in, n_out, rank, n, ids="mixed", x="bf16", w="bf16", y="bf16", base=True, scale=True, seed=0,
                 x_std=1.0, b_std=0.05):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)

        def normal(shape, std, dtype):
            return (torch.randn(shape, generator=g, device="cuda") * std).to(T16[dtype])

        self.T, self.n_in, self.n_out, self.rank, self.n = T, n_in, n_out, rank, n
        self.x = normal((T, n_in), x_std, x)
        self.a, self.b = normal((n, rank, n_in), n_in ** -0.5, w), normal((n, n_out, rank), b_std, w)
        self.base = normal((T, n_out), 0.5, y) if base else None
        self.base_x = normal((T, n_in), 0.5, x) if base else None
        self.dy = normal((T, n_out), x_std, y)
        self.scale = torch.rand((n,), generator=g, device="cuda") + 0.5 if scale else None
        if ids == "mixed":  # any order, some without an adapter, some adapters perhaps without tokens
            self.ids = torch.randint(-1, n, (T,), generator=g, device="cuda").to(torch.int32)
        elif ids == "requests":
            self.ids = torch.sort(torch.randint(0, n, (T,), generator=g, device="cuda")).values.flip(0).to(torch.int32)
        elif ids == "foreign":  # ids far outside the range, and one adapter only
            self.ids = torch.tensor([0, -1, n, 1 << 30, -(1 << 31), n - 1], device="cuda")[torch.arange(T, device="cuda") % 6].to(torch.int32)
        elif ids == "none":
            self.ids = torch.full((T,), -1, dtype=torch.int32, device="cuda")
        else:  # one adapter for all, by no ids
            self.ids = None
        self.adapters = hymoe.Adapters(self.a, self.b, self.scale)
        self.y_type = T16[y]

    def rows(self):
        for k in range(self.n):
            yield k, (torch.arange(self.T, device="cuda") if self.ids is None and k == 0 else
                      torch.arange(0, device="cuda") if self.ids is None else (self.ids == k).nonzero().flatten())

    def f(self, k):
        return 1.0 if self.scale is None else self.scale[k].double()

    def forward(self, mag=False):
        z = torch.abs if mag else (lambda v: v)
        out = torch.zeros(self.T, self.n_out, dtype=torch.double, device="cuda")
        for k, r in self.rows():
            low = z(self.x[r].double()) @ z(self.a[k].double()).t()
            out[r] = self.f(k) * (low @ z(self.b[k].double()).t())
        return out

    def gradients(self, mag=False):
        z = torch.abs if mag else (lambda v: v)
        dx = torch.zeros(self.T, self.n_in, dtype=torch.double, device="cuda")
        da = torch.zeros(self.a.shape, dtype=torch.double, device="cuda")
        db = torch.zeros(self.b.shape, dtype=torch.double, device="cuda")
        for k, r in self.rows():
            x, dy, a, b = z(self.x[r].double()), z(self.dy[r].double()), z(self.a[k].double()), z(self.b[k].double())
            u = self.f(k) * (dy @ b)
            dx[r] = u @ a
            da[k] = u.t() @ x
            db[k] = self.f(k) * (dy.t() @ (x @ a.t()))
        return {"dx": dx, "da": da, "db": db}


def near(got, want, mag, base, n):
    """`want` and `mag`: the products' part; base: added to both (None: 0)."""
    t = got.dtype
    full = want if base is None else want + base.double()
    size = mag if base is None else mag + base.double().abs()
    err = (got.double() - full).abs()
    lim = (n / 16 + 32) * 2.0 ** -23 * size + PARTS[t] * mag + 1.01 * HALF_STEP[t] * full.abs() + SMALLEST[t]
    # Rounding to nearest gives infinity from the largest number plus half its step on (fp16: 65504 +
    # 16 = 65520).  A sum within its bound of that border may go either way: where the result is
    # infinite, the sum itself has to reach it.
    border = torch.finfo(t).max * (1 + torch.finfo(t).eps / 4)
    beyond = got.isinf() & (got.sign() == full.sign()) & (full.abs() + lim >= border)
    full, want, err = (torch.where(beyond, 0.0, v) for v in (full, want, err))
    assert bool((err <= lim).all()), f"element off by {float((err / lim).max()):.2f} of its bound"
    two = (n / 24 + 24) * 2.0 ** -23 * float(full.norm()) + (PARTS[t] + (n / 24 + 24) * 2.0 ** -23) * float(want.norm())
    two += HALF_STEP[t] * float(full.norm()) + SMALLEST[t] * max(1, full.numel()) ** 0.5
    assert float(err.norm()) <= two, f"2-norm {float(err.norm()):.3e} over {two:.3e}"


def check(p, grads=True, **kw):
    out = p.adapters.apply(p.x, p.ids, base=p.base, **kw)
    near(out, p.forward(), p.forward(True), p.base, p.n_in + p.rank)
    if grads:
        check_grads(p)
    return out


def check_grads(p):
    got = p.adapters.backward(p.x, p.dy, p.ids, base=p.base_x)
    want, mag = p.gradients(), p.gradients(True)
    near(got["dx"], want["dx"], mag["dx"], p.base_x, p.n_out + p.rank)
    near(got["da"], want["da"], mag["da"], None, p.n_out + p.T)
    near(got["db"], want["db"], mag["db"], None, p.n_in + p.T)
    return got


SHAPES = [  # T, in, out, rank, adapters
    (1, 128, 128, 8, 1), (1, 256, 64, 16, 4), (2, 64, 264, 4, 2), (3, 512, 512, 64, 3), (5, 136, 72, 1, 2),
    (8, 1024, 768, 32, 8), (16, 256, 256, 128, 5), (31, 128, 640, 16, 3), (33, 320, 192, 24, 33), (64, 512, 384, 64, 4),
    (65, 256, 256, 16, 1), (100, 128, 128, 128, 7), (129, 512, 520, 40, 2), (200, 264, 128, 12, 64),
    (257, 640, 256, 64, 5), (513, 256, 1032, 8, 3), (1000, 128, 192, 16, 130)]


@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
@pytest.mark.parametrize("types", [("bf16", "bf16", "bf16"), ("f16", "f16", "f32"), ("f32", "bf16", "f32"), ("f32", "f16", "f16")],
                         ids="-".join)
def test_shapes(shape, types):
    x, w, y = types
    check(Problem(*shape, x=x, w=w, y=y))


@pytest.mark.parametrize("ids", ["requests", "foreign", "none", "one"])
@pytest.mark.parametrize("T", [1, 6, 40, 300])
def test_ids(ids, T):
    check(Problem(T, 256, 136, 16, 5, ids=ids))
    check(Problem(T, 128, 128, 8, 3, ids=ids, base=False, scale=False, x="f16", w="f16", y="f32"))


@pytest.mark.parametrize("T", [1, 9, 70, 140])
@pytest.mark.parametrize("n_in,n_out,rank", [(1, 1, 1), (7, 5, 3), (65, 33, 17), (127, 129, 127), (100, 97, 8), (96, 100, 5)])
def test_odd_sizes(T, n_in, n_out, rank):
    """Rows that are not whole 16-byte pieces."""
    check(Problem(T, n_in, n_out, rank, 3))
    check(Problem(T, n_in, n_out, rank, 2, x="f32", w="f16", y="f32"))


@pytest.mark.parametrize("T", [4, 90])
def test_strides_and_alignment(T):
    """Rows inside wider buffers, starting at odd elements; what lies between stays as it was."""
    for off, pad in ((0, 8), (8, 24), (1, 7), (3, 0)):
        p = Problem(T, 128, 192, 16, 4)

        def wide(t):
            ld = t.shape[1] + pad
            buf = torch.full((t.shape[0] * ld + off,), 3.0, dtype=t.dtype, device="cuda")
            v = buf.as_strided(t.shape, (ld, 1), off)
            v.copy_(t)
            return v, buf

        p.x, _ = wide(p.x)
        p.dy, _ = wide(p.dy)
        p.base, _ = wide(p.base)
        p.base_x, _ = wide(p.base_x)
        out, buf = wide(torch.zeros(T, 192, dtype=torch.bfloat16, device="cuda"))
        before = buf.clone()
        check(p, out=out)
        mask = torch.ones_like(buf, dtype=torch.bool)
        mask.as_strided(out.shape, out.stride(), off).fill_(False)
        assert torch.equal(buf[mask], before[mask])


def test_unaligned_weights():
    """Adapters that start at an odd element of a larger buffer."""
    p = Problem(70, 128, 128, 16, 3)
    for off in (1, 4):
        bufs = []
        for t in (p.a, p.b):
            buf = torch.zeros(t.numel() + off, dtype=t.dtype, device="cuda")
            buf[off:].copy_(t.reshape(-1))
            bufs.append(buf[off:].view(t.shape))
        p.adapters = hymoe.Adapters(bufs[0], bufs[1], p.scale)
        check(p)
        p.x, p.dy, p.base, p.base_x, p.ids, p.T = p.x[:5], p.dy[:5], p.base[:5], p.base_x[:5], p.ids[:5], 5
        check(p)
        p = Problem(70, 128, 128, 16, 3)


@pytest.mark.parametrize("T", [3, 50, 200])
def test_in_place(T):
    p = Problem(T, 256, 128, 16, 4)
    want = p.adapters.apply(p.x, p.ids, base=p.base)
    y = p.base.clone()
    assert p.adapters.apply(p.x, p.ids, base=y, out=y) is y and torch.equal(y, want)


def test_rows_behind_the_last_token():
    p = Problem(77, 128, 128, 16, 4)
    big = torch.full((90, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    p.adapters.apply(p.x, p.ids, base=p.base, out=big[:77])
    assert bool((big[77:] == 5.0).all())


@pytest.mark.parametrize("T", [2, 80])
def test_large_and_tiny_values(T):
    """Intermediates beyond fp16's range either way keep their digits."""
    for std in (3e4, 1e-5):
        p = Problem(T, 512, 128, 16, 3, x="f16", w="f16", y="f32", base=False)
        p.x = (p.x.float() * std).clamp(-6e4, 6e4).half()
        p.dy = p.dy * (std if std < 1 else 1e6)
        check(p)
    p = Problem(T, 256, 128, 32, 3, x="f32", w="f16", y="f32", base=False, x_std=1e-7)
    check(p)
    p = Problem(T, 256, 128, 32, 3, x="f32", w="bf16", y="f32", base=False, x_std=1e9)
    check(p)


@pytest.mark.parametrize("T", [4, 100])
def test_infinities_stay_in_their_rows(T):
    """A token whose inputs are not finite spoils its own row, whatever shares its tile."""
    p = Problem(T, 128, 128, 16, 2, ids="requests")
    want = p.adapters.apply(p.x, p.ids, base=p.base)
    p.x[1, 5], p.x[3, 0] = float("inf"), float("nan")
    got = p.adapters.apply(p.x, p.ids, base=p.base)
    rest = [t for t in range(T) if t not in (1, 3)]
    assert torch.equal(got[rest], want[rest])
    assert not bool(torch.isfinite(got[[1, 3]]).any())
    # a token without an adapter: its input does not matter
    ids = p.ids.clone()
    ids[[1, 3]] = -1
    got = p.adapters.apply(p.x, ids, base=p.base)
    assert torch.equal(got[[1, 3]], p.base[[1, 3]]) and torch.equal(got[rest], want[rest])
    g = p.adapters.backward(p.x, p.dy, ids)
    assert all(bool(torch.isfinite(v).all()) for v in g.values())


def test_gradients_one_by_one_and_empty_adapters():
    p = Problem(150, 128, 256, 16, 6, ids="mixed")
    p.ids[p.ids == 2] = 4  # adapter 2 has no tokens
    p2 = p.adapters.backward(p.x, p.dy, p.ids, base=p.base_x)
    assert float(p2["da"][2].abs().max()) == 0 and float(p2["db"][2].abs().max()) == 0
    for name in ("dx", "da", "db"):
        one = p.adapters.backward(p.x, p.dy, p.ids, base=p.base_x if name == "dx" else None, want=(name,))
        assert list(one) == [name] and torch.equal(one[name], p2[name])
    z = p.adapters.backward(p.x[:0], p.dy[:0], p.ids[:0])
    assert float(z["da"].abs().max()) == 0 and float(z["db"].abs().max()) == 0 and z["dx"].shape == (0, 128)


def test_gradients_against_differences():
    """The loss <dy, out> is linear in x and in each of a and b: a difference of any width gives its
    slope, up to the rounding of double precision."""
    p = Problem(40, 24, 16, 4, 3, x="f32", w="f16", y="f32")
    got = p.adapters.backward(p.x, p.dy, p.ids)
    mags = p.gradients(True)
    base = float((p.forward() * p.dy.double()).sum())

    def slope(t, at, h):
        keep = t[at].clone()
        t[at] = keep + h
        d = (float((p.forward() * p.dy.double()).sum()) - base) / float(t[at].double() - keep.double())
        t[at] = keep
        return d

    g = torch.Generator().manual_seed(1)
    for name, t, n in (("dx", p.x, 20), ("da", p.a, 64), ("db", p.b, 64)):
        for _ in range(12):
            at = tuple(int(torch.randint(0, s, (1,), generator=g)) for s in t.shape)
            lim = (n / 16 + 32) * 2.0 ** -23 * float(mags[name][at]) + 1e-7
            assert abs(slope(t, at, 1.0) - float(got[name][at])) <= lim, (name, at)


def test_same_bits_every_time():
    for T in (7, 64, 900):
        p = Problem(T, 256, 512, 32, 5)
        first = p.adapters.apply(p.x, p.ids, base=p.base)
        g1 = p.adapters.backward(p.x, p.dy, p.ids, base=p.base_x)
        for _ in range(5):
            assert torch.equal(p.adapters.apply(p.x, p.ids, base=p.base), first)
            g2 = p.adapters.backward(p.x, p.dy, p.ids, base=p.base_x)
            assert all(torch.equal(g1[k], g2[k]) for k in g1)


@pytest.mark.parametrize("T", [5, 300])
def test_graph_and_streams(T):
    """Two captured graphs and eager calls on two streams, with changed inputs and ids."""
    ps = [Problem(T, 256, 384, 16, 4, seed=s) for s in (1, 2)]
    live = [dict(x=p.x.clone(), dy=p.dy.clone(), ids=p.ids.clone(), base=p.base.clone()) for p in ps]
    graphs, outs = [], []
    for p, v in zip(ps, live):
        p.adapters.apply(v["x"], v["ids"], base=v["base"])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = p.adapters.apply(v["x"], v["ids"], base=v["base"])
            d = p.adapters.backward(v["x"], v["dy"], v["ids"])
        graphs.append(g)
        outs.append((o, d))
    for turn in range(3):
        for p, v in zip(ps, live):
            p.x, p.ids = p.x.roll(1, 0).contiguous(), p.ids.roll(turn + 1, 0).contiguous()
            v["x"].copy_(p.x)
            v["ids"].copy_(p.ids)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        eager = []
        for s, p in zip(streams, ps):
            with torch.cuda.stream(s):
                eager.append(p.adapters.apply(p.x, p.ids, base=p.base))
        torch.cuda.synchronize()
        for p, (o, d), e in zip(ps, outs, eager):
            assert torch.equal(o, e)
            near(o, p.forward(), p.forward(True), p.base, 256 + 16)
            g = p.adapters.backward(p.x, p.dy, p.ids)
            assert all(torch.equal(g[k], d[k]) for k in g)


def test_largest_ranges():
    """The block's own sizes, and a batch of more than 2^31 elements in its output's buffer."""
    check(Problem(4160, 4096, 4096, 16, 3, ids="requests", x="f16", w="f16", y="f32"))
    p = Problem(300, 64, 64, 8, 3, base=False)
    ld = 1 << 23  # 300 rows of 2^23 elements: 2^31 and more between the first and the last
    buf = torch.empty(299 * ld + 64, dtype=torch.bfloat16, device="cuda")
    out = buf.as_strided((300, 64), (ld, 1))
    want = p.adapters.apply(p.x, p.ids)
    p.adapters.apply(p.x, p.ids, out=out)
    assert torch.equal(out, want)


def test_refuses_other_memory():
    p = Problem(80, 128, 128, 16, 2)
    with pytest.raises(ValueError):
        p.adapters.apply(p.x.cpu(), p.ids)
    with pytest.raises(ValueError):
        p.adapters.apply(p.x, p.ids.cpu())
    with pytest.raises(ValueError):
        p.adapters.apply(p.x, p.ids.long())
    with pytest.raises(hymoe.HymoeError):
        p.adapters.apply(p.x.half(), p.ids)
    with pytest.raises(hymoe.HymoeError):
        p.adapters.apply(p.x, p.ids, out=p.x)
