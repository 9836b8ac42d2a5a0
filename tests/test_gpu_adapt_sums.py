"""GPU tests of the narrow products' sums over long rows (hymoe_adapt, hymoe_adapt_backward): the
intermediate A x (B^T dy) itself, read through one-hot weights on the other side, against double
precision.

Tolerances.  An addition of the matrix pipe truncates the products that it takes in (8 or 16) and its
running sum; two steps of 2^-23 of the running sum are allowed for it.  An accumulator that takes `adds`
of them, of terms of one sign, so loses at most (adds + 1) / 2 times that of its sum; of terms of
either sign, 2/3 adds times in the 2-norm (the running sum grows like a square root, and the blocks'
errors add up like the blocks).  The blocks' sums are added in fp32, each rounding half a step of
2^-23 either way: beyond six standard deviations, 2 sqrt(blocks) half steps of the largest error and
sqrt(blocks) of the norm; and the parts of the CTAs that share a tile, 16 at most.  An fp32 row is
taken in two parts that leave 3 of 2^23, and the one-hot product adds three parts: 7 with the last
roundings.  Nothing of this grows with the length of the rows but the fp32 sums' square root."""
import pytest

import hymoe

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

T16 = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = 64          # columns of a block's sum in the mma.sync kernels
SEGMENT = 512       # the fewest columns of a segment on the 5th-generation tensor cores
SPLITS = 16


def limits(K, adds, block):
    blocks = K / block
    one = (2 * (adds + 1) / 2 + 7) * 2.0 ** -23 + (2 * blocks ** 0.5 + SPLITS + 4) * 2.0 ** -24
    two = (2 * 2 * adds / 3 + 7) * 2.0 ** -23 + (blocks ** 0.5 + SPLITS + 4) * 2.0 ** -24
    return one, two


def weights(g, K, R, w, signs):
    a = torch.rand((R, K), generator=g, device="cuda") + 0.5
    if signs:
        a = torch.randn((R, K), generator=g, device="cuda")
    return (a * 2.0 ** -10).to(T16[w])


def check(got, x, a, K, signs, adds, block):
    """got [T, R] against x [T, K] a^T, some columns at a time."""
    want = torch.zeros(got.shape, dtype=torch.double, device="cuda")
    for k in range(0, K, 1 << 16):
        want += x[:, k:k + (1 << 16)].double() @ a[:, k:k + (1 << 16)].double().t()
    one, two = limits(K, adds, block)
    err = (got.double() - want).abs()
    if signs:
        assert float(err.norm()) <= two * float(want.norm()), (float(err.norm() / want.norm()), two)
    else:
        assert bool((err <= one * want).all()), (float((err / want).max()), one)


CASES = [  # tokens, columns, rank, x, weights, additions of one accumulator, columns of a block
    (100, 1 << 16, 4, "f32", "bf16", 16, BLOCK),
    (300, 1 << 16, 8, "f32", "f16", 16, BLOCK),
    (300, (1 << 18) + 1, 3, "f32", "bf16", 16, BLOCK),
    (300, 1 << 18, 100, "f32", "bf16", 16, BLOCK),
    (4200, 8192, 16, "f32", "bf16", 16, BLOCK),
    (300, (1 << 18) + 1, 5, "bf16", "bf16", 4, BLOCK),    # off 16-byte boundaries
    (300, (1 << 18) + 4, 40, "f16", "f16", 4, BLOCK),
    (100, 1 << 18, 8, "bf16", "bf16", 4, BLOCK),          # few tokens
    # the 5th-generation tensor cores: 64 additions (rank 128: 128) where the accumulators take all of a CTA's columns
    (300, 1 << 15, 8, "bf16", "bf16", 64, 1 << 12),
    (300, 1 << 15, 128, "f16", "f16", 128, 1 << 12),
    # longer rows in segments of 32
    (300, 1 << 20, 8, "bf16", "bf16", 32, SEGMENT),
    (300, 1 << 20, 128, "bf16", "bf16", 32, SEGMENT),
    (300, 1 << 18, 64, "f16", "f16", 32, SEGMENT),
    (300, 200 * 1024 + 72, 32, "bf16", "bf16", 32, SEGMENT),
    (300, (1 << 15) + 64, 24, "f16", "f16", 32, SEGMENT),   # one stage more in some CTAs
    (300, (1 << 15) + 520, 128, "bf16", "bf16", 32, SEGMENT),
    (2000, 1 << 16, 16, "f16", "f16", 32, SEGMENT),
]
NAMES = ["-".join(map(str, c[:5])) for c in CASES]


def problem(case, signs, order):
    T, K, R, x, w, adds, block = case
    g = torch.Generator(device="cuda")
    g.manual_seed(K + R)
    a = weights(g, K, R, w, signs)
    v = torch.randn((T, K), generator=g, device="cuda") if signs else torch.rand((T, K), generator=g, device="cuda") + 0.5
    M = max(64, (R + 7) // 8 * 8)
    hot = torch.zeros((M, R), dtype=T16[w], device="cuda")
    hot[torch.arange(R), torch.arange(R)] = 1.0
    ids = torch.zeros((T,), dtype=torch.int32, device="cuda")
    if order == "any":  # rows without an adapter between the others: copied, not loaded in runs
        ids[::7] = -1
    return v.to(T16[x]), a, hot, ids


@pytest.mark.parametrize("order", ["run", "any"])
@pytest.mark.parametrize("signs", [False, True], ids=["positive", "signed"])
@pytest.mark.parametrize("case", CASES, ids=NAMES)
def test_forward(case, signs, order):
    T, K, R, x, w, adds, block = case
    v, a, hot, ids = problem(case, signs, order)
    out = torch.empty((T, hot.shape[0]), device="cuda")
    hymoe.Adapters(a[None], hot[None]).apply(v, ids, out=out)
    rows = ids >= 0
    check(out[rows, :R], v[rows], a, K, signs, adds, block)


@pytest.mark.parametrize("signs", [False, True], ids=["positive", "signed"])
@pytest.mark.parametrize("case", CASES, ids=NAMES)
def test_backward(case, signs):
    """B^T dy, whose weights lie the other way: the sums run over the output's columns."""
    T, K, R, x, w, adds, block = case
    v, b, hot, ids = problem(case, signs, "any")
    xin = torch.zeros((T, hot.shape[0]), device="cuda")
    ad = hymoe.Adapters(hot.t().contiguous()[None], b.t().contiguous()[None])
    rows = ids >= 0
    for want in (("dx",), ("dx", "db")):
        check(ad.backward(xin, v, ids, want=want)["dx"][rows, :R], v[rows], b, K, signs, adds, block)
