"""GPU tests of the adapters' workspace in Python: a workspace of the caller's own gives the same
results, and its status can be read."""
import pytest

import hymoe
from test_gpu_adapt import Problem

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("T", [5, 64, 65, 300])
def test_status_can_be_read(T):
    p = Problem(T, 256, 264, 16, 4)
    ad = p.adapters
    want, grads = ad.apply(p.x, p.ids, base=p.base), ad.backward(p.x, p.dy, p.ids, base=p.base_x)
    one, two = ad.workspace(T), ad.workspace(T, backward=True)
    assert (one is None) == (T <= 64) and two is not None
    more = ad.workspace(T + 1000)
    for ws in (one, more):
        if ws is not None:
            ws.fill_(0xFF)
        assert torch.equal(ad.apply(p.x, p.ids, base=p.base, workspace=ws), want)
        if ws is not None and ws.numel() and T > 64:
            ad.check(ws)
    two.fill_(0xFF)
    got = ad.backward(p.x, p.dy, p.ids, base=p.base_x, workspace=two)
    ad.check(two)
    assert all(torch.equal(got[k], grads[k]) for k in grads)
    ad.check(None)
    two[2] = 1  # as an expired wait leaves it
    with pytest.raises(hymoe.HymoeError) as e:
        ad.check(two)
    assert e.value.status == 6 and "TIMEOUT" in str(e.value)


def test_refused_workspaces():
    p = Problem(100, 256, 264, 16, 4)
    ad = p.adapters
    n = ad.workspace(100).numel()
    for bad in (torch.empty(n, dtype=torch.uint8), torch.empty(n, dtype=torch.int8, device="cuda"),
                torch.empty(2 * n, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(ValueError):
            ad.apply(p.x, p.ids, base=p.base, workspace=bad)
        with pytest.raises(ValueError):
            ad.backward(p.x, p.dy, p.ids, workspace=bad)
    big = torch.empty(n + 512, dtype=torch.uint8, device="cuda")
    for bad in (big[:n - 256], big[16:16 + n]):
        with pytest.raises(hymoe.HymoeError) as e:
            ad.apply(p.x, p.ids, base=p.base, workspace=bad)
        assert e.value.status == 1 and "workspace" in str(e.value)


def test_captured_with_its_own_workspace():
    p = Problem(200, 256, 264, 16, 4)
    ad, ws = p.adapters, p.adapters.workspace(200)
    want = ad.apply(p.x, p.ids, base=p.base)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ad.apply(p.x, p.ids, base=p.base, workspace=ws)
    for _ in range(3):
        ws.fill_(0xFF)
        graph.replay()
        ad.check(ws)
        assert torch.equal(out, want)


def test_few_tokens_leave_the_status_alone():
    """A serving loop's one workspace for batches of every size: steps of a few tokens do not use it."""
    p = Problem(300, 256, 264, 16, 4)
    ad = p.adapters
    for _ in range(3):
        junk = torch.full((ad.workspace(300).numel(),), 0xFF, dtype=torch.uint8, device="cuda")
        del junk  # the next workspace is likely to be this memory
        ws = ad.workspace(300)
        for T in (5, 64, 300, 5):
            ad.apply(p.x[:T], p.ids[:T], base=p.base[:T], workspace=ws)
            ad.check(ws)
