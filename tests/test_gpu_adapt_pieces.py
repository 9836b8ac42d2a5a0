"""GPU tests of hymoe_adapt_backward for long adapters, whose gradients come in pieces, at odd ranks and
widths: the pieces' sums of both gradients start on their own boundaries in the workspace whatever
number of elements the other one's pieces have.  The tolerances are those of test_gpu_adapt.py."""
import pytest

from test_gpu_adapt import Problem, check_grads

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("T", [520, 600, 1023, 1100, 1700, 3000, 3700, 4500])
@pytest.mark.parametrize("n_in,n_out,rank", [(5, 4, 3), (49, 8, 85), (1, 20, 49), (33, 468, 43), (63, 12, 1), (10, 6, 2), (7, 9, 4)])
def test_odd_sizes_in_pieces(T, n_in, n_out, rank):
    check_grads(Problem(T, n_in, n_out, rank, 1, ids="one", x="f32", w="bf16", y="f32"))
    p = Problem(T, n_in, n_out, rank, 3, ids="mixed", x="f16", w="f16", y="f16")
    p.ids[:] = 1  # one adapter has all but a few tokens
    p.ids[::97] = 2
    check_grads(p)
    only = p.adapters.backward(p.x, p.dy, p.ids, want=("db",))["db"]
    assert torch.equal(only, p.adapters.backward(p.x, p.dy, p.ids)["db"])


def test_workspace_parts_start_on_256_bytes():
    """The workspace's size as the sum of parts of whole 256 bytes."""
    for T in (600, 1700, 3000):
        for n_in, n_out, rank in ((5, 4, 3), (33, 468, 43)):
            p = Problem(T, n_in, n_out, rank, 1, ids="one")
            assert p.adapters.workspace(T, backward=True).numel() % 256 == 0
