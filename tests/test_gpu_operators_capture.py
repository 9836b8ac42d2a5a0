"""The routing and adapter operators captured into CUDA graphs by a process that has called none of
them before, and used from several threads at once."""
import os
import subprocess
import sys
import threading

import pytest

import hymoe
from test_gpu_adapt import Problem
from test_gpu_gate import bias_of, logits_of

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

FIRST = """
import sys
sys.path[:0] = {paths!r}
import torch, hymoe
from test_gpu_adapt import Problem
from test_gpu_gate import bias_of, logits_of
op, T = sys.argv[1], int(sys.argv[2])
torch.zeros(1, device="cuda")
if op == "adapt":
    p = Problem(T, 256, 264, 16, 4)
    run = lambda: (p.adapters.apply(p.x, p.ids, base=p.base), *p.adapters.backward(p.x, p.dy, p.ids, base=p.base_x).values())
else:
    z, b, dw = logits_of(T, 128, torch.bfloat16).cuda(), bias_of(128).cuda(), torch.ones(T, 6, device="cuda")
    gate = hymoe.Gate(128, 6, score="sigmoid")
    def run():
        r = gate.route(z, bias=b, counts=True)
        return (*r.values(), gate.backward(z, r["idx"], dw))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, run()))
print("same")
"""


@pytest.mark.parametrize("op,T", [("adapt", 3), ("adapt", 100), ("adapt", 700), ("route", 5), ("route", 20000)])
def test_first_call_is_captured(op, T):
    here = os.path.dirname(os.path.abspath(__file__))
    paths = [here, os.path.dirname(os.path.abspath(hymoe.__file__))]
    r = subprocess.run([sys.executable, "-c", FIRST.format(paths=paths), op, str(T)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip().endswith("same"), r.stderr[-2000:]


def test_threads_with_their_own_streams():
    """Calls from several threads at once, each on its own stream, over shared adapters and a shared gate."""
    ps = [Problem(T, 256, 264, 16, 4, seed=T) for T in (7, 90, 400, 1500)]
    for p in ps[1:]:
        p.a, p.b, p.scale, p.adapters = ps[0].a, ps[0].b, ps[0].scale, ps[0].adapters
    gate, z, b = hymoe.Gate(128, 6, score="sigmoid"), logits_of(20000, 128, torch.bfloat16).cuda(), bias_of(128).cuda()

    def work(p):
        r = gate.route(z[:50 * p.T], bias=b, counts=True)
        return (p.adapters.apply(p.x, p.ids, base=p.base), *p.adapters.backward(p.x, p.dy, p.ids, base=p.base_x).values(), *r.values())

    want = [work(p) for p in ps]
    torch.cuda.synchronize()
    wrong = []

    def many(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = work(ps[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(x, y) for x, y in zip(got, want[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=many, args=(i,)) for i in range(len(ps))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
