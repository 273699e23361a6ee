"""A backward pass of the head's loss and of the rotation captured while an older graph of the same leaves lives: refused where the leaf comes reshaped, sliced or cast, too.  It would end
the process.  In a process of its own; without the older graph it is captured."""
import pathlib
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CAPTURE = """
import torch
from randumb_amd import ops
x3, w, t = torch.randn(4, 6, 64, device="cuda"), torch.randn(300, 64, device="cuda"), torch.randint(0, 300, (4, 6), device="cuda")
low = x3.bfloat16()
qkv, freq = torch.randn(2, 5, 7, 8, device="cuda"), ops.rotary_frequencies(8, device="cuda")[0]
for name, leaf, call in (("reshaped", x3, lambda: ops.linear_cross_entropy(x3, w.detach(), t)),
                         ("cast", w, lambda: ops.linear_cross_entropy(low, w.to(torch.bfloat16), t)),
                         ("sliced", qkv, lambda: sum(o.square().sum() for o in ops.rotary(qkv[:, :, :4], qkv[:, :, 4:6], freq)))):
    leaf.requires_grad_()
    held = call()
    want = torch.autograd.grad(held, [leaf], retain_graph=True)
    torch.cuda.synchronize()
    try:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(call(), [leaf])
    except RuntimeError as e:
        assert "an earlier graph of the same leaf" in str(e), e
        print(name, "refused", flush=True)
    torch.cuda.synchronize()
    del held
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(call(), [leaf])
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    print(name, "captured", flush=True)
"""


def test_a_capture_beside_an_older_graph_of_the_same_leaves():
    done = subprocess.run([sys.executable, "-c", CAPTURE], cwd=pathlib.Path(__file__).parents[1], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and done.stdout.split() == [w for n in ("reshaped", "cast", "sliced") for w in (n, "refused", n, "captured")], (done.returncode, done.stdout, done.stderr[-2000:])
