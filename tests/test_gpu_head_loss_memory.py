"""What ops.linear_cross_entropy allocates: logits that are kept are kept once, and only where there will be a backward pass."""
import pytest
import torch

from randumb_amd import ops

pytestmark = pytest.mark.gpu


def peak(call):
    """Bytes that a call needs at most beside what is there, and what it leaves."""
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = call()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before, torch.cuda.memory_allocated() - before, out


@pytest.mark.parametrize("tokens,dim,classes", [(12, 2048, 40001), (256, 1024, 60000)])
def test_logits_that_are_kept(tokens, dim, classes):
    logits = 4 * tokens * classes
    w = torch.nn.Parameter(torch.randn(classes, dim, device="cuda") * 0.02)
    x, t = torch.randn(tokens, dim, device="cuda"), torch.randint(0, classes, (tokens,), device="cuda")
    some = 1 << 20
    with torch.no_grad():   # a piece of the logits in the workspace, and nothing left
        most, left, scored = peak(lambda: ops.linear_cross_entropy(x, w, t, reduction="none"))
    assert most <= logits + some and left <= some
    most, left, loss = peak(lambda: ops.linear_cross_entropy(x, w, t, reduction="none"))
    assert most <= logits + some and logits <= left
    assert torch.equal(loss.detach(), scored)
    most, left, _ = peak(lambda: ops.linear_cross_entropy(x, w.detach(), t))   # nothing wants a gradient
    assert most <= logits + some and left <= some
