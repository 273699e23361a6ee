"""ops.linear_cross_entropy of tokens whose own class has nearly all of the probability: the loss is not below zero, and off by what rounds a sum near one, not by what rounds
logits of hundreds."""
import math

import pytest
import torch

from randumb_amd import ops

pytestmark = pytest.mark.gpu


# few tokens as they are and gathered, one and two blocks a compute unit, many tokens; fp32: few, products of fp32, planes; several pieces of the vocabulary
CASES = [(24, 1000, 5000), (24, 1001, 5000), (64, 256, 40001), (150, 1000, 3001), (1300, 264, 12001), (8200, 128, 3000), (640, 520, 12000), (64, 8, 1100000)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,dim,classes", CASES)
def test_confident_tokens(tokens, dim, classes, dtype):
    """Own logits of 16, 60 and 300 above nearly everybody else's.  log sum exp(l - l_own) has a sum of 1 and something: every addition on the way (64 of a lane's, then one for each
    tile of 64 classes or more) rounds by 2^-24 of it, exponentials and the logarithm by a few times that; the small terms are off by their logits, in relation to the loss."""
    print(f"case confident {tokens} x {dim} -> {classes} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(classes)
    w = (torch.randn(classes, dim, device="cuda", generator=g) * (2.0 / math.sqrt(dim))).to(dtype)
    t = torch.randint(0, classes, (tokens,), device="cuda", generator=g)
    own = w[t].float()
    height = torch.tensor([16.0, 60.0, 300.0], device="cuda")[torch.arange(tokens, device="cuda") % 3]
    x = (own * (height / own.square().sum(1))[:, None]).to(dtype)
    t[5] = -100
    loss = ops.linear_cross_entropy(x, w, t, reduction="none")
    logits = x.double() @ w.double().T
    picked = logits.gather(1, t.clamp_min(0)[:, None])
    want = torch.where(t >= 0, torch.logsumexp(logits - picked, 1), 0.0)
    assert bool((loss >= 0).all()) and float(loss[5]) == 0.0
    # half of the difference of two logits is off by dim additions and their products, 2^-23 of each
    off = 2 * (dim + 16) * 2.0**-23 * (x.double().abs() * (w[t.clamp_min(0)].double().abs() + w.double().abs().amax(0))).sum(1)
    tol = (100 + classes / 64) * 2.0**-24 + (off.exp() - 1) * want + 2.0**-22 * want
    assert bool(((loss.double() - want).abs() <= tol).all()), float(((loss.double() - want).abs() / tol).max())
    for reduction, exact in (("sum", want.sum()), ("mean", want.sum() / (tokens - 1))):
        got = ops.linear_cross_entropy(x, w, t, reduction=reduction)
        assert 0 <= float(got) and abs(float(got) - float(exact)) <= float(tol.sum()) * (1 if reduction == "sum" else 1 / (tokens - 1)) + tokens * 2.0**-24 * float(exact)
