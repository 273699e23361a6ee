"""ops.linear_cross_entropy where whole ranges of classes are masked by huge negative weights, as the padding of a vocabulary is: tiles with nothing else in them."""
import math

import pytest
import torch

from randumb_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("low", [-3.0e4, -1.0e10, -1.0e30, -2.0e38, -math.inf])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,dim,classes", [(24, 64, 3000), (24, 65, 3000), (300, 64, 3000), (1300, 40, 12001), (2100, 520, 4000), (640, 520, 12000)])
def test_masked_ranges(tokens, dim, classes, dtype, low):
    """Nothing of them is in the loss or its gradients: what the other classes alone give, a logit's dim additions and products apart (2^-23 of each), and sums in other groups."""
    print(f"case masked ranges {tokens} x {dim} -> {classes} {dtype} {low}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(classes)
    x = torch.randn(tokens, dim, device="cuda", generator=g).to(dtype)
    w = (torch.randn(classes, dim, device="cuda", generator=g) / math.sqrt(dim)).to(dtype)
    x[:, 0] = 1.0 + torch.rand(tokens, device="cuda", generator=g).to(dtype) * 0.5
    some = torch.ones(classes, dtype=torch.bool, device="cuda")
    some[512:1100] = False        # whole tiles in the middle
    some[classes - 300:] = False   # and the last ones
    w[~some] = 0
    w[~some, 0] = low
    t = torch.randint(0, 500, (tokens,), device="cuda", generator=g)
    t[7] = -100
    x.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, t, reduction="none")
    dx, dw = torch.autograd.grad(loss, [x, w], torch.ones(tokens, device="cuda"))
    xd, wd = x.detach().double(), w.detach().double()[some]
    logits = xd @ wd.T
    lse = torch.logsumexp(logits, 1)
    keep = t >= 0
    label = t.clamp_min(0)   # the first 512 classes are in their places
    want = torch.where(keep, lse - logits.gather(1, label[:, None])[:, 0], 0.0)
    tol = (dim + 16) * 2.0**-23 * float((xd.abs() @ wd.abs().T).max()) + 2.0**-20
    assert bool(((loss.detach().double() - want).abs() <= tol).all())
    p = (logits - lse[:, None]).exp() * keep[:, None]
    G = p.clone()
    G[torch.arange(tokens, device="cuda"), label] -= keep.double()
    half = torch.finfo(dtype).eps / 2
    off = 2 * tol * p + half * G.abs()
    columns = slice(1 if low == -math.inf else 0, None)   # an infinity by nothing is undefined
    for got, exact, err, size, n in ((dx, G @ wd, off @ wd.abs(), G.abs() @ wd.abs(), classes), (dw[some], G.T @ xd, off.T @ xd.abs(), G.abs().T @ xd.abs(), tokens)):
        c = columns if got is dx else slice(None)
        assert bool(((got.double() - exact).abs() <= err + (n + 16) * 2.0**-23 * size + half * exact.abs())[:, c].all())
    assert not bool(dw[~some].any())


@pytest.mark.parametrize("height", [2.0e3, 1.0e6, 1.0e9, 1.0e30])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,dim,classes", [(24, 64, 3000), (24, 65, 3000), (300, 64, 3000), (1300, 40, 12001), (2100, 520, 4000), (640, 520, 12000)])
def test_far_logits(tokens, dim, classes, dtype, height):
    """One class a token far above the others, by more than logits of that size are rounded by: a loss of zero, or of the distance, and a gradient that is one class or two.  A
    value of the softmax is off by its logit's error e, in relation, and at most 1 in any case: by min(1, exp(2 e) - 1)."""
    print(f"case far logits {tokens} x {dim} -> {classes} {dtype} {height}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(dim)
    w = torch.randn(classes, dim, device="cuda", generator=g)
    w = (w / w.norm(dim=1, keepdim=True)).to(dtype)
    own = torch.randint(0, classes, (tokens,), device="cuda", generator=g)
    x = (w[own].float() * height).to(dtype)
    t = torch.where(torch.arange(tokens, device="cuda") % 2 == 0, own, (own + 1) % classes)
    x.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, t, reduction="none")
    dx, dw = torch.autograd.grad(loss, [x, w], torch.ones(tokens, device="cuda"))
    xd, wd = x.detach().double(), w.detach().double()
    logits = xd @ wd.T
    lse = torch.logsumexp(logits, 1)
    tol = (dim + 16) * 2.0**-23 * float((xd.abs() @ wd.abs().T).max()) + 2.0**-20
    assert bool((loss >= 0).all()) and bool(((loss.detach().double() - (lse - logits.gather(1, t[:, None])[:, 0])).abs() <= 2 * tol).all())
    p = (logits - lse[:, None]).exp()
    G = p.clone()
    G[torch.arange(tokens, device="cuda"), t] -= 1.0
    half = torch.finfo(dtype).eps / 2
    off = min(1.0, math.expm1(min(2 * tol, 1.0))) * p + half * G.abs()
    for got, exact, err, size, n in ((dx, G @ wd, off @ wd.abs(), G.abs() @ wd.abs(), classes), (dw, G.T @ xd, off.T @ xd.abs(), G.abs().T @ xd.abs(), tokens)):
        assert bool(((got.double() - exact).abs() <= err + (n + 16) * 2.0**-23 * size + half * exact.abs() + 1e-30).all())
