"""ops.linear_cross_entropy of infinities and of the types' largest values, which mask classes: the same answer at every size, whichever kernels take it."""
import math

import pytest
import torch

from randumb_amd import ops

pytestmark = pytest.mark.gpu


# fp32: few tokens, products of fp32, planes going forward only, planes both ways; bf16: few tokens, one and two blocks a compute unit
SIZES = [(24, 64, 700), (300, 64, 1000), (1300, 40, 12001), (611, 333, 33001), (640, 520, 12000)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,dim,classes", SIZES)
def test_masked_classes(tokens, dim, classes, dtype):
    """Classes 0 to 4 have a weight that makes their logit -infinity, or the lowest value: they count for nothing.  Losses against 64 bits: a logit's dim additions and its products
    (2^-23 of each in all), a few roundings of the logarithm.  The masked classes' dW is zero, everybody else's finite; dx is a number but for the columns of the infinities, whose
    gradient is theirs (NaN by nothing)."""
    print(f"case masked classes {tokens} x {dim} -> {classes} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    x = torch.randn(tokens, dim, device="cuda", generator=g)
    x[:, 0], x[:, 1] = x[:, 0].abs() + 0.25, -x[:, 1].abs() - 0.25
    w = torch.randn(classes, dim, device="cuda", generator=g) / math.sqrt(dim)
    x, w = x.to(dtype), w.to(dtype)
    top = torch.finfo(dtype).max
    w[0, 0], w[1, 1], w[2, 0] = -math.inf, math.inf, -top
    w[3] = 0
    w[3, 0] = -top * 0.75
    w[4, 0], w[4, 1] = -math.inf, math.inf
    w[classes - 1, 0] = -math.inf   # in the last tile
    t = torch.randint(5, classes - 1, (tokens,), device="cuda", generator=g)
    t[3] = -100
    masked = torch.tensor([0, 1, 2, 3, 4, classes - 1], device="cuda")
    x.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, t, reduction="none")
    dx, dw = torch.autograd.grad(loss, [x, w], torch.ones(tokens, device="cuda"))
    xd, wd, some = x.detach().double(), w.detach().double(), torch.ones(classes, dtype=torch.bool, device="cuda")
    some[masked] = False
    logits = xd @ wd[some].T
    label = (torch.cumsum(some, 0) - 1)[t.clamp_min(5)]   # 5: an ignored row, of any class
    want = torch.where(t >= 0, torch.logsumexp(logits, 1) - logits.gather(1, label[:, None])[:, 0], 0.0)
    tol = (dim + 16) * 2.0**-23 * float((xd.abs() @ wd[some].abs().T).max()) + 2.0**-20
    assert bool(((loss.detach().double() - want).abs() <= tol).all())
    assert bool(dw.isfinite().all()) and not bool(dw[masked].any())
    assert bool(dx[:, 2:].isfinite().all())
    p = (logits - torch.logsumexp(logits, 1)[:, None]).exp()
    p[t < 0] = 0.0
    G = p.clone()
    G[torch.arange(tokens, device="cuda"), label] -= (t >= 0).double()
    half = torch.finfo(dtype).eps / 2
    # of G: twice its logit's error, relative to p, and its own rounding; then the sums and the result's rounding
    off = 2 * tol * p + half * G.abs()
    for got, exact, err, size, n in ((dx[:, 2:], (G @ wd[some])[:, 2:], (off @ wd[some].abs())[:, 2:], (G.abs() @ wd[some].abs())[:, 2:], classes), (dw[some], G.T @ xd, off.T @ xd.abs(), G.abs().T @ xd.abs(), tokens)):
        assert bool(((got.double() - exact).abs() <= err + (n + 16) * 2.0**-23 * size + half * exact.abs()).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,dim,classes", SIZES)
def test_infinite_hidden_states_and_logits(tokens, dim, classes, dtype):
    """An infinite or undefined hidden state reaches its own row's loss, an infinite logit every row that has it; the other rows' losses keep their bits."""
    print(f"case infinite rows {tokens} x {dim} -> {classes} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.randn(tokens, dim, device="cuda", generator=g)
    x[:, 0] = x[:, 0].abs() + 0.25
    x, w = x.to(dtype), (torch.randn(classes, dim, device="cuda", generator=g) / math.sqrt(dim)).to(dtype)
    t = torch.randint(0, classes - 1, (tokens,), device="cuda", generator=g)
    want = ops.linear_cross_entropy(x, w, t, reduction="none")
    for row, value in ((0, math.inf), (tokens // 2, -math.inf), (tokens - 1, math.nan)):
        y = x.clone()
        y[row, dim - 1] = value
        loss = ops.linear_cross_entropy(y, w, t, reduction="none")
        same = torch.arange(tokens, device="cuda") != row
        assert bool(loss[row].isnan()) and torch.equal(loss[same], want[same])
    v = w.clone()
    v[classes - 1, 0] = math.inf
    assert bool(ops.linear_cross_entropy(x, v, t, reduction="none").isnan().all())
    # every logit of a class -infinity, and the class a target: its loss is infinite
    v[classes - 1, 0], t[1] = -math.inf, classes - 1
    loss = ops.linear_cross_entropy(x, v, t, reduction="none")
    assert float(loss[1]) == math.inf and int(loss.isfinite().sum()) == tokens - 1
