"""What tests/head_bounds.py lets pass and what not: results with the roundings that there are, and results with a mistake in them, planted into the oracle."""
import math

import pytest
import torch

from head_bounds import IGNORED, check, exact_logits, losses_are_exact


def inputs(tokens, dim, classes, dtype, ignored=0.2):
    g = torch.Generator().manual_seed(tokens + dim)
    x = torch.randn(tokens, dim, generator=g).to(dtype)
    w = (torch.randn(classes, dim, generator=g) * (2.0 / math.sqrt(dim))).to(dtype)
    t = torch.randint(0, classes, (tokens,), generator=g)
    return x, w, torch.where(torch.rand(tokens, generator=g) < ignored, torch.full_like(t, IGNORED), t)


def planes(v, count):
    out, v = [], v.float()
    for _ in range(count):
        out.append(v.bfloat16().float())
        v = v - out[-1]
    return [p.double() for p in out]


ALL = ((1, 1), (2, 0), (0, 2), (1, 0), (0, 1), (0, 0))


def product(a, b, pairs):
    """a . b^T of fp32 matrices from the products of their planes that are in `pairs`; None: as fp32 values."""
    if pairs is None:
        return (a.double() @ b.double().T).float()
    pa, pb = planes(a, 3), planes(b, 3)
    return sum(pa[i] @ pb[j].T for i, j in pairs).float()


def results(x, w, t, reduction, dloss, pairs=None, forward=None, low_g=False):
    """As the kernels do it: logits and gradients in fp32, G in bf16 for bf16 (without the factor that rows share)."""
    keep = t != IGNORED
    xf, wf = torch.where(keep[:, None], x.float(), 0.0), w.float()
    logits = product(xf, wf, forward or pairs)
    lse = torch.logsumexp(logits.double(), 1).float()
    label = torch.where(keep, t, 0)
    at = torch.arange(len(t))
    nll = torch.where(keep, lse - logits[at, label], 0.0)
    G = (logits - lse[:, None]).exp()
    G[at, label] -= 1.0
    factor = dloss if reduction == "none" else torch.ones(len(t))
    G = G * (factor * keep)[:, None]
    scale = 1.0 if reduction == "none" else float(dloss) / (int(keep.sum()) if reduction == "mean" else 1)
    if x.dtype == torch.bfloat16 or low_g:
        G = G.bfloat16().float()
    dx, dw = product(G, wf.T, pairs) * scale, product(G.T, xf.T, pairs) * scale
    loss = nll if reduction == "none" else nll.double().sum().float() / (int(keep.sum()) if reduction == "mean" else 1)
    return loss, dx.to(x.dtype), dw.to(x.dtype)


def rejected(*args):
    with pytest.raises(AssertionError):
        check(*args)


CASES = [(65, 72, 513), (300, 33, 1001), (257, 256, 999), (577, 101, 2400)]


def dloss_of(reduction, tokens):
    return torch.linspace(0.25, 1.5, tokens) if reduction == "none" else torch.tensor(0.75)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("reduction", ["mean", "none", "sum"])
@pytest.mark.parametrize("tokens,dim,classes", CASES)
def test_what_passes_and_what_does_not(tokens, dim, classes, reduction, dtype):
    x, w, t = inputs(tokens, dim, classes, dtype)
    d = dloss_of(reduction, tokens)
    loss, dx, dw = results(x, w, t, reduction, d)
    check(x, w, t, reduction, loss, d, dx, dw)
    undefined = dx.clone()
    undefined[int((t != IGNORED).nonzero()[-1]), dim - 1] = math.nan
    for bad in (undefined, torch.full_like(dx, math.nan), torch.zeros_like(dx), dx.roll(1, 0), dx * (1 + 2.0**-5)):
        rejected(x, w, t, reduction, loss, d, bad, dw)
    short = dw.clone()
    short[classes - 40:] = 0   # the last tile of classes left out
    undefined = dw.clone()
    undefined[classes - 1, 0] = math.nan
    for bad in (undefined, torch.full_like(dw, math.nan), torch.zeros_like(dw), dw.roll(1, 0), short, dw * (1 + 2.0**-5)):
        rejected(x, w, t, reduction, loss, d, dx, bad)
    # a stage of the tokens missing in dW, and one of the classes in dx
    fewer = t.clone()
    fewer[:32] = IGNORED
    scale = float((t != IGNORED).sum()) / float((fewer != IGNORED).sum()) if reduction == "mean" else 1.0
    rejected(x, w, t, reduction, loss, d, dx, (results(x, w, fewer, reduction, d)[2].float() / scale).to(dtype))
    rejected(x, w, t, reduction, loss * 1.01, d, dx, dw)
    rejected(x, w, t, reduction, loss * math.nan, d, dx, dw)


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("tokens,dim,classes", CASES)
def test_planes_of_fp32(tokens, dim, classes, reduction):
    """The six products pass; five of them, two planes, bf16 operands and G in bf16 do not."""
    x, w, t = inputs(tokens, dim, classes, torch.float32)
    d = dloss_of(reduction, tokens)
    loss, dx, dw = results(x, w, t, reduction, d, ALL)
    check(x, w, t, reduction, loss, d, dx, dw)
    # from the gradients' products alone; the smallest, two middle planes', is as large as the bound (exact_logits below has it), and without factors of their own the targets' G is so near to -1
    # that its third plane is nothing
    for left_out in range(1 if reduction == "none" else 2, 6):
        rejected(x, w, t, reduction, loss, d, *results(x, w, t, reduction, d, ALL[:left_out] + ALL[left_out + 1:], ALL)[1:])
    rejected(x, w, t, reduction, loss, d, *results(x, w, t, reduction, d, ((1, 1), (1, 0), (0, 1), (0, 0)))[1:])
    rejected(x, w, t, reduction, loss, d, *results(x, w, t, reduction, d, ((0, 0),))[1:])
    rejected(x, w, t, reduction, loss, d, *results(x, w, t, reduction, d, ALL, low_g=True)[1:])


@pytest.mark.parametrize("kind", ["weight", "hidden", "middle"])
def test_exact_logits(kind):
    """Every one of the six products is missed by one of the three kinds."""
    x, w, t = exact_logits(kind, 300, 72, 1001, "cpu")
    d = torch.ones(300)
    assert losses_are_exact(results(x, w, t, "none", d, ALL)[0], x, w, t)
    needed = {"weight": ((2, 0), (1, 0), (0, 0)), "hidden": ((0, 2), (0, 1), (0, 0)), "middle": ((1, 1), (1, 0), (0, 1), (0, 0))}[kind]
    for pair in needed:   # (plane of the weight, plane of x)
        some = tuple((b, a) for a, b in ALL if (a, b) != pair)
        assert not losses_are_exact(results(x, w, t, "none", d, some)[0], x, w, t)
