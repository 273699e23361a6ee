"""The loss of an output head and its gradients in 64 bits, with bounds for every value and for norms that follow from the roundings on the way.

A logit is a sum of ``dim`` products in fp32: off by (dim + 16) 2^-24 of its absolute values' sum at most (fp32: products off by one rounding more, in planes a tenth more additions of
small values).  Values of the softmax are off by their logit and their row's lse, in relation; in bf16 G is rounded once more.  A gradient is a sum of G times the other factor, and is
rounded once.

``values`` holds every element to the worst of that.  ``norms`` holds whole gradients to what independent roundings give: their squares add up, a sum of n terms has no more than one rounding for every
8 of them (a matrix instruction takes 16 at a time), each of at most half a step of what has been added up, which is about the sum of the terms' squares."""
import math

import torch

IGNORED = -100
U = 2.0**-24


class Exact:
    """loss, dx, dw; their bounds by value (``*_tol``) and the squares of their expected errors' norms (``dx_sq``, ``dw_sq``)."""

    def __init__(self, x, w, t, reduction, dloss):
        half, bf16 = torch.finfo(x.dtype).eps / 2, x.dtype == torch.bfloat16
        self.half = half
        tokens, dim = x.shape
        classes = w.shape[0]
        wd = w.detach().double()
        wa = wd.abs()
        keep_all = t != IGNORED
        count = int(keep_all.sum())
        adds = dim + 16 if bf16 else 1.1 * dim + 26
        of = lambda n: (4 + 0.6 * math.sqrt(n / 8)) * U   # noqa: E731
        dev = x.device
        nll, nll_tol = torch.zeros(tokens, dtype=torch.float64, device=dev), torch.zeros(tokens, dtype=torch.float64, device=dev)
        self.dx, self.dx_tol = (torch.zeros(tokens, dim, dtype=torch.float64, device=dev) for _ in range(2))
        self.dw, self.dw_tol, dw_sq, dw_sums = (torch.zeros(classes, dim, dtype=torch.float64, device=dev) for _ in range(4))
        self.dx_sq = 0.0
        rows = max(1, (1 << 26) // classes)
        for r in range(0, tokens, rows):
            part = slice(r, min(tokens, r + rows))
            keep, xd, label = keep_all[part], x.detach()[part].double(), t[part]
            n = len(keep)
            at = torch.arange(n, device=dev)
            xd = torch.where(keep[:, None], xd, 0.0)
            label = torch.where(keep, label, 0).long()
            logits = xd @ wd.T
            lse = torch.logsumexp(logits, 1)
            p = (logits - lse[:, None]).exp() * keep[:, None]
            e = adds * U * (xd.abs() @ wa.T)
            lse_tol = (p * e).sum(1) + (100 + classes / 64) * U + 8 * U * lse.abs()
            nll[part] = torch.where(keep, lse - logits[at, label], 0.0)
            nll_tol[part] = (lse_tol + e[at, label] + 8 * U * logits[at, label].abs()) * keep
            share = keep.double() * (dloss.double()[part] if reduction == "none" else dloss.double().reshape(()))
            if reduction == "mean":
                share = share / max(count, 1)
            off = (e + lse_tol[:, None] + U * (4 * (logits - lse[:, None]).abs() + 4 * lse.abs()[:, None] + 16)).expm1_().mul_(p)
            # by norm: a logit's own error, and what the row has in common
            own = of(dim) * (xd.square() @ wd.square().T).sqrt_() + U * ((logits - lse[:, None]).abs() + logits.abs() + 4)
            common = U * (2 * lse.abs() + 8 + 0.6 * math.sqrt(classes / 8)) * share
            pw, px = p * share.abs()[:, None], None
            G = p
            G[at, label] -= keep.double()
            G *= share[:, None]
            size = G.abs()
            off = off * share.abs()[:, None] + (half * size if bf16 else 0.0) + 4 * U * size
            self.dx[part] = G @ wd
            self.dw += G.T @ xd
            sums = size @ wa
            self.dx_tol[part] = off @ wa + (classes + 16) * U * sums + (half + 4 * U) * self.dx[part].abs() + 1e-37
            self.dw_tol += off.T @ xd.abs()
            dw_sums += size.T @ xd.abs()
            rounded = half * half if bf16 else 0.0
            var = (own * pw).square() + (rounded + of(classes) ** 2) * G.square()
            self.dx_sq += float((var @ wd.square()).sum() + (common[:, None] * (pw / share.abs().clamp_min(1e-300)[:, None] @ wd)).square().sum())
            dw_sq += ((own * pw).square() + (rounded + of(tokens) ** 2) * G.square() + (common[:, None] * pw / share.abs().clamp_min(1e-300)[:, None]).square()).T @ xd.square()
        self.dw_tol += (tokens + 16) * U * dw_sums + (half + 4 * U) * self.dw.abs() + 1e-37
        self.dx_sq += (half**2 + of(classes) ** 2) * float(self.dx.square().sum())
        self.dw_sq = float(dw_sq.sum()) + (half**2 + of(tokens) ** 2) * float(self.dw.square().sum())
        self.loss, self.loss_tol = nll, nll_tol
        if reduction != "none":
            n = max(count, 1) if reduction == "mean" else 1
            self.loss = nll.sum() / (count if reduction == "mean" else 1)
            self.loss_tol = nll_tol.sum() / n + (tokens + 8) * U * nll.sum() / n


def check(x, w, t, reduction, loss, dloss, dx=None, dw=None):
    """All of it; what is not a number passes nowhere."""
    want = Exact(x, w, t, reduction, dloss)
    assert loss.dtype == torch.float32 and loss.shape == want.loss.shape
    if reduction != "mean" or bool((t != IGNORED).any()):
        assert bool(((loss.double() - want.loss).abs() <= want.loss_tol).all()), float(((loss.double() - want.loss).abs() / want.loss_tol).max())
    for name, got, exact, tol, sq in (("dx", dx, want.dx, want.dx_tol, want.dx_sq), ("dw", dw, want.dw, want.dw_tol, want.dw_sq)):
        if got is None:
            continue
        assert got.dtype == x.dtype and got.shape == exact.shape
        err = (got.double() - exact).abs()
        assert bool((err <= tol).all()), (name, float((err / tol).max()), int((~(err <= tol)).sum()))
        assert float(err.norm()) <= math.sqrt(sq) + 1e-37, (name, float(err.norm()) / math.sqrt(sq), float(err.norm() / exact.norm()))


def exact_logits(kind, tokens, dim, classes, device):
    """fp32 inputs whose logits are single products, between -40 and 40, that fp32 holds, and so does every sum of their planes' products on the way ("middle": but for the last product
    of two lower planes).  "weight": rows of x with a single 1; "hidden": rows of the weight; "middle": a single 1 + 2^-8 in either, so that products of the middle planes matter."""
    g = torch.Generator().manual_seed(tokens + classes)
    if kind == "weight":
        x = torch.zeros(tokens, dim)
        x[torch.arange(tokens), torch.arange(tokens) % dim] = 1.0
        w = torch.rand(classes, dim, generator=g) * 80 - 40
    elif kind == "hidden":
        w = torch.zeros(classes, dim)
        w[torch.arange(classes), torch.arange(classes) % dim] = 1.0
        x = torch.rand(tokens, dim, generator=g) * 80 - 40
    else:
        x = torch.zeros(tokens, dim)
        x[torch.arange(tokens), torch.arange(tokens) % dim] = 1.0 + 2.0**-8
        w = torch.where(torch.rand(classes, dim, generator=g) < 0.5, 32.0, -32.0) * (1.0 + 2.0**-8)
        w[1::2] = 0   # half of the classes at zero: a loss is 32 (1 + 2^-8)^2 and a logarithm, or twice that
    t = torch.randint(0, classes, (tokens,), generator=g)
    return x.to(device), w.to(device), t.to(device)


def losses_are_exact(loss, x, w, t):
    """Within what the logarithm and the exponentials of such logits are rounded by: a few times 2^-24 of 80 (2 (1.5 + 1.5) |l|: products with log2 e and their differences), and of their sum's additions.
    A plane less is 2^-17 of the logits, 300 of these units at 40."""
    logits = x.double() @ w.double().T
    want = torch.logsumexp(logits, 1) - logits.gather(1, t[:, None])[:, 0]
    return bool(((loss.double() - want).abs() <= (6 * 40 + 4 * 80 + 100 + w.shape[0] / 64) * U).all())
