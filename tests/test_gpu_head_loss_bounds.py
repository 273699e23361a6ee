"""ops.linear_cross_entropy by tests/head_bounds.py: every value and whole gradients, at the sizes of each of its forms; what is not a number, zeros, another class's row, a part left out or a plane of fp32
left out passes nowhere (tests/test_head_bounds_cpu.py)."""
import math

import pytest
import torch

from head_bounds import IGNORED, check, exact_logits, losses_are_exact
from randumb_amd import hip, ops

pytestmark = pytest.mark.gpu


def inputs(tokens, dim, classes, dtype, ignored=0.0, scale=2.0):
    g = torch.Generator(device="cuda").manual_seed(tokens * 7 + classes)
    x = torch.randn(tokens, dim, device="cuda", generator=g).to(dtype)
    w = (torch.randn(classes, dim, device="cuda", generator=g) * (scale / math.sqrt(dim))).to(dtype)
    t = torch.randint(0, classes, (tokens,), device="cuda", generator=g)
    return x, w, torch.where(torch.rand(tokens, device="cuda", generator=g) < ignored, torch.full_like(t, IGNORED), t)


def held(x, w, t, reduction):
    a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = ops.linear_cross_entropy(a, b, t, ignore_index=IGNORED, reduction=reduction)
    dloss = torch.linspace(0.25, 1.5, len(t), device="cuda") if reduction == "none" else torch.tensor(0.75, device="cuda")
    dx, dw = torch.autograd.grad(loss, [a, b], dloss)
    check(x, w, t, reduction, loss.detach(), dloss, dx, dw)


SIZES = [(1, 8, 1), (1, 64, 2), (2, 1, 7), (3, 7, 257), (17, 100, 1000), (63, 64, 255), (64, 72, 256), (65, 256, 513), (129, 200, 1025), (257, 768, 999), (300, 33, 4001), (511, 520, 300),
         (1025, 257, 777), (24, 960, 9000), (5, 64, 1792)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,dim,classes", SIZES)
def test_small_and_odd(tokens, dim, classes, dtype):
    print(f"case bounds {tokens} x {dim} -> {classes} {dtype}", flush=True)
    for reduction, ignored in (("mean", 0.0), ("none", 0.3), ("sum", 0.1)):
        held(*inputs(tokens, dim, classes, dtype, ignored), reduction)


# one and two blocks a compute unit, one stage of the contraction and several; pieces of the vocabulary: four of 10240 classes and less, four of which the last is a single class, two
@pytest.mark.parametrize("tokens,dim,classes", [(1300, 72, 7000), (1300, 64, 6000), (130, 200, 33000), (130, 600, 32000), (2100, 520, 4000), (1900, 1000, 4300), (700, 1024, 9000), (1025, 999, 10001),
                                                (20011, 72, 40007), ((1 << 20) - 37, 16, 769), (8192, 72, 33003)])
def test_many_tokens_in_bf16(tokens, dim, classes):
    print(f"case bounds {tokens} x {dim} -> {classes} bf16", flush=True)
    for reduction, ignored in (("mean", 0.1), ("none", 0.3)):
        held(*inputs(tokens, dim, classes, torch.bfloat16, ignored), reduction)


# few tokens (the last in pieces); products of fp32, in pieces; planes both ways, in pieces; planes going forward only
@pytest.mark.parametrize("tokens,dim,classes", [(1, 1000, 3001), (5, 259, 5000), (12, 2048, 1500), (32, 128, 2048), (33, 1030, 3001), (64, 300, 4099), (64, 8, 1100000), (400, 512, 6000), (20011, 40, 5003),
                                                (611, 333, 33001), (640, 520, 12000), (577, 1001, 6400), (2050, 260, 50001), (1300, 40, 12001), (4100, 64, 4300)])
def test_many_tokens_in_fp32(tokens, dim, classes):
    print(f"case bounds {tokens} x {dim} -> {classes} fp32", flush=True)
    for reduction, ignored in (("mean", 0.0), ("none", 0.4)):
        held(*inputs(tokens, dim, classes, torch.float32, ignored), reduction)


@pytest.mark.parametrize("kind", ["weight", "hidden", "middle"])
@pytest.mark.parametrize("tokens,dim,classes", [(24, 72, 1001), (300, 72, 1001), (2050, 264, 50001), (4100, 64, 6400)])
def test_exact_logits_in_fp32(tokens, dim, classes, kind):
    """The last two in planes."""
    x, w, t = exact_logits(kind, tokens, dim, classes, "cuda")
    assert losses_are_exact(ops.linear_cross_entropy(x, w, t, reduction="none"), x, w, t)


def test_fp32_without_planes():
    """The same size on fp32 matrix instructions."""
    before = hip.set_f32_split(0)
    try:
        held(*inputs(640, 520, 12000, torch.float32, 0.1), "mean")
        x, w, t = exact_logits("middle", 2050, 264, 50001, "cuda")
        assert losses_are_exact(ops.linear_cross_entropy(x, w, t, reduction="none"), x, w, t)
    finally:
        hip.set_f32_split(before)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_rows_than_a_block_counts_at_once(dtype):
    """Past 16384 tokens a block gathers 64 rows: ignored ones in whole blocks, none, alternating and in the ragged last block; what they hold reaches nothing."""
    tokens, dim, classes = 16384 + 64 * 3 + 21, 24, 1030 if dtype == torch.bfloat16 else 33000
    x, w, t = inputs(tokens, dim, classes, dtype)
    t[64:64 * 40] = IGNORED
    t[64 * 40:64 * 80] = torch.where(torch.arange(64 * 40, device="cuda") % 2 == 0, t[64 * 40:64 * 80], IGNORED)
    t[tokens - 7:] = IGNORED
    for dirty in (False, True):
        if dirty:
            x[t == IGNORED] = math.nan
        held(x, w, t, "none" if dirty else "mean")
