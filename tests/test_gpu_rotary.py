"""ops.rotary against the formula in 64 bits: cosine and sine are good to 2^-22 (their argument, reduced in 64 bits, is rounded to 32, and so are they), three roundings follow
in fp32 and one to the result's type."""
import math

import pytest
import torch

from randumb_amd import ops
from randumb_amd.gpt import Rotary

pytestmark = pytest.mark.gpu


def turned(x, freq, positions, interleaved, scale, inverse=False):
    r, x = 2 * len(freq), x.detach().double().clone()
    angle = (positions.double()[..., None] * freq.double())[:, :, None]
    c, s = angle.cos() * scale, angle.sin() * scale * (-1 if inverse else 1)
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., first].clone(), x[..., second].clone()
    x[..., first], x[..., second] = a * c + b * s, b * c - a * s
    return x


def close(got, x, want, freq, interleaved, scale):
    r, half = 2 * len(freq), torch.finfo(got.dtype).eps / 2
    x = x.detach().double().abs()
    pair = x[..., :r].view(*x.shape[:-1], -1, 2).sum(-1).repeat_interleave(2, -1) if interleaved else (x[..., :r // 2] + x[..., r // 2:r]).repeat(1, 1, 1, 2)
    tol = half * want[..., :r].abs() + (1 + half) * pair * scale * (2.0**-22 + 3 * 2.0**-24) + 1e-37
    assert got.shape == x.shape and bool(((got[..., :r].double() - want[..., :r]).abs() <= tol).all())
    assert torch.equal(got[..., r:].double(), want[..., r:])


CASES = [  # batch, time, heads, kv heads, head dim, rotary dim
    (1, 1, 1, 1, 2, 2), (2, 3, 4, 2, 64, 64), (1, 5, 3, 1, 128, 64), (3, 7, 2, 2, 80, 32), (2, 33, 5, 1, 90, 46), (1, 130, 8, 8, 96, 96), (4, 1, 32, 8, 128, 128),
    (2, 257, 12, 12, 64, 64), (1, 2, 1, 1, 2048, 2048), (1, 700, 3, 3, 24, 8), (1, 3, 2, 1, 257, 10)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_values_and_gradients(case, interleaved, dtype):
    batch, time, heads, kv, dim, rdim = case
    print(f"case rotary {case} {interleaved} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(sum(case))
    qkv = torch.randn(batch, time, heads + 2 * kv, dim, device="cuda", generator=g).to(dtype)
    freq, _ = ops.rotary_frequencies(rdim, device="cuda")
    positions = torch.randint(0, 1 << 20, (batch, 1), device="cuda", generator=g) + torch.arange(time, device="cuda")
    for scale, pos in ((1.0, positions), (1.25, None)):
        q, k = qkv[:, :, :heads].detach().requires_grad_(), qkv[:, :, heads:heads + kv].detach().requires_grad_()
        oq, ok = ops.rotary(q, k, freq, pos, interleaved=interleaved, scale=scale)
        at = torch.arange(time, device="cuda").expand(batch, time) if pos is None else pos
        assert oq.is_contiguous() and ok.is_contiguous() and oq.dtype == dtype
        close(oq.detach(), q, turned(q, freq, at, interleaved, scale), freq, interleaved, scale)
        close(ok.detach(), k, turned(k, freq, at, interleaved, scale), freq, interleaved, scale)
        dq, dk = (torch.randn(t.shape, device="cuda", generator=g).to(dtype) for t in (oq, ok))
        for got, d in zip(torch.autograd.grad([oq, ok], [q, k], [dq, dk]), (dq, dk)):
            close(got, d, turned(d, freq, at, interleaved, scale, True), freq, interleaved, scale)


def test_strides_positions_and_one_side():
    g = torch.Generator(device="cuda").manual_seed(1)
    base = torch.randn(2, 9, 4, 64, device="cuda", generator=g)
    freq, _ = ops.rotary_frequencies(32, device="cuda")
    pos = torch.tensor([[0, 5, 2, 2, 100, -3, 1 << 30, 7, 8], [9, 8, 7, 6, 5, 4, 3, 2, 1]], device="cuda")
    want, _ = ops.rotary(base, None, freq, pos)
    close(want, base, turned(base, freq, pos, False, 1.0), freq, False, 1.0)
    views = [base.transpose(1, 2).contiguous().transpose(1, 2), base.transpose(0, 1).contiguous().transpose(0, 1), base.transpose(2, 3).contiguous().transpose(2, 3)]
    room = torch.full((2, 9, 4, 67), math.nan, device="cuda")
    room[..., 1:65] = base
    views += [room[..., 1:65], torch.flip(base, [1]).flip([1])]
    for v in views:
        assert torch.equal(ops.rotary(v, None, freq, pos)[0], want) and ops.rotary(v, None, freq, pos)[1] is None
    for p in (pos.int(), pos.T.contiguous().T, torch.stack([pos, pos], -1)[..., 0]):
        assert torch.equal(ops.rotary(base, None, freq, p)[0], want)
    one = pos[:1]
    same = ops.rotary(base, base[:, :, :2], freq, one)
    for other in (one[0], one.expand(2, 9)):
        assert all(torch.equal(a, b) for a, b in zip(same, ops.rotary(base, base[:, :, :2], freq, other)))
    assert torch.equal(same[1], same[0][:, :, :2])
    # a query broadcast over the sequences: its gradient is the sum over them
    q = torch.randn(1, 9, 4, 64, device="cuda", generator=g).requires_grad_()
    out = ops.rotary(q.expand(2, 9, 4, 64), None, freq, pos)[0]
    d = torch.randn(out.shape, device="cuda", generator=g)
    assert torch.allclose(torch.autograd.grad(out, q, d)[0].double(), turned(d, freq, pos, False, 1.0, True).sum(0, keepdim=True), rtol=0, atol=1e-5)
    for shape in ((0, 9, 4, 64), (2, 0, 4, 64), (2, 9, 0, 64)):
        assert ops.rotary(torch.empty(shape, device="cuda"), None, freq)[0].shape == shape
    # keys alone wanted, and a gradient of one side alone
    k = base[:, :, :1].detach().requires_grad_()
    oq, ok = ops.rotary(base, k, freq, pos)
    dk = torch.randn(ok.shape, device="cuda", generator=g)
    close(torch.autograd.grad(ok, k, dk)[0], dk, turned(dk, freq, pos, False, 1.0, True), freq, False, 1.0)


def test_the_model_s_own_rotation():
    """The default layout and frequencies turn as the model's stock rotation does, which forms its angles in 32 bits."""
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(2, 50, 3, 80, device="cuda", generator=g)
    freq, scale = ops.rotary_frequencies(80, device="cuda")
    assert scale == 1.0
    assert float((ops.rotary(x, None, freq)[0] - Rotary(80).cuda()(x)).abs().max()) < 50 * 2.0**-22 * float(x.abs().max()) * 2


def test_gradients_of_higher_order_and_operators():
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(1, 4, 2, 16, device="cuda", generator=g).requires_grad_()
    freq, _ = ops.rotary_frequencies(16, device="cuda")
    out = ops.rotary(q, None, freq)[0]
    first = torch.autograd.grad((out**2).sum() / 2, q, create_graph=True)[0]
    assert torch.allclose(first, q, atol=1e-5)   # a rotation keeps lengths
    second = torch.autograd.grad(first.sum(), q)[0]
    assert torch.allclose(second, torch.ones_like(q), atol=1e-5)
    again = torch.ops.rten.rotary(q, None, freq, None, False, 1.0, False)[0]
    assert torch.equal(again, out)
    d = torch.randn(out.shape, device="cuda", generator=g)
    assert torch.equal(torch.autograd.grad(again, q, d)[0], torch.autograd.grad(ops.rotary(q, None, freq)[0], q, d)[0])


def test_streams_and_graphs():
    g = torch.Generator(device="cuda").manual_seed(4)
    q, k = (torch.randn(2, 64, h, 64, device="cuda", generator=g).bfloat16().requires_grad_() for h in (6, 2))
    freq, _ = ops.rotary_frequencies(64, device="cuda")
    pos = torch.arange(64, device="cuda")
    d = [torch.randn_like(t) for t in (q, k)]

    def step():
        out = ops.rotary(q, k, freq, pos)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, [q, k], d))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(want, step()))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        pos.add_(1000)
        with torch.no_grad():
            q.mul_(0.5)
        eager = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, out))


@pytest.mark.parametrize("heads", [40, 256])
def test_large_ones(heads):
    """More than the chip's last-level cache holds, and more than 2^31 values: the first, the middle and the last positions."""
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.empty(2, 35000, heads, 128, device="cuda", dtype=torch.bfloat16).uniform_(-1, 1, generator=g)
    freq, _ = ops.rotary_frequencies(128, device="cuda")
    for interleaved in (False, True):
        out = ops.rotary(q, None, freq, interleaved=interleaved)[0]
        for at in (slice(0, 40), slice(17000, 17040), slice(34960, 35000)):
            pos = torch.arange(35000, device="cuda")[at].expand(2, 40)
            close(out[:, at], q[:, at], turned(q[:, at], freq, pos, interleaved, 1.0), freq, interleaved, 1.0)
        del out


def test_more_blocks_than_one_launch():
    """2^24 + 5 sequences of one token, a block each: the first, the last, and those around the ends of a launch."""
    n = (1 << 24) + 5
    q = torch.arange(n, device="cuda", dtype=torch.int32).remainder(251).sub(125).div(125).to(torch.bfloat16).view(n, 1, 1, 1).expand(n, 1, 1, 4).contiguous()
    pos = torch.arange(n, device="cuda", dtype=torch.int32).view(n, 1)
    freq, _ = ops.rotary_frequencies(4, device="cuda")
    out = ops.rotary(q, None, freq, pos)[0]
    for at in (slice(0, 40), slice((1 << 23) - 20, (1 << 23) + 20), slice((1 << 24) - 20, (1 << 24) + 5)):
        close(out[at], q[at], turned(q[at], freq, pos[at], False, 1.0), freq, False, 1.0)


def test_refusals_on_the_gpu():
    """The same errors as on the CPU, where the extension does not see the call."""
    q, f = torch.randn(2, 3, 4, 8, device="cuda"), ops.rotary_frequencies(8, device="cuda")[0]
    pos = torch.arange(3, device="cuda")
    for error, args in [(TypeError, (q.half(), None, f)), (TypeError, (q, q.bfloat16(), f)), (ValueError, (q[0], None, f)), (ValueError, (q, q[:, :2], f)), (ValueError, (q, q[..., :4], f)),
                        (ValueError, (q, None, f.double())), (ValueError, (q, None, f[:0])), (ValueError, (q, None, torch.cat([f, f]))), (ValueError, (q, None, f, pos.float())),
                        (ValueError, (q, None, f, pos[:2])), (ValueError, (q, None, f, pos.expand(3, 3))), (ValueError, (q, None, f, pos[0]))]:
        with pytest.raises(error, match="rotary: "):
            ops.rotary(*args)
    with pytest.raises(ValueError, match="1024 at most"):
        ops.rotary(torch.randn(1, 1, 1, 2050, device="cuda"), None, torch.ones(1025, device="cuda"))
