"""Negated frequencies turn the other way: pairs as complex numbers times exp(+i angle), in 64 bits; cosine and sine are good to 2^-22, three roundings follow and one to the result's type."""
import pytest
import torch

from randumb_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_negated_frequencies(interleaved, dtype):
    g = torch.Generator(device="cuda").manual_seed(9)
    q, k = (torch.randn(2, 33, h, 48, device="cuda", generator=g).to(dtype).requires_grad_() for h in (4, 2))
    freq, scale = ops.rotary_frequencies(32, scaling="parts", factor=4.0, original_context=512, device="cuda")
    positions = torch.randint(0, 1 << 20, (2, 33), device="cuda", generator=g)
    out = ops.rotary(q, k, -freq, positions, interleaved=interleaved, scale=scale)
    d = [torch.randn(o.shape, device="cuda", generator=g).to(dtype) for o in out]
    grads = torch.autograd.grad(out, [q, k], d)
    turn = torch.polar(torch.full((), scale, dtype=torch.float64, device="cuda"), (positions.double()[..., None] * freq.double())[:, :, None])
    first, second = (slice(0, 32, 2), slice(1, 32, 2)) if interleaved else (slice(0, 16), slice(16, 32))
    half = torch.finfo(dtype).eps / 2
    for x, got, by in ((q, out[0], turn), (k, out[1], turn), (d[0], grads[0], turn.conj()), (d[1], grads[1], turn.conj())):
        x = x.detach().double()
        z = torch.complex(x[..., first], x[..., second]) * by
        size = (x[..., first].abs() + x[..., second].abs()) * scale
        for part, want in ((first, z.real), (second, z.imag)):
            assert bool(((got.detach().double()[..., part] - want).abs() <= half * want.abs() + (1 + half) * size * (2.0**-22 + 3 * 2.0**-24)).all())
        assert torch.equal(got.detach().double()[..., 32:], x[..., 32:])
