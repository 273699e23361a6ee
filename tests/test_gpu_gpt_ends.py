"""The GPT with the operators at its two ends, rotary positions of another layout and the loss without logits, as it trains with them: against the same model with
stock operators in their place."""
import math

import pytest
import torch
import torch.nn.functional as F

from randumb_amd import gpt, listgen, ops, stepgen

pytestmark = pytest.mark.gpu


def make(dtype, random_head=False, heads=2, rotary=None, **config):
    torch.manual_seed(3)
    n = 8 + 2 * random_head
    with torch.device("cuda"):
        model = gpt.RT_GPT(gpt.RT_GPTConfig(int_dim_gen=listgen([32] * n), seed_gen=stepgen(0, 1), vocab_size=1000, n_layer=2, n_head=heads, n_embd=128,
                                            random_embedding_and_head=random_head, rotary=rotary, **config))
    with torch.no_grad():   # weights that matter: the linears' are 20 times smaller at first than a trained model's
        for name, p in model.named_parameters():
            if name.endswith("weight_coef"):
                p.mul_(4.0)
    return model.to(dtype)


def batch(B=3, T=37):
    g = torch.Generator(device="cuda").manual_seed(5)
    tokens = torch.randint(0, 1000, (B, T + 1), device="cuda", generator=g)
    target = tokens[:, 1:].clone()
    target[0, 20:] = -100   # a padded sequence
    return tokens[:, :-1].contiguous(), target


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


def stock_rotary(self, q, k, positions=None):
    """ops.rotary's formula, in fp32 with angles in fp64."""
    def turn(x):
        freq = self.freq_bits.view(torch.float32).double()
        r = 2 * len(freq)
        angle = torch.arange(x.shape[1], device=x.device).double()[:, None] * freq
        c, s = ((f * self.scale).float()[None, :, None] for f in (angle.cos(), angle.sin()))
        a, b = (x[..., 0:r:2], x[..., 1:r:2]) if self.interleaved else (x[..., :r // 2], x[..., r // 2:r])
        pair = a * c + b * s, b * c - a * s
        return torch.cat((torch.stack(pair, -1).flatten(-2) if self.interleaved else torch.cat(pair, -1), x[..., r:]), -1)
    return turn(q), turn(k)


@pytest.mark.parametrize("rotary", [None, {"interleaved": True}, {"rotary_dim": 32, "scaling": "parts", "factor": 4.0, "original_context": 512},
                                    {"interleaved": True, "rotary_dim": 24, "scaling": "linear", "factor": 2.0, "base": 500.0}])
@pytest.mark.parametrize("random_head", [False, True])
def test_training_step_in_fp32(monkeypatch, rotary, random_head):
    """Everything fp32: two routes of fp32 operators through a model of two blocks, each off by a few of its roundings; 2^-13 leaves them 2000."""
    print(f"case gpt ends {rotary} {random_head}", flush=True)
    idx, target = batch()
    model = make(torch.float32, random_head, rotary=rotary, loss_without_logits=True)
    assert model._loss_without_logits(torch.randn(1, 2, 128, device="cuda"), target[:1, :2]) is not None
    loss = model(idx, target)
    loss.backward()
    stock = make(torch.float32, random_head, rotary=rotary)
    if rotary:
        monkeypatch.setattr(gpt.Rotary, "both", stock_rotary)
    want = stock(idx, target)
    want.backward()
    assert abs(float(loss.detach()) - float(want.detach())) < 2.0**-13 * float(want.detach())
    for (name, p), (_, q) in zip(model.named_parameters(), stock.named_parameters()):
        if q.grad is not None:
            assert rel(p.grad, q.grad) < 2.0**-13, name


@pytest.mark.parametrize("random_head", [False, True])
def test_training_step_in_bf16(random_head):
    """The default model rounds its logits to bf16, each by up to 2^-9 of itself, and its loss moves by no more than the largest of these; the gradients of both are within a
    few roundings of bf16 of each other."""
    idx, target = batch()
    model, stock = make(torch.bfloat16, random_head, loss_without_logits=True), make(torch.bfloat16, random_head)
    loss, want = model(idx, target), stock(idx, target)
    assert loss.dtype == torch.float32
    captured = []
    hook = stock.lm_head.register_forward_hook(lambda m, i, o: captured.append(o))
    stock(idx, target)
    hook.remove()
    top = float(captured[0].detach().float().abs().max())
    # z, which both heads round to bf16, may be rounded to either side: as many roundings again, times the coefficients it meets
    assert abs(float(loss.detach()) - float(want.detach())) <= 2 * 2.0**-8 * top
    loss.backward(), want.backward()
    for (name, p), (_, q) in zip(model.named_parameters(), stock.named_parameters()):
        if q.grad is not None:
            assert p.grad.dtype == torch.bfloat16 and rel(p.grad, q.grad) < 0.05, name


@pytest.mark.parametrize("rotary", [{"interleaved": True}, {"rotary_dim": 32, "scaling": "linear", "factor": 4.0}, {"scaling": "parts", "factor": 4.0, "original_context": 512}])
def test_attention_of_what_is_turned_already(monkeypatch, rotary):
    """bf16: attention's own kernels behind the rotation (of the length that they were: the last one is not) against the stock operators, both by their distance from fp32: q and k
    are rounded once more, every other rounding has its counterpart."""
    idx, target = batch()
    model, stock, exact = (make(torch.bfloat16, rotary=rotary) for _ in range(3))
    exact = exact.float()
    for m in (model, exact):
        m(idx, target).backward()
    monkeypatch.setattr(gpt, "_fused", lambda x: None)
    stock(idx, target).backward()
    for (name, p), (_, q), (_, e) in zip(*(m.named_parameters() for m in (model, stock, exact))):
        if e.grad is not None:
            assert rel(p.grad, e.grad) < 2 * rel(q.grad, e.grad) + 2.0**-8, name


def test_types_devices_and_states():
    """The frequencies survive a change of the module's type, and neither they nor the identity are in its state."""
    model = make(torch.bfloat16, True, rotary={"rotary_dim": 20}, loss_without_logits=True)
    rotary = model.h[0].attn.rotary
    want, _ = ops.rotary_frequencies(20, device="cuda")
    assert torch.equal(rotary.freq_bits.view(torch.float32), want) and model.unit_coefs.dtype == torch.bfloat16
    assert list(model.state_dict()) == list(make(torch.bfloat16, True).state_dict())
    with pytest.raises(ValueError):
        gpt.Rotary(16, rotary_dim=18)


def test_a_head_that_is_more_than_its_product():
    """Hooks see the logits: the default route."""
    idx, target = batch()
    model = make(torch.float32, loss_without_logits=True)
    want = float(model(idx, target))
    seen = []
    hook = model.lm_head.register_forward_hook(lambda m, i, o: seen.append(o.shape))
    assert abs(float(model(idx, target)) - want) < 1e-4 and seen == [(3, 37, 1000)]
    hook.remove()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert math.isfinite(float(model(idx, target)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_step_in_a_graph(dtype):
    """Captured once, replayed with other tokens and eager steps in between.  A layer's weight keeps its coefficients' accumulators, which belong to the stream on which the
    layer was made: here the one that captures."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        captured_and_replayed(dtype, side)
    torch.cuda.synchronize()


def captured_and_replayed(dtype, side):
    model = make(dtype, rotary={"interleaved": True}, loss_without_logits=True)
    params = [p for n, p in model.named_parameters() if "scale_bias" not in n]
    idx, target = batch()

    def step():
        loss = model(idx, target)
        return [loss.detach(), *torch.autograd.grad(loss, params)]

    for _ in range(2):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    for i in range(3):
        idx.copy_((idx * 7 + i) % 1000)
        eager = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert rel(a, b) < (1e-2 if dtype == torch.bfloat16 else 1e-5)
        assert F.mse_loss(out[0], eager[0]) < 1e-6
