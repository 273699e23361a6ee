"""RT_GPT's rotation of another layout is a module like any other: hooks on it see it called, and what they return is used; so is a replaced forward."""
import pytest
import torch

from randumb_amd import gpt, listgen, stepgen

pytestmark = pytest.mark.gpu


def make(dtype):
    torch.manual_seed(3)
    with torch.device("cuda"):
        model = gpt.RT_GPT(gpt.RT_GPTConfig(int_dim_gen=listgen([32] * 8), seed_gen=stepgen(0, 1), vocab_size=1000, n_layer=2, n_head=2, n_embd=128, rotary={"interleaved": True}))
    return model.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_hooks_and_replaced_forwards(dtype, monkeypatch):
    model = make(dtype)
    idx, target = (torch.randint(0, 1000, (2, 21), device="cuda") for _ in range(2))
    want = model(idx, target)
    rotary = model.h[1].attn.rotary
    seen = []
    hook = rotary.register_forward_hook(lambda m, i, o: seen.append(o.shape))
    hooked = model(idx, target)
    assert seen == [(2, 21, 2, 64)] * 2   # queries and keys
    if dtype == torch.float32:
        assert torch.equal(hooked, want)   # the same turns of the same values
    hook.remove()
    hook = rotary.register_forward_hook(lambda m, i, o: o * float("nan"))
    assert bool(model(idx, target).isnan())
    hook.remove()
    assert torch.equal(model(idx, target), want)
    rotary.forward = lambda x: x * float("nan")
    assert bool(model(idx, target).isnan())
    del rotary.forward
    with monkeypatch.context() as m:
        m.setattr(gpt.Rotary, "forward", lambda self, x: x * float("nan"))
        assert bool(model(idx, target).isnan())
    assert torch.equal(model(idx, target), want)
