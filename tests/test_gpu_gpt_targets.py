"""RT_GPT's loss without logits takes the targets that the loss with logits takes: of the tokens' shape, and flat."""
import pytest
import torch

from randumb_amd import gpt, listgen, stepgen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("random_head", [False, True])
def test_flat_targets(random_head, dtype):
    torch.manual_seed(3)
    n = 4 + 2 * random_head
    with torch.device("cuda"):
        model = gpt.RT_GPT(gpt.RT_GPTConfig(int_dim_gen=listgen([32] * n), seed_gen=stepgen(0, 1), vocab_size=1000, n_layer=1, n_head=2, n_embd=128, random_embedding_and_head=random_head,
                                            loss_without_logits=True)).to(dtype)
    idx = torch.randint(0, 1000, (3, 21), device="cuda")
    target = torch.randint(0, 1000, (3, 21), device="cuda")
    target[1, 5:] = -100
    shaped, flat = model(idx, target), model(idx, target.view(-1))
    assert torch.equal(shaped, flat)
    model.loss_without_logits = False
    assert bool(model(idx, target.view(-1)).isfinite())   # which takes them, too
