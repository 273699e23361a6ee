"""The registered operators and the wrappers below them, which the checks of ops.linear_cross_entropy and ops.rotary do not stand before: the library takes raw pointers and
reads as far as it is told, so what does not go together is refused there too."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from randumb_amd import hip


def head(**changed):
    with FakeTensorMode():
        empty = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="cuda")   # noqa: E731
        a = dict(x=empty(6, 8), weight=empty(10, 8), target=empty(6, dtype=torch.int64), reduction=1, dloss=empty(()), stats=empty(7))
        a.update({k: empty(*v[0], dtype=v[1]) if isinstance(v, tuple) else v for k, v in changed.items()})
        return a


@pytest.mark.parametrize("changed,error", [
    ({"target": ((6,), torch.int32)}, TypeError), ({"x": ((6, 8), torch.float16), "weight": ((10, 8), torch.float16)}, TypeError), ({"weight": ((10, 8), torch.bfloat16)}, TypeError),
    ({"target": ((5,), torch.int64)}, ValueError), ({"target": ((6, 1), torch.int64)}, ValueError), ({"weight": ((10, 7), torch.float32)}, ValueError),
    ({"weight": ((0, 8), torch.float32)}, ValueError), ({"x": ((2, 3, 8), torch.float32)}, ValueError), ({"reduction": 3}, ValueError), ({"reduction": -1}, ValueError)])
def test_head_loss(changed, error):
    a = head(**changed)
    with FakeTensorMode():
        with pytest.raises(error, match="linear_cross_entropy: "):
            hip.linear_cross_entropy_fwd(a["x"], a["weight"], a["target"], -100, a["reduction"])
        with pytest.raises(error, match="linear_cross_entropy: "):
            hip.linear_cross_entropy_bwd(a["dloss"], a["stats"], a["x"], a["weight"], a["target"], -100, a["reduction"])


@pytest.mark.parametrize("changed", [{"stats": ((6,), torch.float32)}, {"stats": ((7,), torch.bfloat16)}, {"dloss": ((6,), torch.float32)}, {"reduction": 0}])
def test_head_loss_statistics(changed):
    a = head(**changed)
    with FakeTensorMode(), pytest.raises(ValueError, match="another size"):
        hip.linear_cross_entropy_bwd(a["dloss"], a["stats"], a["x"], a["weight"], a["target"], -100, a["reduction"])


@pytest.mark.parametrize("q,k,freq,positions,error", [
    (((2, 3, 4, 8), torch.float16), None, ((4,), torch.float32), None, TypeError),
    (((2, 3, 4, 8), torch.float32), ((2, 3, 1, 8), torch.bfloat16), ((4,), torch.float32), None, TypeError),
    (((2, 3, 4, 8), torch.float32), ((2, 2, 1, 8), torch.float32), ((4,), torch.float32), None, ValueError),
    (((2, 3, 4, 8), torch.float32), ((2, 3, 1, 6), torch.float32), ((3,), torch.float32), None, ValueError),
    (((2, 3, 4, 8), torch.float32), None, ((5,), torch.float32), None, ValueError),
    (((2, 3, 4, 8), torch.float32), None, ((4,), torch.float64), None, ValueError),
    (((2, 3, 4, 8), torch.float32), None, ((4,), torch.float32), ((2,), torch.int64), ValueError),
    (((2, 3, 4, 8), torch.float32), None, ((4,), torch.float32), ((3,), torch.int16), ValueError),
    (((2, 3, 4, 8), torch.float32), None, ((4,), torch.float32), ((3, 3), torch.int64), ValueError)])
def test_rotary(q, k, freq, positions, error):
    with FakeTensorMode():
        empty = [None if a is None else torch.empty(a[0], dtype=a[1], device="cuda") for a in (q, k, freq, positions)]
        with pytest.raises(error, match="rotary: "):
            hip.rotary(*empty, False, 1.0)
