"""ops.linear_cross_entropy and ops.rotary without a GPU: what they refuse, what a tracer is told, and the frequencies."""
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from randumb_amd import SillyLinear, _lib, ops

X, W, T = torch.zeros(4, 8), torch.zeros(10, 8), torch.zeros(4, dtype=torch.int64)


@pytest.mark.parametrize("args,kwargs,error", [
    ((X, W, T), {"reduction": "average"}, ValueError),
    ((X.double(), W.double(), T), {}, TypeError),
    ((X.half(), W.half(), T), {}, TypeError),
    ((X.bfloat16(), W, T), {}, TypeError),
    ((X, W, T.float()), {}, TypeError),
    ((X, W, T.bool()), {}, TypeError),
    ((X, W[:, :7], T), {}, ValueError),
    ((X, W, T[:3]), {}, ValueError),
    ((X, W, T[:, None]), {}, ValueError),
    ((X, W[0], T), {}, ValueError),
    ((X, W[:0], T), {}, ValueError),
    ((X[:, :0], W[:, :0], T), {}, ValueError),
    ((X[0, 0], W, T[0]), {}, ValueError),
    ((X, W, T), {}, NotImplementedError),   # no CPU path
])
def test_head_loss_refuses(args, kwargs, error):
    with pytest.raises(error):
        ops.linear_cross_entropy(*args, **kwargs)


def test_head_loss_refuses_a_pseudorandom_weight():
    with pytest.raises(TypeError, match="dense"):
        ops.linear_cross_entropy(X, SillyLinear(8, 10, [4, 4], [0, 1]).weight, T)


Q, K, FREQ = torch.zeros(2, 3, 4, 8), torch.zeros(2, 3, 1, 8), torch.ones(4)


@pytest.mark.parametrize("args,kwargs,error", [
    ((Q.half(), None, FREQ), {}, TypeError),
    ((Q, K.bfloat16(), FREQ), {}, TypeError),
    ((Q[0], None, FREQ), {}, ValueError),
    ((Q, K[:1], FREQ), {}, ValueError),
    ((Q, K[..., :6], FREQ), {}, ValueError),
    ((Q, K, torch.ones(5)), {}, ValueError),
    ((Q, K, FREQ[:0]), {}, ValueError),
    ((Q, K, FREQ.double()), {}, ValueError),
    ((Q, K, FREQ[None]), {}, ValueError),
    ((torch.zeros(1, 1, 1, 4096), None, torch.ones(1025)), {}, ValueError),
    ((Q, K, FREQ, torch.zeros(3)), {}, ValueError),
    ((Q, K, FREQ, torch.zeros(2, dtype=torch.int64)), {}, ValueError),
    ((Q, K, FREQ, torch.zeros(3, 3, dtype=torch.int64)), {}, ValueError),
    ((Q, K, FREQ), {}, NotImplementedError),
])
def test_rotary_refuses(args, kwargs, error):
    with pytest.raises(error):
        ops.rotary(*args, **kwargs)


@pytest.mark.parametrize("args,kwargs", [((7,), {}), ((0,), {}), ((8, -1.0), {}), ((8,), {"factor": 2.0}), ((8,), {"scaling": "other"}), ((8,), {"scaling": "linear", "factor": 0.0}),
                                         ((2,), {"scaling": "base", "factor": 2.0}), ((8,), {"scaling": "parts", "factor": 2.0}),
                                         ((8,), {"scaling": "parts", "factor": 2.0, "original_context": 64, "low": 4.0, "high": 2.0})])
def test_frequencies_refuse(args, kwargs):
    with pytest.raises(ValueError):
        ops.rotary_frequencies(*args, **kwargs)


def test_frequencies():
    plain, scale = ops.rotary_frequencies(128, 500000.0)
    assert plain.dtype == torch.float32 and scale == 1.0
    want = [500000.0 ** (-2 * i / 128) for i in range(64)]
    assert plain.tolist() == torch.tensor(want, dtype=torch.float64).float().tolist()
    assert torch.equal(ops.rotary_frequencies(128, 500000.0, scaling="linear", factor=4.0)[0], plain / 4)
    larger, scale = ops.rotary_frequencies(128, scaling="base", factor=8.0)
    plain = ops.rotary_frequencies(128)[0]
    assert scale == 1.0 and float(larger[0]) == 1.0 and math.isclose(float(larger[-1]), float(plain[-1]) / 8, rel_tol=1e-6)
    parts, scale = ops.rotary_frequencies(128, scaling="parts", factor=8.0, original_context=4096)
    assert math.isclose(scale, 0.1 * math.log(8.0) + 1.0)
    turns = 4096 * plain.double() / (2 * math.pi)
    assert torch.equal(parts[turns > 33 * 1.2], plain[turns > 33 * 1.2])
    slow = turns < 0.8
    assert bool(slow.any()) and torch.allclose(parts[slow], plain[slow] / 8, rtol=1e-6)
    assert bool((parts <= plain).all()) and bool((parts >= plain / 8 * (1 - 1e-6)).all())


def test_a_tracer_sees_sizes():
    with FakeTensorMode():
        x, w = torch.empty(2, 6, 16, device="cuda", dtype=torch.bfloat16), torch.empty(50, 16, device="cuda", dtype=torch.bfloat16)
        t = torch.empty(2, 6, device="cuda", dtype=torch.int64)
        for reduction, shape in (("mean", ()), ("sum", ()), ("none", (2, 6))):
            loss = ops.linear_cross_entropy(x, w, t, reduction=reduction)
            assert loss.shape == shape and loss.dtype == torch.float32
        grads = torch.ops.rten.linear_cross_entropy_bwd(loss.view(-1), torch.empty(13, device="cuda"), x.view(12, 16), w, t.view(12), -100, 0, True, True)
        assert [g.shape for g in grads] == [(12, 16), w.shape] and grads[0].dtype == grads[1].dtype == torch.bfloat16
        q, k = (torch.empty(2, 6, h, 16, device="cuda") for h in (4, 2))
        out = ops.rotary(q, k, torch.empty(8, device="cuda"))
        assert [o.shape for o in out] == [q.shape, k.shape]


def test_the_library_refuses():
    """Argument errors come back as codes before anything is launched."""
    L = _lib.load()
    one = 4096   # an address that nothing reads
    size = L.rdb_linear_cross_entropy_workspace_bytes
    assert size(8, 64, 100, _lib.RDB_BF16, one, 64, one, 64, 0, 0, 0) > 0
    assert size(8, 64, 100, 7, one, 64, one, 64, 0, 0, 0) == 0 and size(0, 64, 100, 1, one, 64, one, 64, 0, 0, 0) == 0
    assert size(1 << 20, 1 << 10, 100, 1, one, 1 << 10, one, 1 << 10, 0, 0, 0) == 0
    fwd = lambda **k: L.rdb_linear_cross_entropy_fwd(*{**dict(loss=one, stats=one, logits=None, x=one, ldx=64, w=one, ldw=64, dtype=1, target=one, tokens=8, dim=64, classes=100,  # noqa: E731
                                                             ignore=-100, reduction=1, ws=one, n=0, stream=None), **k}.values())
    assert fwd() == -6 and fwd(dtype=2) == -3 and fwd(tokens=0) == -2 and fwd(dim=0) == -2 and fwd(classes=0) == -2 and fwd(ldx=63) == -2 and fwd(ldw=63) == -2
    assert fwd(reduction=3) == -2 and fwd(loss=None) == -1 and fwd(ws=None, n=1 << 40) == -6 and fwd(ldw=1 << 20) == -5 and fwd(tokens=1 << 23) == -5
    bwd = lambda **k: L.rdb_linear_cross_entropy_bwd(*{**dict(dx=one, dw=one, dloss=one, stats=one, logits=None, x=one, ldx=64, w=one, ldw=64, dtype=1, target=one, tokens=8, dim=64,  # noqa: E731
                                                             classes=100, ignore=-100, reduction=1, ws=one, n=0, stream=None), **k}.values())
    assert bwd() == -6 and bwd(dx=None, dw=None) == 0 and bwd(dx=one + 2) == -4 and bwd(dloss=None) == -1 and bwd(reduction=-1) == -2
    rows = lambda heads=2: _lib.ctypes.byref(_lib.RotaryRows(one, one, heads, 64, 64, 16))  # noqa: E731
    rot = lambda **k: L.rdb_rotary(*{**dict(q=rows(), k=None, dtype=1, batch=1, seq=1, dim=16, freq=one, pairs=8, pos=None, pos_bytes=0, pb=0, pt=0, interleaved=0,  # noqa: E731
                                            scale=1.0, inverse=0, stream=None), **k}.values())
    assert rot(dtype=3) == -3 and rot(q=None) == -1 and rot(freq=None) == -1 and rot(pairs=9) == -2 and rot(dim=0) == -2 and rot(pos=one, pos_bytes=2) == -3
    assert rot(dim=4096, pairs=1025) == -5 and rot(batch=0) == 0 and rot(q=rows(0)) == 0


def test_more_logits_than_a_launch_has_threads_are_refused():
    """2^21 - 1 tokens of 8 values and 2^30 classes: by memory they would fit; the number of tiles is past 2^32."""
    L = _lib.load()
    sizes = ((1 << 21) - 1, 8, 1 << 30)
    for tokens, dim, classes in (sizes, (1 << 20, 8, 1 << 18)):
        assert L.rdb_linear_cross_entropy_workspace_bytes(tokens, dim, classes, _lib.RDB_BF16, 4096, 8, 4096, 8, 0, 0, 0) == 0
        assert L.rdb_linear_cross_entropy_fwd(4096, 4096, None, 4096, 8, 4096, 8, _lib.RDB_BF16, 4096, tokens, dim, classes, -100, 1, 4096, 1 << 62, None) == -5
    assert L.rdb_linear_cross_entropy_workspace_bytes((1 << 20) - 128, 8, 1 << 18, _lib.RDB_BF16, 4096, 8, 4096, 8, 0, 0, 0) > 0


def test_logits_that_are_kept():
    """fp32, few beside the weight and in one piece; others are refused."""
    L = _lib.load()
    keeps = lambda tokens, dim, classes, dtype=_lib.RDB_F32, ldw=0: L.rdb_linear_cross_entropy_keeps(tokens, dim, classes, dtype, ldw or dim)  # noqa: E731
    assert keeps(16, 64, 1000) == 16000 and keeps(17, 64, 1000) == 0 and keeps(16, 64, 1000, _lib.RDB_BF16) == 0 and keeps(0, 64, 1000) == 0
    assert keeps(512, 2048, 1 << 17) == 1 << 26 and keeps(512, 2048, 1 << 18) == 0 and keeps(16, 64, 100000, ldw=1 << 19) == 0
    sizes = 4096, 64, 4096, 64, _lib.RDB_F32, 4096, 17, 64, 1000, -100, 1, 4096, 1 << 40, None
    assert L.rdb_linear_cross_entropy_fwd(4096, 4096, 4096, *sizes) == -5 and L.rdb_linear_cross_entropy_bwd(4096, 4096, 4096, 4096, 4096, *sizes) == -5
