"""The operators at the two ends of a language model, as cases that can be timed and compared: the loss of its output head and
the rotary positions of its attention.

head    ``ops.linear_cross_entropy``: softmax cross entropy of ``x @ weight.T`` over a large vocabulary, logits never kept; a row's
        logits are scored once (``train`` false) or the loss is followed by the gradients of x and of the weight
rotary  ``ops.rotary``: queries and keys turned by their positions, pairs half a rotary dimension apart or side by side, all of a head or
        its first part, with given frequencies and a scale; ``train``: and the gradients of both

Sizes are those of this repository's configurations (GPT-2 small: 8 x 1024 tokens, 12 heads of 64, 50304 classes, k = 256; 4096
features) and the ranges around them.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_IGNORED = -100


def listed():
    return [
        # 16 continuations scored by their next token: the weight is read once, launches and latency count
        {"name": "head_score_16tok", "kind": "head", "tokens": 16, "dim": 768, "classes": 50304, "dtype": "bf16", "reduction": "none", "ignored": 0.0, "train": False},
        # evaluation of a text, nothing a multiple of anything
        {"name": "head_eval_odd", "kind": "head", "tokens": 1999, "dim": 1001, "classes": 30011, "dtype": "bf16", "reduction": "mean", "ignored": 0.1, "train": False},
        # GPT-2 small's head, 8 sequences of 1024
        {"name": "head_gpt2_train", "kind": "head", "tokens": 8192, "dim": 768, "classes": 50304, "dtype": "bf16", "reduction": "mean", "ignored": 0.0, "train": True},
        # the same model's head as a product with the coefficients of a pseudorandom weight
        {"name": "head_coefs_train", "kind": "head", "tokens": 8192, "dim": 256, "classes": 50304, "dtype": "bf16", "reduction": "mean", "ignored": 0.0, "train": True},
        # a wide model with a large vocabulary
        {"name": "head_wide_train", "kind": "head", "tokens": 4096, "dim": 4096, "classes": 65536, "dtype": "bf16", "reduction": "mean", "ignored": 0.0, "train": True},
        # torch's default type, a micro-batch
        {"name": "head_fp32_train", "kind": "head", "tokens": 2048, "dim": 768, "classes": 50304, "dtype": "fp32", "reduction": "mean", "ignored": 0.0, "train": True},
        # padded sequences, their tokens' losses weighted by the program; no size a multiple of 8
        {"name": "head_odd_weighted_train", "kind": "head", "tokens": 1025, "dim": 999, "classes": 10001, "dtype": "bf16", "reduction": "none", "ignored": 0.3, "train": True},
        # the smallest training step
        {"name": "head_small_fp32_train", "kind": "head", "tokens": 128, "dim": 256, "classes": 1000, "dtype": "fp32", "reduction": "mean", "ignored": 0.0, "train": True},
        # one new token for each of 16 sequences of different lengths
        {"name": "rotary_decode", "kind": "rotary", "batch": 16, "seq": 1, "heads": 32, "kv_heads": 8, "head_dim": 128, "rotary_dim": 128, "dtype": "bf16",
         "interleaved": False, "scale": 1.0, "context": 131072, "train": False},
        # GPT-2 small's attention
        {"name": "rotary_gpt2_train", "kind": "rotary", "batch": 8, "seq": 1024, "heads": 12, "kv_heads": 12, "head_dim": 64, "rotary_dim": 64, "dtype": "bf16",
         "interleaved": False, "scale": 1.0, "context": 1024, "train": True},
        # a long prompt, neighbouring pairs of half of each head, frequencies stretched to the context
        {"name": "rotary_long_partial", "kind": "rotary", "batch": 1, "seq": 32768, "heads": 32, "kv_heads": 8, "head_dim": 128, "rotary_dim": 64, "dtype": "bf16",
         "interleaved": True, "scale": 1.2, "context": 1048576, "train": False},
        # torch's default type; odd numbers of everything, a part of the head
        {"name": "rotary_odd_fp32_train", "kind": "rotary", "batch": 3, "seq": 1001, "heads": 5, "kv_heads": 1, "head_dim": 90, "rotary_dim": 46, "dtype": "fp32",
         "interleaved": False, "scale": 1.0, "context": 4096, "train": True},
    ]


# ------------------------------------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """Mostly a multiple of 64, as nearly all models' sizes are; one in four any number."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.25 else max(64, (n + 32) // 64 * 64)


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    train = rng.random() < 0.7
    if rng.random() < 0.6:
        tokens, dim, classes = _log(rng, 1, 8192), _size(rng, 64, 4096), _size(rng, 1000, 131072)
        most = (4096 * 4096 * 65536 if dtype == "bf16" else 2048 * 768 * 50304) // (dim * classes)
        return {"kind": "head", "tokens": max(1, min(tokens, most)), "dim": dim, "classes": classes, "dtype": dtype,
                "reduction": rng.choice(["mean", "mean", "sum", "none"]), "ignored": rng.choice([0.0, 0.1, 0.5]), "train": train}
    kv_heads = rng.randint(1, 8)
    head_dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 256, 2 * rng.randint(8, 128)])
    rotary_dim = head_dim if rng.random() < 0.6 else 2 * rng.randint(1, head_dim // 2)
    heads = kv_heads * rng.randint(1, 8)
    seq = _log(rng, 1, 32768)
    batch = _log(rng, 1, max(1, min(64, 32768 * 40 * 128 // (seq * (heads + kv_heads) * head_dim * (2 if train else 1) * (2 if dtype == "fp32" else 1)))))
    return {"kind": "rotary", "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "rotary_dim": rotary_dim, "dtype": dtype,
            "interleaved": rng.random() < 0.5, "scale": rng.choice([1.0, 1.2]), "context": max(seq, _log(rng, 1024, 1048576)), "train": train}


# ------------------------------------------------------------------------------------------------ what the program has in hand
def _inputs(case, seed):
    """The tensors of a case.  head: hidden states after a normalisation and a weight that has learned something: a token's own class scores
    about 6 above the others, whose logits have a deviation of 2.  rotary: queries and keys as views of one projection's output."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    if case["kind"] == "head":
        t, d, v = case["tokens"], case["dim"], case["classes"]
        w = torch.randn(v, d, device="cuda", generator=g) * (2.0 / math.sqrt(d))
        target = torch.randint(0, v, (t,), device="cuda", generator=g)
        x = torch.randn(t, d, device="cuda", generator=g) + 1.5 * w[target]
        target = torch.where(torch.rand(t, device="cuda", generator=g) < case["ignored"], torch.full_like(target, _IGNORED), target)
        if case["ignored"]:
            target[0] = 0   # a mean over nothing is no case that counts
        dloss = torch.rand(t, device="cuda", generator=g) if case["reduction"] == "none" else torch.full((), 0.5, device="cuda")
        return {"x": x.to(dtype), "w": w.to(dtype), "target": target, "dloss": dloss}
    b, t, h, k, d, r = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "head_dim", "rotary_dim"))
    qkv = torch.randn(b, t, h + 2 * k, d, device="cuda", generator=g).to(dtype)
    first = torch.randint(0, case["context"] - t + 1, (b, 1), device="cuda", generator=g)
    freq = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    if case["context"] > 8192:   # turns that a context of 8192 does not complete are stretched
        freq = torch.where(freq * 8192 < 2 * math.pi, freq * (8192 / case["context"]), freq)
    return {"q": qkv[:, :, :h], "k": qkv[:, :, h:h + k], "positions": first + torch.arange(t, device="cuda"), "freq": freq.float().cuda(),
            "dq": torch.randn(b, t, h, d, device="cuda", generator=g).to(dtype), "dk": torch.randn(b, t, k, d, device="cuda", generator=g).to(dtype)}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["train"]:
        for n in ("x", "w") if case["kind"] == "head" else ("q", "k"):
            s[n] = s[n].detach().requires_grad_()
    return s


# ------------------------------------------------------------------------------------------------ one pass
def _head(s):
    case, target = s["case"], s["target"]
    x, w = s["x"].detach().float(), s["w"].detach().float()
    logits = x @ w.T
    counts = target != _IGNORED
    own_class = torch.where(counts, target, torch.zeros_like(target))[:, None]
    top = logits.amax(1, keepdim=True)
    lse = (logits - top).exp().sum(1, keepdim=True).log() + top
    nll = torch.where(counts, (lse - logits.gather(1, own_class))[:, 0], torch.zeros_like(top[:, 0]))
    weight = counts.float()
    loss = nll
    if case["reduction"] != "none":
        weight = weight / weight.sum() if case["reduction"] == "mean" else weight
        loss = (nll * (1.0 if case["reduction"] == "sum" else weight)).sum()
    if not case["train"]:
        return [loss]
    g = (logits - lse).exp()
    g.scatter_add_(1, own_class, torch.full_like(own_class, -1, dtype=torch.float32))
    g *= (weight * s["dloss"])[:, None]
    return [loss, (g @ w).to(s["x"].dtype), (g.T @ x).to(s["w"].dtype)]


def _turn(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    f = x.detach().float()
    a, b = (f[..., 0:r:2], f[..., 1:r:2]) if interleaved else (f[..., :r // 2], f[..., r // 2:r])
    pair = (a * cos + b * sin, b * cos - a * sin)
    turned = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
    return torch.cat((turned, f[..., r:]), -1).to(x.dtype)


def _rotary(s):
    case = s["case"]
    angle = (s["positions"].double()[..., None] * s["freq"].double())[:, :, None]   # far positions: 32 bits lose the angle
    cos, sin = (angle.cos() * case["scale"]).float(), (angle.sin() * case["scale"]).float()
    out = [_turn(s["q"], cos, sin, case["interleaved"]), _turn(s["k"], cos, sin, case["interleaved"])]
    if case["train"]:
        out += [_turn(s["dq"], cos, -sin, case["interleaved"]), _turn(s["dk"], cos, -sin, case["interleaved"])]
    return out


def run(s):
    case = s["case"]
    if not own:
        return _head(s) if case["kind"] == "head" else _rotary(s)
    from randumb_amd import ops

    if case["kind"] == "head":
        loss = ops.linear_cross_entropy(s["x"], s["w"], s["target"], ignore_index=_IGNORED, reduction=case["reduction"])
        return [loss.detach(), *torch.autograd.grad(loss, [s["x"], s["w"]], s["dloss"])] if case["train"] else [loss]
    q, k = ops.rotary(s["q"], s["k"], s["freq"], s["positions"], interleaved=case["interleaved"], scale=case["scale"])
    return [q.detach(), k.detach(), *torch.autograd.grad([q, k], [s["q"], s["k"]], [s["dq"], s["dk"]])] if case["train"] else [q, k]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    """head: the product of x with the weight, and for the gradients one for each of them.  rotary: four multiplications and two additions a pair."""
    size = 2.0 if case["dtype"] == "bf16" else 4.0
    times = 2 if case["train"] else 1
    if case["kind"] == "head":
        t, d, v = case["tokens"], case["dim"], case["classes"]
        loss = 4.0 * (t if case["reduction"] == "none" else 1)
        return {"bytes": size * times * (t + v) * d + 8.0 * t + times * loss, "flops": (6.0 if case["train"] else 2.0) * t * d * v}
    rows = case["batch"] * case["seq"]
    values = rows * (case["heads"] + case["kv_heads"])
    return {"bytes": times * 2 * size * values * case["head_dim"] + 8.0 * rows + 2.0 * case["rotary_dim"], "flops": times * 3.0 * values * case["rotary_dim"]}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "head":
        x, w, target = s["x"].double(), s["w"].double(), s["target"]
        logits = torch.mm(x, w.t())
        kept = torch.nonzero(target != _IGNORED)[:, 0]
        lse = torch.logsumexp(logits, 1)
        nll = torch.zeros_like(lse)
        nll[kept] = lse[kept] - logits[kept, target[kept]]
        share = torch.zeros_like(lse)
        share[kept] = 1.0 / kept.numel() if case["reduction"] == "mean" else 1.0
        loss = nll if case["reduction"] == "none" else (nll * share).sum()
        if not case["train"]:
            return [loss]
        p = logits.sub_(lse[:, None]).exp_()
        p[kept, target[kept]] -= 1.0
        p *= (share * s["dloss"].double())[:, None]
        return [loss, torch.mm(p, w), torch.mm(p.t(), x)]
    r, scale = case["rotary_dim"], case["scale"]
    turn = torch.polar(torch.full((), scale, dtype=torch.float64, device="cuda"), s["positions"].double()[:, :, None, None] * s["freq"].double())

    def turned(v, by):
        v = v.double().clone()
        first, second = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
        z = torch.complex(v[..., first], v[..., second]) * by   # against the direction in which angles grow
        v[..., first], v[..., second] = z.real, z.imag
        return v

    out = [turned(s["q"], turn.conj()), turned(s["k"], turn.conj())]
    return out + [turned(s["dq"], turn), turned(s["dk"], turn)] if case["train"] else out
