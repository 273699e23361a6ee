"""GPT-2-small-shaped model whose linears are random-backed, for the end-to-end step-time configuration.

Mirrors the reference's RT_* classes (modded-nanogpt/gpt_models.py:186-257: RT_norm, RT_CastedLinear,
RT_CausalSelfAttention, RT_MLP, RT_Block) with the deviations the benchmark configuration states: the four linears of a
block are qkv (d -> 3d), proj (d -> d), fc (d -> 4d) and mlp-proj (4d -> d), all in matrix-coef form with coefficient
dimension k and seeds taken in layer order from one generator (0..47 for 12 layers); attention is plain causal
scaled-dot-product attention (the reference's FlexAttention document mask needs a tracing compiler); the token embedding
and the language-model head are ordinary dense layers unless the configuration asks for the reference's random-backed ones
(modded-nanogpt/gpt_models.py:303, 310).  This file wires layers: the linears' kernels are reached through SillyLinear, but for an MLP of two
plain layers, whose squared ReLU is formed and differentiated in the kernels that store their rows (RT_MLP).  The rest of a
block (normalisation, rotary attention with a head dimension of 64, squared ReLU, the loss) is stock PyTorch, except in bf16 on the
GPU, run eagerly: chains of stock operators took 6 times what the linears' kernels take there, most of it in passes over memory
that the fused ones do not make.  Where the configuration asks for it, the loss is formed without the logits (ops.linear_cross_entropy) and positions
turn other pairs, parts of the heads or by other frequencies (ops.rotary).
"""
from dataclasses import dataclass
from typing import Generator, Optional

import torch
import torch.nn.functional as F
from torch import nn

from . import _lib, ops
from .SillyLayers import SillyEmbedding, SillyLinear


def _fused(x: torch.Tensor):
    """The extension module where ``x`` is what its kernels take, else None: bf16 on the GPU, run eagerly.  Its methods return None
    for tensors that stand for something else than their memory (under a transform or a dispatch mode)."""
    if x.dtype is torch.bfloat16 and x.is_cuda and type(x) in _PLAIN and not torch.compiler.is_compiling() and not torch.is_autocast_enabled():
        return _lib._ext or _lib.extension()
    return None


_PLAIN = (torch.Tensor, nn.Parameter)
_EPS = torch.finfo(torch.float32).eps   # F.rms_norm's default for bf16 and fp32


def _norm_kernel_takes(x: torch.Tensor) -> bool:
    return 0 < x.size(-1) <= 4096 and x.size(-1) % 4 == 0 and x.numel() > 0


def RT_norm(x: torch.Tensor) -> torch.Tensor:
    ext = _fused(x)
    y = ext.rms_norm(x, _EPS) if ext is not None and _norm_kernel_takes(x) else None
    return F.rms_norm(x, (x.size(-1),)) if y is None else y


def _add_norm(x: torch.Tensor, delta: torch.Tensor):
    """``x + delta`` and its normalisation."""
    ext = _fused(x)
    if ext is not None and delta.dtype is torch.bfloat16 and delta.shape == x.shape and _norm_kernel_takes(x):
        both = ext.add_rms_norm(x, delta, _EPS)
        if both is not None:
            return both
    x = x + delta
    return x, RT_norm(x)


class Rotary(nn.Module):
    """Rotary position embedding over (batch, time, head, head_dim), as gpt_models.py:29-49.  With any of the further arguments its layout and
    frequencies are those of :func:`ops.rotary` and :func:`ops.rotary_frequencies`, on the GPU, the frequencies fp32 whatever the module's type:
    neighbouring pairs (``interleaved``), the first ``rotary_dim`` values of a head, ``scaling`` for longer contexts."""

    stock = True   # also of a module that was stored before there was another

    def __init__(self, dim: int, base: float = 10000.0, *, interleaved: bool = False, rotary_dim: Optional[int] = None, **scaling):
        super().__init__()
        self.stock = not interleaved and rotary_dim is None and not scaling
        self.interleaved, self.scale = interleaved, 1.0
        if self.stock:
            self.register_buffer("inv_freq", (1.0 / base) ** (torch.arange(0, dim, 2) / dim), persistent=False)
        else:
            if rotary_dim is not None and not 2 <= rotary_dim <= dim:
                raise ValueError(f"Rotary: between 2 and {dim} values of a head, got {rotary_dim}")
            freq, self.scale = ops.rotary_frequencies(dim if rotary_dim is None else rotary_dim, base, **scaling)
            self.register_buffer("freq_bits", freq.view(torch.int32), persistent=False)   # as whole numbers: a module's change of type leaves them alone
            self.register_buffer("no_turn", torch.zeros(dim // 2), persistent=False)      # frequencies of what is turned already

    def both(self, q: torch.Tensor, k: Optional[torch.Tensor], positions: Optional[torch.Tensor] = None):
        """Queries and keys (or None) in one launch."""
        return ops.rotary(q, k, self.freq_bits.to(q.device).view(torch.float32), positions, interleaved=self.interleaved, scale=self.scale)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not self.stock:
            return self.both(x, None)[0]
        t = torch.arange(x.shape[1], device=x.device)
        freqs = torch.outer(t, self.inv_freq.to(x.device))
        cos, sin = freqs.cos()[None, :, None, :], freqs.sin()[None, :, None, :]
        x1, x2 = x.float().chunk(2, dim=3)
        return torch.cat((x1 * cos + x2 * sin, x2 * cos - x1 * sin), 3).type_as(x)


@dataclass
class RT_GPTConfig:
    int_dim_gen: Generator
    seed_gen: Generator
    vocab_size: int = 50304
    n_layer: int = 12
    n_head: int = 12
    n_embd: int = 768
    # True: the token embedding and the output head are random-backed too, as in the reference's model
    # (modded-nanogpt/gpt_models.py:303, 310); they then draw the first and the last (k, seed) of the generators
    random_embedding_and_head: bool = False
    # True: the loss comes from the head's input and weight (or coefficients), on the GPU, without the logits being in memory
    # (ops.linear_cross_entropy), and without their rounding to bf16
    loss_without_logits: bool = False
    # further arguments of Rotary (interleaved, rotary_dim, base, scaling, factor, ...)
    rotary: Optional[dict] = None


class RT_CastedLinear(SillyLinear):
    """Bias-free random-backed linear in matrix-coef form; the fused kernels run in the activations' dtype."""

    def __init__(self, in_features: int, out_features: int, config: RT_GPTConfig):
        k, seed = next(config.int_dim_gen), next(config.seed_gen)
        super().__init__(in_features, out_features, [k, k], [seed, seed], bias=False, matrix_coef=True)
        std = 0.02
        with torch.no_grad():   # C ~ N(0, 3*std^2/k): the weight then has standard deviation ~std
            self.weight_coef.normal_(0.0, (3.0 * std * std / k) ** 0.5)
            self.weight_scale_bias.zero_()


class RT_CausalSelfAttention(nn.Module):
    def __init__(self, dim: int, n_head: int, config: RT_GPTConfig):
        super().__init__()
        assert dim % n_head == 0
        self.n_head = n_head
        self.c_qkv = RT_CastedLinear(dim, 3 * dim, config)
        self.rotary = Rotary(dim // n_head, **(config.rotary or {}))
        self.c_proj = RT_CastedLinear(dim, dim, config)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        B, T, D = x.shape
        qkv = self.c_qkv(x)
        ext = _fused(qkv)
        stock = getattr(self.rotary, "stock", True)
        # somebody's own rotation, and one with hooks, is called with one side at a time
        both = not stock and type(self.rotary) is Rotary and Rotary.forward is _ROTARY_FORWARD and _unhooked(self.rotary)
        # q and k that turn without becoming longer may do so before they are normalised as well as behind: the kernel that normalises them then has nothing to turn
        turned = both and self.rotary.scale == 1.0
        if ext is not None and (stock or turned) and D == 64 * self.n_head and 0 < T * 3 * D < 1 << 29 and B > 0:
            if turned:
                q, k, v = qkv.split(D, 2)
                q, k = self.rotary.both(q.view(B, T, self.n_head, 64), k.view(B, T, self.n_head, 64))
                y = ext.causal_attention(torch.cat((q.view(B, T, D), k.view(B, T, D), v), 2), self.rotary.no_turn, self.n_head, _EPS)
            else:
                y = ext.causal_attention(qkv, self.rotary.inv_freq, self.n_head, _EPS)
            if y is not None:
                return self.c_proj(y)
        q, k, v = qkv.view(B, T, 3, self.n_head, D // self.n_head).unbind(2)
        q, k = RT_norm(q), RT_norm(k)
        q, k = self.rotary.both(q, k) if both else (self.rotary(q), self.rotary(k))
        y = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), is_causal=True)
        return self.c_proj(y.transpose(1, 2).reshape(B, T, D))


def _unhooked(m: nn.Module) -> bool:
    """Nothing that has to see ``m`` called: no replaced method, no compiled call, no hooks."""
    return ("forward" not in m.__dict__ and type(m).__call__ is _MODULE_CALL and m._compiled_call_impl is None and not torch.nn.modules.module._has_any_global_hook()
            and not (m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks))


def _plain_layer(m: nn.Module, x: torch.Tensor):
    """(coefficients, seed) of a layer that is its forward's product in x's dtype and nothing else, or None."""
    if not (type(m) is RT_CastedLinear and RT_CastedLinear.forward is _LINEAR_FORWARD and _unhooked(m)):
        return None
    w, coef = m._buffers.get("weight"), m._parameters.get("weight_coef")
    if w is None or coef is None or w.fused_bias or m.bias is not None or not m.fused or x.dtype != w.dtype or ops._tracing():
        return None
    return coef, w.seed


class RT_MLP(nn.Module):
    def __init__(self, dim: int, config: RT_GPTConfig):
        super().__init__()
        self.c_fc = RT_CastedLinear(dim, 4 * dim, config)
        self.c_proj = RT_CastedLinear(4 * dim, dim, config)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        y = self._in_two_nodes(x)
        if y is not None:
            return y
        h = self.c_fc(x)
        ext = _fused(h)
        if ext is None:
            return self.c_proj(F.relu(h).square())
        y = self._proj_of_relu_square(h, ext)
        if y is not None:
            return y
        a = ext.relu_square(h)
        return self.c_proj(F.relu(h).square() if a is None else a)

    def _in_two_nodes(self, x: torch.Tensor):
        """With the activation's value from c_fc's kernel and its gradient from c_proj's; None where a layer is more than its forward."""
        ext = _fused(x) if torch.is_grad_enabled() else None
        f, p = None if ext is None else _plain_layer(self.c_fc, x), self.c_proj
        if f is None:
            return None
        q = _plain_layer(p, x)
        if q is None or p.in_features != self.c_fc.out_features:
            return None
        in_f, hidden, out_f = self.c_fc.in_features, p.in_features, p.out_features
        if x.shape[-1] != in_f:
            return None
        x2 = x.reshape(-1, in_f)
        # c_proj's is the same question of as many rows
        if not (ext.takes_projected(x2, f[0], in_f, hidden, in_f, 1, None, None) and ext.takes_projected(x2, q[0], hidden, out_f, hidden, 1, None, None)):
            return None
        y = ext.squared_relu_mlp(x2, f[0], q[0], in_f, hidden, out_f, f[1], q[1])
        return None if y is None else y.reshape(*x.shape[:-1], out_f)

    def _proj_of_relu_square(self, h: torch.Tensor, ext):
        """Both in one autograd node, whose backward pass needs no pass over memory of its own for the activation; None where the layer is
        more than its forward, or h wants no gradient.  For MLPs whose c_fc is called for itself: it has a hook, a bias, another class.  Forward and backward of
        8192 tokens, 768 -> 3072 -> 768, c_fc with a hook: k = 256 189 -> 173 us, 128 172 -> 154; 1024 -> 4096 -> 1024, k = 256 254 -> 220; 2048 tokens even."""
        p = self.c_proj
        q = _plain_layer(p, h) if torch.is_grad_enabled() else None
        in_f, out_f = p.in_features, p.out_features
        if q is None or h.shape[-1] != in_f:
            return None
        x = h.reshape(-1, in_f)
        if not ext.takes_projected(x, q[0], in_f, out_f, in_f, 1, None, None):
            return None
        y = ext.relu_square_linear(x, q[0], in_f, out_f, q[1])
        return None if y is None else y.reshape(*h.shape[:-1], out_f)


class RT_Block(nn.Module):
    def __init__(self, config: RT_GPTConfig):
        super().__init__()
        self.attn = RT_CausalSelfAttention(config.n_embd, config.n_head, config)
        self.mlp = RT_MLP(config.n_embd, config)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        x, h = _add_norm(x, self.attn(RT_norm(x)))
        return x + self.mlp(h)

    def _with_norm(self, x: torch.Tensor, normed: torch.Tensor):
        """``forward`` between blocks that hand each other their output's normalisation: it and the addition are one pass over memory,
        forwards and backwards (24 additions of 7.5 us a step of GPT-2 small otherwise)."""
        x, h = _add_norm(x, self.attn(normed))
        return _add_norm(x, self.mlp(h))

    def _plain(self) -> bool:
        """Nothing that has to see ``forward`` run: no subclass, no replaced method, no compiled call, no hooks."""
        return type(self) is RT_Block and RT_Block.forward is _BLOCK_FORWARD and _unhooked(self)


# as they stand here: replaced ones are called
_BLOCK_FORWARD, _LINEAR_FORWARD, _EMBEDDING_FORWARD, _DENSE_FORWARD = RT_Block.forward, RT_CastedLinear.forward, nn.Embedding.forward, nn.Linear.forward
_ROTARY_FORWARD, _MODULE_CALL = Rotary.forward, nn.Module.__call__


def _embed(wte: nn.Module, idx: torch.Tensor) -> torch.Tensor:
    """``wte(idx)``; of a plain table with a gradient of one launch (stock, a sort of the indices and a dozen small ones)."""
    if type(wte) is nn.Embedding and nn.Embedding.forward is _EMBEDDING_FORWARD and _unhooked(wte) and torch.is_grad_enabled() and type(idx) in _PLAIN:
        w = wte._parameters.get("weight")
        if w is not None and wte.padding_idx is None and wte.max_norm is None and not (wte.scale_grad_by_freq or wte.sparse) and idx.is_cuda and not ops._tracing():
            ext = _fused(w)
            y = None if ext is None else ext.embedding(w, idx)
            if y is not None:
                return y
    return wte(idx)


class RT_GPT(nn.Module):
    """Seeds are drawn qkv, proj, fc, mlp-proj per block, block after block."""

    loss_without_logits = False

    def __init__(self, config: RT_GPTConfig):
        super().__init__()
        if config.random_embedding_and_head:
            self.wte = SillyEmbedding(config.vocab_size, config.n_embd, config.int_dim_gen, config.seed_gen)
        else:
            self.wte = nn.Embedding(config.vocab_size, config.n_embd)
        self.h = nn.ModuleList([RT_Block(config) for _ in range(config.n_layer)])
        if config.random_embedding_and_head:
            self.lm_head = RT_CastedLinear(config.n_embd, config.vocab_size, config)
        else:
            self.lm_head = nn.Linear(config.n_embd, config.vocab_size, bias=False)
        self.loss_without_logits = config.loss_without_logits
        if config.loss_without_logits and config.random_embedding_and_head:
            self.register_buffer("unit_coefs", torch.eye(self.lm_head.weight_coef.shape[1]), persistent=False)

    def _loss_without_logits(self, x: torch.Tensor, target: torch.Tensor) -> Optional[torch.Tensor]:
        """The loss of the head's input; None where the head is more than its product, not on the GPU, or of more tokens than the operator takes."""
        head = self.lm_head
        if not x.is_cuda or x.dtype not in (torch.bfloat16, torch.float32) or torch.is_autocast_enabled() or x.numel() >= 1 << 28 or target.numel() >= 1 << 21:
            return None
        if type(head) is nn.Linear and nn.Linear.forward is _DENSE_FORWARD:
            w = head._parameters.get("weight")
            if not _unhooked(head) or head.bias is not None or w is None or w.dtype != x.dtype:
                return None
            return ops.linear_cross_entropy(x.reshape(-1, x.shape[-1]), w, target.reshape(-1))
        if type(head) is not RT_CastedLinear or RT_CastedLinear.forward is not _LINEAR_FORWARD or not _unhooked(head):
            return None
        w, coef = head.weight, head.weight_coef
        if w.fused_bias or head.bias is not None or coef.dtype != x.dtype:
            return None
        # logits = z . C^T with z = x . N^T, which is what a layer with the identity's coefficients gives: the vocabulary meets k values a token
        k, d = coef.shape[1], head.in_features
        z = ops.linear(x.reshape(-1, d), self.unit_coefs, d, k, d, 1, w.seed, None, None)
        return ops.linear_cross_entropy(z, coef, target.reshape(-1))

    def forward(self, idx: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
        x = _embed(self.wte, idx)
        x = RT_norm(x.to(self.h[0].mlp.c_fc.weight_coef.dtype))
        normed = None   # RT_norm(x) where it is at hand
        for block in self.h:
            if isinstance(block, RT_Block) and block._plain():
                x, normed = block._with_norm(x, RT_norm(x) if normed is None else normed)
            else:
                x, normed = block(x), None
        normed = RT_norm(x) if normed is None else normed
        loss = self._loss_without_logits(normed, target) if self.loss_without_logits else None
        if loss is not None:
            return loss
        logits = self.lm_head(normed)
        ext = _fused(logits)
        if ext is not None and logits.size(-1) % 8 == 0 and logits.numel() and target.dtype is torch.int64:
            loss = ext.cross_entropy(logits.view(-1, logits.size(-1)), target.view(-1), -100)
            if loss is not None:
                return loss
        logits = logits.float()
        return F.cross_entropy(logits.view(-1, logits.size(-1)), target.view(-1))
