"""Llama-style decoder: RMSNorm, rotary position embedding, SwiGLU feed-forward, untied output
head.  Defaults are the 1B configuration of the benchmarks: 16 layers, d_model 2048, 32 heads,
FFN 8192, vocabulary 32000.

With ``fused=True`` (default) RMSNorm and the head + cross-entropy go through
``optimizers_b200.models.fused_ops``.  ``fused_embedding`` takes the token embedding from there too.
``fp8`` runs the seven linear layers of a block on 8-bit operands (``optimizers_b200.models.fp8``) and joins every residual
addition with the RMSNorm behind it; without gradients the norms hand their rows over in 8 bits, and
``hold_fp8_weights()`` keeps the weights in 8 bits between calls."""

from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from optimizers_b200.models import fp8, fused_ops
from optimizers_b200.utils.kept import Kept


@dataclass
class LlamaConfig:
    vocab_size: int = 32000
    n_layer: int = 16
    n_head: int = 32
    d_model: int = 2048
    d_ffn: int = 8192
    max_seq: int = 2048
    rope_theta: float = 10000.0
    norm_eps: float = 1e-5
    fused: bool = True
    fused_embedding: bool = False
    fp8: bool = False


class RMSNorm(nn.Module):
    def __init__(self, dim: int, eps: float, fused: bool = True) -> None:
        super().__init__()
        self.eps = eps
        self.fused = fused
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x: torch.Tensor, branch: torch.Tensor | None = None, joined: bool = False):
        """The norm of x, or of ``x + branch``; with ``joined`` a pair of it and the sum, in 8 bits where no gradient is wanted."""
        if joined:
            return _norm_of_sum(branch, x, self)
        if branch is not None:
            return fused_ops.add_rms_norm(branch, x, self.weight, self.eps)[0]
        if self.fused:
            return fused_ops.rms_norm(x, self.weight, self.eps)
        scale = torch.rsqrt(x.float().pow(2).mean(-1, keepdim=True) + self.eps)
        return (x.float() * scale).to(x.dtype) * self.weight


def _rope_tables(seq: int, head_dim: int, theta: float, device: torch.device) -> tuple[torch.Tensor, torch.Tensor]:
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, device=device).float() / head_dim))
    angles = torch.outer(torch.arange(seq, device=device).float(), inv)
    return angles.cos(), angles.sin()


def _apply_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    a, b = x[..., 0::2], x[..., 1::2]
    out = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1)
    return out.flatten(-2).to(x.dtype)


class _Layer(nn.Module):
    def __init__(self, cfg: LlamaConfig) -> None:
        super().__init__()
        self.n_head = cfg.n_head
        self.attn_norm = RMSNorm(cfg.d_model, cfg.norm_eps, cfg.fused)
        self.wq = nn.Linear(cfg.d_model, cfg.d_model, bias=False)
        self.wk = nn.Linear(cfg.d_model, cfg.d_model, bias=False)
        self.wv = nn.Linear(cfg.d_model, cfg.d_model, bias=False)
        self.wo = nn.Linear(cfg.d_model, cfg.d_model, bias=False)
        self.ffn_norm = RMSNorm(cfg.d_model, cfg.norm_eps, cfg.fused)
        self.w_gate = nn.Linear(cfg.d_model, cfg.d_ffn, bias=False)
        self.w_up = nn.Linear(cfg.d_model, cfg.d_ffn, bias=False)
        self.w_down = nn.Linear(cfg.d_ffn, cfg.d_model, bias=False)

    def forward(self, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, branch: torch.Tensor | None = None, fp8: bool = False):
        if fp8:
            return self.forward_fp8(branch, x, cos, sin)
        B, T, C = x.shape
        h = self.attn_norm(x)
        shape = (B, T, self.n_head, C // self.n_head)
        q = _apply_rope(self.wq(h).view(shape).transpose(1, 2), cos, sin)
        k = _apply_rope(self.wk(h).view(shape).transpose(1, 2), cos, sin)
        v = self.wv(h).view(shape).transpose(1, 2)
        a = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        x = x + self.wo(a.transpose(1, 2).reshape(B, T, C))
        h = self.ffn_norm(x)
        return x + self.w_down(F.silu(self.w_gate(h)) * self.w_up(h))

    _LINEARS = ("wq", "wk", "wv", "wo", "w_gate", "w_up", "w_down")

    def _fp8(self, x, out_dtype: torch.dtype, *names: str):
        held = None if torch.is_grad_enabled() else getattr(self, "_held", None)
        return fp8.linear(x, tuple(getattr(self, n).weight if held is None else self._current(n) for n in names), out_dtype)

    def _current(self, name: str) -> torch.Tensor | fp8.Weight:
        """The kept copy of a weight, or the weight itself if it has changed since."""
        weight, kept = getattr(self, name).weight, self._held.get(name)
        if kept is not None and kept.of(weight):
            return kept.value
        self._held.pop(name, None)
        return weight

    def forward_fp8(self, branch: torch.Tensor | None, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor):
        """The block on 8-bit products: takes and returns the last branch's output and the stream that it is still to be added to.  (The
        linear layers are read, not called: several share one conversion, so hooks of theirs do not run; the block's and the norms' do.)"""
        B, T, C = x.shape
        dtype = fused_ops._compute_dtype(x)
        h, x = self.attn_norm(x, branch, joined=True)
        shape = (B, T, self.n_head, C // self.n_head)
        q, k, v = (t.view(shape).transpose(1, 2) for t in self._fp8(h, dtype, "wq", "wk", "wv"))
        a = F.scaled_dot_product_attention(_apply_rope(q, cos, sin), _apply_rope(k, cos, sin), v, is_causal=True)
        (branch,) = self._fp8(a.transpose(1, 2).reshape(B, T, C), dtype, "wo")
        h, x = self.ffn_norm(x, branch.view(x.shape), joined=True)
        gate, up = self._fp8(h, dtype, "w_gate", "w_up")
        (branch,) = self._fp8(F.silu(gate) * up, dtype, "w_down")
        return branch.view(x.shape), x


def _norm_of_sum(branch: torch.Tensor | None, x: torch.Tensor, norm: RMSNorm):
    """``x + branch`` and its RMSNorm: ``(normalised, sum)``; the normalised rows come in 8 bits where no gradient is wanted."""
    if not torch.is_grad_enabled():
        return fp8.add_rms_norm(x, None, norm.weight, norm.eps) if branch is None else fp8.add_rms_norm(branch, x, norm.weight, norm.eps)
    if branch is None:
        return fused_ops.rms_norm(x, norm.weight, norm.eps), x
    return fused_ops.add_rms_norm(branch, x, norm.weight, norm.eps)


class Llama(nn.Module):
    def __init__(self, cfg: LlamaConfig | None = None) -> None:
        super().__init__()
        self.cfg = cfg = cfg or LlamaConfig()
        self.embed = fused_ops.TokenEmbedding(cfg.vocab_size, cfg.d_model)
        self.layers = nn.ModuleList(_Layer(cfg) for _ in range(cfg.n_layer))
        self.norm = RMSNorm(cfg.d_model, cfg.norm_eps, cfg.fused)
        self.head = nn.Linear(cfg.d_model, cfg.vocab_size, bias=False)
        for m in self.modules():
            if isinstance(m, (nn.Linear, nn.Embedding)):
                nn.init.normal_(m.weight, mean=0.0, std=0.02)

    def hold_fp8_weights(self) -> None:
        """Keep the blocks' weights in 8 bits for calls without gradients, until ``train()``.  A weight that changes meanwhile is converted in every
        call again, until the next call of this; changes that PyTorch does not count need that call (``utils/kept.py`` says which), and a
        captured graph keeps what it was captured with."""
        if not self.cfg.fp8:
            raise ValueError("hold_fp8_weights needs a model with fp8=True")
        held = []
        for layer in self.layers:
            weights = {n: getattr(layer, n).weight for n in layer._LINEARS}
            if any(type(w) not in (torch.Tensor, nn.Parameter) or w.dim() != 2 for w in weights.values()):
                raise ValueError("hold_fp8_weights needs whole weights; shards are converted in every call")
            held.append({n: Kept(w, fp8.quantize_weight(w)) for n, w in weights.items()})
        for layer, kept in zip(self.layers, held):
            layer._held = kept

    def train(self, mode: bool = True):
        if mode:
            for layer in self.layers:
                layer._held = None
        return super().train(mode)

    def forward(self, idx: torch.Tensor, targets: torch.Tensor | None = None):
        T = idx.shape[1]
        cos, sin = _rope_tables(T, self.cfg.d_model // self.cfg.n_head, self.cfg.rope_theta, idx.device)
        x = fused_ops.embed(self.embed, idx) if self.cfg.fused_embedding else self.embed(idx)
        if self.cfg.fp8:
            branch = None
            for layer in self.layers:
                branch, x = layer(x, cos, sin, branch, fp8=True)
            h = self.norm(x) if branch is None else self.norm(x, branch)
        else:
            for layer in self.layers:
                x = layer(x, cos, sin)
            h = self.norm(x)
        if self.cfg.fused and targets is not None:
            return fused_ops.lm_head_cross_entropy(h, self.head.weight, targets)
        logits = self.head(h)
        if targets is None:
            return logits
        return F.cross_entropy(logits.view(-1, logits.size(-1)).float(), targets.reshape(-1))
