"""The operators in autograd: reverse mode of the first order. Double backward, forward mode and vmap raise."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import functional as F


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = F.layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = F.layer_norm_backward(dy, x, weight, mean, rstd, *ctx.needs_input_grad[:3], dtype=ctx.bias_dtype)
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last axis; weight and bias are float32 or of x's dtype."""
    return _LayerNorm.apply(x, weight, bias, eps)


class LayerNorm(torch.nn.Module):
    """`layer_norm` with its parameters, named as torch.nn.LayerNorm's over one axis. There is a weight always,
    and the result has x's dtype, also under autocast (where torch's is float32)."""

    def __init__(self, width: int, eps: float = 1e-5, bias: bool = True, device=None, dtype=None) -> None:
        super().__init__()
        self.width, self.eps = width, eps
        self.weight = torch.nn.Parameter(torch.ones(width, device=device, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(width, device=device, dtype=dtype)) if bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self) -> str:
        return f"{self.width}, eps={self.eps}, bias={self.bias is not None}"


class TokenScores(NamedTuple):
    """What `token_log_probs` returns; the last two are None without alternatives."""
    log_probs: torch.Tensor
    entropy: torch.Tensor
    top_log_probs: Optional[torch.Tensor]
    top_tokens: Optional[torch.Tensor]


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature, top):
        out = F.token_log_probs_forward(logits, tokens, temperature, top)
        ctx.save_for_backward(logits, tokens, out.stats, out.entropy)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        if out.top_tokens is None:
            return out.log_probs, out.entropy
        ctx.mark_non_differentiable(out.top_log_probs, out.top_tokens)
        return out.log_probs, out.entropy, out.top_log_probs, out.top_tokens

    @staticmethod
    @once_differentiable
    def backward(ctx, d_log_probs, d_entropy, *_):
        if not ctx.needs_input_grad[0] or (d_log_probs is None and d_entropy is None):
            return None, None, None, None
        logits, tokens, stats, entropy = ctx.saved_tensors
        return (F.token_log_probs_backward(d_log_probs, d_entropy, logits, tokens, stats, entropy, ctx.temperature),
                None, None, None)


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor, temperature: float = 1.0, top: int = 0) -> TokenScores:
    """Log probability of each position's token (0 for a token outside the vocabulary, such as -100)
    and entropy of softmax(logits / temperature) over the last axis, both differentiable, and the `top`
    most likely tokens with their log probabilities, which are not."""
    out = _TokenLogProbs.apply(logits, tokens, temperature, top)
    return TokenScores(*out) if len(out) == 4 else TokenScores(*out, None, None)


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_tokens, teacher_logits, temperature):
        loss, stats = F.distill_loss_forward(logits, teacher_tokens, teacher_logits, temperature)
        ctx.save_for_backward(logits, teacher_tokens, teacher_logits, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, d_loss):
        if not ctx.needs_input_grad[0]:
            return None, None, None, None
        logits, tokens, values, stats = ctx.saved_tensors
        return F.distill_loss_backward(d_loss, logits, tokens, values, stats, ctx.temperature), None, None, None


def distill_loss(logits: torch.Tensor, teacher_tokens: torch.Tensor, teacher_logits: torch.Tensor,
                 temperature: float = 1.0, reduction: str = "mean") -> torch.Tensor:
    """Distillation from a teacher's k logits per position: temperature^2 KL(q || p), q the softmax of
    the teacher's logits over its own tokens, p the student's over the vocabulary, both at the
    temperature. Tokens outside the vocabulary (such as -100) are padding. reduction: "none" (one loss
    per position), "sum", or "mean" over the positions that have a teacher. Differentiable in the
    student's logits."""
    if reduction not in ("none", "sum", "mean"):
        raise ValueError(f"LuminaV: reduction must be 'none', 'sum' or 'mean', got {reduction!r}.")
    loss = _DistillLoss.apply(logits, teacher_tokens, teacher_logits, temperature)
    if reduction == "none":
        return loss
    if reduction == "sum":
        return loss.sum()
    there = ((teacher_tokens >= 0) & (teacher_tokens < logits.shape[-1])).any(-1)
    return loss.sum() / there.sum().clamp(min=1)
