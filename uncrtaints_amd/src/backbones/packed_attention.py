"""Attention between the tokens of packed image time series (date, row, column), beside the L-TAE classes of ltae.py, whose queries
are one learned vector per head and whose keys are the dates of one pixel.

    qkv projection [tokens, heads, d] -> HeadNormRotary (queries and keys) -> PackedAttention

Tokens of all series lie behind one another, without padding: series b owns the rows offsets[b] .. offsets[b + 1] - 1."""
import torch
import torch.nn as nn

from ... import engine as E


class _HeadNormRotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, eps, plan):
        ctx.save_for_backward(q, k, wq, wk)
        ctx.eps, ctx.plan = eps, plan
        return E.headnorm_rotary_forward(q, k, wq, wk, eps, plan)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        q, k, wq, wk = ctx.saved_tensors
        return (*E.headnorm_rotary_backward(gq, gk, q, k, wq, wk, ctx.eps, ctx.plan), None, None)


class HeadNormRotary(nn.Module):
    """Root-mean-square norms of queries and keys for each head, with the rotation of their positions in the same pass:
    y = rotate(weight * x / sqrt(mean(x^2) + eps)), the mean over the d values of one head.

    d: head size (even, at most 256); q_weight, k_weight: fp32 parameters [d], shared by the heads.  rotary: a
    positional_encoding.RotaryAxes of the same head size, or None for the norms alone.

    forward(q [..., heads, d], k [..., kv_heads, d], positions [..., axes]) -> (q, k), contiguous, in the inputs' storage type."""

    def __init__(self, d, rotary=None, eps=1e-6):
        super().__init__()
        if d <= 0 or d % 2 or d > 256:
            raise ValueError(f"head size {d}: an even size up to 256 is required")
        if rotary is not None and rotary.d != d:
            raise ValueError(f"rotary turns heads of size {rotary.d}, not {d}")
        if not eps >= 0.0:
            raise ValueError(f"eps {eps}: must not be negative")
        self.d, self.eps, self.rotary = d, float(eps), rotary
        self.q_weight = nn.Parameter(torch.ones(d))
        self.k_weight = nn.Parameter(torch.ones(d))

    def forward(self, q, k, positions=None):
        for name, t in (("q", q), ("k", k)):
            if t.dim() < 2 or t.shape[-1] != self.d or t.shape[-2] == 0:
                raise ValueError(f"{name}: expected tokens [..., heads, {self.d}], got {tuple(t.shape)}")
        if q.shape[:-2] != k.shape[:-2]:
            raise ValueError(f"q has tokens {tuple(q.shape[:-2])}, k {tuple(k.shape[:-2])}")
        if self.q_weight.dtype != torch.float32 or self.k_weight.dtype != torch.float32:
            raise RuntimeError("the norms' weights stay float32 (activations may be bfloat16)")
        if (positions is None) != (self.rotary is None):
            raise ValueError("positions are required with a rotary, and only with one")
        E.check_tokens(q=q, k=k)
        E.check_device(q=q, q_weight=self.q_weight, k_weight=self.k_weight)
        plan = self.rotary.plan(positions, q.shape[:-2], q.device) if self.rotary is not None else E.RotaryPlan()
        qo, ko = _HeadNormRotaryFn.apply(q.reshape(-1, *q.shape[-2:]), k.reshape(-1, *k.shape[-2:]), self.q_weight, self.k_weight,
                                         self.eps, plan)
        return qo.view(q.shape), ko.view(k.shape)
