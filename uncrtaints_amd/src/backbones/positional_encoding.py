"""PositionalEncoder with the reference's surface (model/src/backbones/positional_encoding.py:5-31).

Only the denominators are computed here (once, on the host, exactly as the reference __init__ does);
the sin/cos table itself is produced inside the L-TAE position-bias HIP kernel (csrc/ltae.hip)."""
import math

import torch
import torch.nn as nn


class PositionalEncoder(nn.Module):
    def __init__(self, d, T=1000, repeat=None, offset=0):
        super().__init__()
        self.d = d
        self.T = T
        self.repeat = repeat
        self.denom = torch.pow(T, 2 * (torch.arange(offset, offset + d).float() // 2) / d)
        self.updated_location = False

    def denom_on(self, device):
        if self.denom.device != device:
            self.denom = self.denom.to(device)
            self.updated_location = True
        return self.denom

    def forward(self, batch_positions):
        """[B,T] -> [B,T,d*repeat] sinusoid table (HIP kernel; bias-free call of the position-bias op)."""
        from ... import engine as E
        from ... import hip_backend as hb
        B, T = batch_positions.shape
        D = self.d * (self.repeat or 1)
        out = torch.empty((B * T, D), device=batch_positions.device, dtype=torch.float32)
        hb.call("uncr_ltae_posbias", batch_positions.reshape(-1).contiguous().float(),
                self.denom_on(batch_positions.device), self.d, None, out, B * T, D, 1, E._stream())
        return out.view(B, T, D)


class _RotaryFn(torch.autograd.Function):
    """The rotation by an orthogonal matrix per token: its gradient is the rotation back."""

    @staticmethod
    def forward(ctx, x, plan):
        from ... import engine as E
        ctx.plan = plan
        ctx.save_for_backward(plan.positions)       # so that a change in place before the backward is an error
        return E.rotary_axes(x, plan)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        from ... import engine as E
        _ = ctx.saved_tensors
        return E.rotary_axes(dy, ctx.plan, inverse=True), None


class RotaryAxes(nn.Module):
    """Rotary positions with several axes: the counterpart of PositionalEncoder for attention between TOKENS (date, row, column) instead of
    between the dates of one pixel.  Each axis owns a section of every head vector, and the pair i of a section of size n is turned by
    `position * T ** (-2 i / n)` radians, so that the product of a query and a key depends on their distance along every axis.

    d: head size (even, at most 256).  sections: elements per axis (even; at most four axes; elements behind the last one pass through);
    default: one axis over the whole head.  T: the longest period / 2 pi, one number or one per axis.
    pairs: "halves" turns (i, i + n/2) of a section, "neighbours" (2i, 2i + 1).

    forward(x [..., heads, d], positions [..., axes]) -> the rotated tensor, contiguous, in x's storage type (fp32 or bf16).  positions:
    int32, int64, fp32 or fp64; they carry no gradient.  Angles are made and reduced in 64 bits: off by about 2^-52 of their value, no more than
    fp32's own rounding up to 2^28 radians, 1e-3 at 2^42.  There is no forward-mode derivative (a tensor with a tangent is refused)."""

    def __init__(self, d, sections=None, T=10000.0, pairs="halves"):
        super().__init__()
        sections = (d,) if sections is None else tuple(int(n) for n in sections)
        if d <= 0 or d % 2 or d > 256:
            raise ValueError(f"head size {d}: an even size up to 256 is required")
        if not 1 <= len(sections) <= 4 or any(n <= 0 or n % 2 for n in sections) or sum(sections) > d:
            raise ValueError(f"sections {sections}: one to four even sizes with a sum of at most {d}")
        if pairs not in ("halves", "neighbours"):
            raise ValueError(f"pairs {pairs!r}: 'halves' or 'neighbours'")
        bases = tuple(float(t) for t in T) if isinstance(T, (tuple, list)) else (float(T),) * len(sections)
        if len(bases) != len(sections) or any(not t > 0.0 for t in bases):
            raise ValueError(f"T {T}: one positive number, or one per axis")
        self.d, self.sections, self.T, self.pairs = d, sections, bases, pairs
        turns = torch.zeros(d // 2, dtype=torch.float64)
        at = 0
        for n, base in zip(sections, bases):
            i = torch.arange(n // 2, dtype=torch.float64)
            turns[at:at + n // 2] = torch.pow(torch.tensor(base, dtype=torch.float64), -2.0 * i / n) / (2.0 * math.pi)
            at += n // 2
        # held as its bits: a cast of the module to another floating type leaves 64-bit turns as they are
        self.register_buffer("turns_bits", turns.view(torch.int64), persistent=False)

    def plan(self, positions, lead, device):
        """Checks positions [..., axes] against the tensor's leading shape -> engine.RotaryPlan"""
        from ... import engine as E
        if positions.dtype not in E._POS_DT:
            raise RuntimeError(f"positions: unsupported dtype {positions.dtype} (int32, int64, float32 or float64)")
        if positions.shape != (*lead, len(self.sections)):
            raise ValueError(f"positions {tuple(positions.shape)}: expected {(*lead, len(self.sections))}")
        if positions.requires_grad:
            raise ValueError("positions carry no gradient: detach them")
        E.check_device(positions=positions, rotary=self.turns_bits)
        if positions.device != device:
            raise RuntimeError(f"positions are on {positions.device}, the tokens on {device}")
        return E.RotaryPlan(positions.contiguous(), self.sections, self.turns_bits,
                            self.pairs == "neighbours")

    def forward(self, x, positions):
        from ... import engine as E
        shape = x.shape
        if len(shape) < 2 or shape[-1] != self.d or shape[-2] == 0:
            raise ValueError(f"expected tokens [..., heads, {self.d}], got {tuple(shape)}")
        E.check_tokens(x=x)
        plan = self.plan(positions, shape[:-2], x.device)
        rows = x if len(shape) == 3 else x.reshape(-1, *shape[-2:])
        y = _RotaryFn.apply(rows, plan) if x.requires_grad and torch.is_grad_enabled() else E.rotary_axes(rows, plan)
        return y if len(shape) == 3 else y.view(shape)
