"""Attention between the tokens of packed image time series (date, row, column), beside the L-TAE classes of ltae.py, whose queries
are one learned vector per head and whose keys are the dates of one pixel.

    qkv projection [tokens, heads, d] -> HeadNormRotary (queries and keys) -> PackedAttention

Tokens of all series lie behind one another, without padding: series b owns the rows offsets[b] .. offsets[b + 1] - 1."""
import math

import torch
import torch.nn as nn

from ... import engine as E


class _HeadNormRotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, eps, plan):
        ctx.save_for_backward(q, k, wq, wk, plan.positions)       # positions too: a change in place before the backward is an error
        ctx.eps, ctx.plan = eps, plan
        return E.headnorm_rotary_forward(q, k, wq, wk, eps, plan)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        q, k, wq, wk, _ = ctx.saved_tensors
        return (*E.headnorm_rotary_backward(gq, gk, q, k, wq, wk, ctx.eps, ctx.plan), None, None)


class HeadNormRotary(nn.Module):
    """Root-mean-square norms of queries and keys for each head, with the rotation of their positions in the same pass:
    y = rotate(weight * x / sqrt(mean(x^2) + eps)), the mean over the d values of one head.

    d: head size (even, at most 256); q_weight, k_weight: fp32 parameters [d], shared by the heads.  rotary: a
    positional_encoding.RotaryAxes of the same head size, or None for the norms alone.  The sum of a head's squares is an fp32 number: values
    from 1e-18 to 1e18, or smaller ones that eps outweighs.  eps may be 0; heads of zeros are NaN then.

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
        for name, w in (("q_weight", self.q_weight), ("k_weight", self.k_weight)):
            if w.shape != (self.d,):
                raise ValueError(f"{name}: expected [{self.d}], got {tuple(w.shape)}")
        if (positions is None) != (self.rotary is None):
            raise ValueError("positions are required with a rotary, and only with one")
        E.check_tokens(q=q, k=k)
        E.check_device(q=q, q_weight=self.q_weight, k_weight=self.k_weight)
        plan = self.rotary.plan(positions, q.shape[:-2], q.device) if self.rotary is not None else E.RotaryPlan()
        rows = (q, k) if q.dim() == 3 else (q.reshape(-1, *q.shape[-2:]), k.reshape(-1, *k.shape[-2:]))
        args = (*rows, self.q_weight, self.k_weight, self.eps, plan)
        qo, ko = _HeadNormRotaryFn.apply(*args) if torch.is_grad_enabled() else E.headnorm_rotary_forward(*args)
        return (qo, ko) if q.dim() == 3 else (qo.view(q.shape), ko.view(k.shape))


class _PackedAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, off_q, off_k, k_len, temperature, causal, max_q, max_k):
        out, lse = E.packed_attention_forward(q, k, v, off_q, off_k, k_len, temperature, causal, True, None, max_q, max_k)
        ctx.save_for_backward(q, k, v, out, lse, off_q, off_k, k_len)
        ctx.args = temperature, causal, max_q, max_k
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        q, k, v, out, lse, off_q, off_k, k_len = ctx.saved_tensors
        grads = E.packed_attention_backward(dout, q, k, v, out, lse, off_q, off_k, k_len, *ctx.args)
        return (*grads, *(None,) * 7)


def pack_offsets(lengths, device):
    """[B] sequence lengths (Python numbers) -> [B + 1] int32 row offsets on the device"""
    offsets = [0]
    for n in lengths:
        if n < 0:
            raise ValueError(f"length {n}: must not be negative")
        offsets.append(offsets[-1] + int(n))
    return torch.tensor(offsets, dtype=torch.int32, device=device)


class PackedAttention(nn.Module):
    """softmax(q k^T / temperature) v within each sequence of a packed batch, heads in groups.

    causal: row i of a sequence's Lq queries sees its keys j <= i + Lk - Lq (the last query sees every key), otherwise all Lk.
    temperature: default sqrt(d), as in the L-TAE classes.

    forward(q [Nq, heads, d], k [Nk, kv_heads, d], v [Nk, kv_heads, d], offsets_q, offsets_k=None, k_len=None, ...) -> out [Nq, heads, d]
      heads is a multiple of kv_heads: query head i reads key head i // (heads // kv_heads).  d is at most 128.  fp32 or bf16; the softmax and
      all sums are fp32 either way.  With bf16 the probabilities, and in the backward pass dS, are rounded to bf16 before they are multiplied by
      values, keys, queries or incoming gradients: gradients are off by about 1.5 times what the rounding of the result alone would leave (heads of
      4 values: twice).  Scores q k / temperature are fp32 numbers, rounded by 2^-24 of their size, and so is the logarithm that gradients
      take their probabilities from: scores of 2^20 leave gradients with one digit, and from 2^30 on a row may not be finite.
      Inputs may be strided (slices of one projection, a cache of any layout with d contiguous).
      offsets_q, offsets_k [B + 1]: int32 on the device, not decreasing; sequence b owns rows offsets[b] .. offsets[b + 1] - 1 (`pack_offsets`).
      Without offsets_k the keys lie like the queries.  They are not read on the host; offsets outside the tensors are clamped on the device.
      Up to 2^30 keys, and 2^30 query rows times heads per key head.
      k_len [B]: int32, used rows of each key sequence; the rest is room in a cache, never read into a result.
      A row that sees no key is 0 and takes no part in any gradient.  Rows of no sequence are zeros, in the gradients too.  Keys and values
      that a row does not see may hold anything, infinities and NaN included (gradients want all of a sequence's own rows finite).  What a row
      that sees an infinity holds is not defined: most often it is not finite; where its only trace is a score of -infinity it may be what the
      other keys make it, or 0 like a row that sees nothing.  A row that sees NaN in a key is NaN, in a value NaN at its place.
      max_q, max_k: the longest sequences as far as the program knows them; they choose among the kernels (few rows per sequence over a cache,
      short sequences) and change nothing else: a wrong one costs time.
      out: contiguous, written in place of a new tensor (only without gradients); rows of no sequence stay as they were.  No input may reach into
      its memory, from an input's first value to its last one.  Where d is a multiple of 4 it starts at a multiple of 4 values.
      return_lse: also the logarithm of each row's sum of exponentials [Nq, heads], fp32, without a gradient; -inf where a row sees nothing.

    Serving: one query row per sequence (offsets_q = 0, 1, 2, ...) against a cache [B * room, kv_heads, d] with offsets_k = b * room and k_len."""

    def __init__(self, causal=False, temperature=None):
        super().__init__()
        if temperature is not None and not 1e-30 <= temperature <= 1e30:
            raise ValueError(f"temperature {temperature}: must be positive, from 1e-30 to 1e30")
        self.causal, self.temperature = bool(causal), temperature

    def forward(self, q, k, v, offsets_q, offsets_k=None, k_len=None, max_q=None, max_k=None, out=None, return_lse=False):
        if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
            raise ValueError(f"expected tokens [N, heads, d], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
        if k.shape != v.shape or q.shape[2] != k.shape[2]:
            raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
        d, heads, kv_heads = q.shape[2], q.shape[1], k.shape[1]
        if d == 0 or d > 128:
            raise ValueError(f"head size {d}: 1 to 128 are built")
        if kv_heads == 0 or heads == 0 or heads % kv_heads:
            raise ValueError(f"{heads} query heads are not a multiple of {kv_heads} key heads")
        if offsets_k is None:
            if q.shape[0] != k.shape[0]:
                raise ValueError(f"{q.shape[0]} query rows and {k.shape[0]} key rows need offsets_k")
            offsets_k = offsets_q
            max_k = max_q if max_k is None else max_k
        for name, t in (("offsets_q", offsets_q), ("offsets_k", offsets_k), ("k_len", k_len)):
            if t is None:
                continue
            if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
                raise ValueError(f"{name}: a contiguous int32 vector is required, got {t.dtype} {tuple(t.shape)}")
        n = offsets_q.numel() - 1
        if n < 1 or offsets_k.numel() != n + 1 or (k_len is not None and k_len.numel() != n):
            raise ValueError("offsets_q and offsets_k need B + 1 entries, k_len B, with at least one sequence")
        for name, m in (("max_q", max_q), ("max_k", max_k)):
            if m is not None and m < 0:
                raise ValueError(f"{name} {m}: must not be negative")
        E.check_tokens(q=q, k=k, v=v)
        E.check_device(q=q, offsets_q=offsets_q, offsets_k=offsets_k, k_len=k_len)
        hints = min(int(max_q or 0), q.shape[0]), min(int(max_k or 0), k.shape[0])
        temperature = math.sqrt(d) if self.temperature is None else float(self.temperature)
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
            if out is not None:
                raise ValueError("out is for calls without gradients")
            res, lse = _PackedAttentionFn.apply(q, k, v, offsets_q, offsets_k, k_len, temperature, self.causal, *hints)
        else:
            if out is not None:
                E.check_tokens(q=q, out=out)
                if out.shape != q.shape or not out.is_contiguous():
                    raise ValueError(f"out {tuple(out.shape)}: a contiguous tensor of q's shape {tuple(q.shape)} is required")
                if out.requires_grad:
                    raise ValueError("out is for calls without gradients: it requires one")
                first, behind = E.extent(out)
                for t in (q, k, v, offsets_q, offsets_k, k_len):
                    if t is not None and E.extent(t)[0] < behind and first < E.extent(t)[1]:
                        raise ValueError("out shares memory with an input")
            res, lse = E.packed_attention_forward(q, k, v, offsets_q, offsets_k, k_len, temperature, self.causal, return_lse, out, *hints)
            if out is not None:
                torch.autograd.graph.increment_version(out)         # a graph that saved it has to notice
        return (res, lse) if return_lse else res
