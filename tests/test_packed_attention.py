"""Attention over packed sequences (packed_attention.PackedAttention) against softmax(q k^T / temperature) v in 64 bits, sequence by sequence.

Tolerances, fixed before the first run; u = 2^-24 (fp32 half step), h = finfo(storage).eps / 2 (a rounding to the storage type), r = h for bf16
storage and 0 for fp32 (there the probabilities are rounded to bf16 before they are multiplied), n = number of keys (rows) summed:
  score      a dot product of d terms in fp32, the scale, the exponent's argument:  e = (d + 8) u max_j sum|q k_j| / temperature
  p          relative: e_p = 2 e + (n + 32) u + 2 u |lse|       (its own score, the reference's, the sum of n terms, exp2 and log2)
  out        (e_p + r + n u) sum p |v| + h |out|
  lse        e + (n + 32) u + 2 u |lse|
  dS         p (e_p |dP - delta| + (d + 8) u sum|dO v| + e_delta) + r |dS|,   e_delta = sum |dO| (error of out) + (d + 8) u sum |dO out|
  dQ, dK     the sum over dS' error times |k| (|q|), n u of the absolute sum, + h |result|;   dV = p^T dO alike with p (e_p + r + n u)
  underflow  a probability, and a dS, below the smallest normal number 2^-126 may be flushed to 0: an absolute error of at most 2^-126 in each
             p and of 2^-126 (|dP - delta| + 1) in each dS, through the same sums.  (Scores of several hundred leave such probabilities, and
             their exact gradients of 1e-37 are in range: seen with test_large_scores_and_a_temperature.)"""
import math

import pytest
import torch

U = 2.0 ** -24
DEV = "cuda"
gpu = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def reference(q, k, v, do, causal, temperature, dtype):
    """One sequence and one group: q [G, Lq, D], k / v [Lk, D] in fp64 -> dict of (value, bound)"""
    G, lq, d = q.shape
    lk = k.shape[0]
    h = torch.finfo(dtype).eps / 2
    r = h if dtype == torch.bfloat16 else 0.0
    if lk == 0 or lq == 0:
        z, zk = torch.zeros_like(q), torch.zeros_like(k)
        return dict(out=(z, z), lse=(torch.full((G, lq), -math.inf, dtype=torch.float64), z[..., 0]), dq=(z, z), dk=(zk, zk), dv=(zk, zk))
    s = q @ k.T / temperature
    see = torch.ones(lq, lk, dtype=torch.bool)
    if causal:
        see = torch.arange(lk)[None] <= torch.arange(lq)[:, None] + (lk - lq)
    none = ~see.any(1)
    lse = torch.logsumexp(s.masked_fill(~see, -math.inf), -1)
    p = torch.exp(s - lse.masked_fill(none, 0.0)[..., None]).masked_fill(~see, 0.0)
    out = p @ v
    e = (d + 8) * U * ((q.abs() @ k.abs().T / temperature).masked_fill(~see, 0.0)).amax(-1)
    base = lse.masked_fill(none, 0.0).abs()
    ep = 2 * e + (lk + 32) * U + 2 * U * base
    flush = 2.0 ** -126 * see.double()
    b_out = (ep + r + lk * U)[..., None] * (p @ v.abs()) + h * out.abs() + flush @ v.abs()
    res = dict(out=(out, b_out), lse=(lse, e + (lk + 32) * U + 2 * U * base))
    dp = do @ v.T
    delta = (do * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_delta = (do.abs() * b_out).sum(-1, keepdim=True) + (d + 8) * U * (do * out).abs().sum(-1, keepdim=True)
    e_ds = p * (ep[..., None] * (dp - delta).abs() + (d + 8) * U * (do.abs() @ v.abs().T) + e_delta) + r * ds.abs() + flush * ((dp - delta).abs() + 1)
    dq = ds @ k / temperature
    res["dq"] = (dq, (e_ds @ k.abs() + lk * U * (ds.abs() @ k.abs())) / temperature + (h + 2 * U) * dq.abs())
    n = G * lq
    dk = (ds.transpose(1, 2) @ q).sum(0) / temperature
    res["dk"] = (dk, ((e_ds.transpose(1, 2) @ q.abs()).sum(0) + n * U * (ds.abs().transpose(1, 2) @ q.abs()).sum(0)) / temperature
                 + (h + 2 * U) * dk.abs())
    dv = (p.transpose(1, 2) @ do).sum(0)
    res["dv"] = (dv, ((p * (ep + r + n * U)[..., None] + flush).transpose(1, 2) @ do.abs()).sum(0) + (h + 2 * U) * dv.abs())
    return res


def _check(name, got, ref, bound):
    got, tiny = got.detach().cpu().double(), 2.0 ** -126
    bad = ~((got - ref).abs() <= bound + tiny) & ~((got == ref) & torch.isinf(ref))
    assert not bad.any(), (name, int(bad.sum()), bad.numel(), bad.nonzero()[0].tolist(), float(got[bad][0]), float(ref[bad][0]), float(bound[bad][0]))


def _offsets(lengths, front=0):
    return torch.tensor([front] + [front + sum(lengths[:i + 1]) for i in range(len(lengths))], dtype=torch.int32)


def _run(lq, lk, hq, hk, d, causal, dtype, room=None, front=0, behind=0, temperature=None, train=True, scale=1.0, layout="plain", seed=0, hints=True):
    """lq, lk: lengths; room: rows each key sequence owns (>= lk, or None); front / behind: rows of no sequence.  Everything outside is NaN."""
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention
    own = room if room is not None else lk
    off_q, off_k = _offsets(lq, front), _offsets(own, front)
    nq, nk = int(off_q[-1]) + behind, int(off_k[-1]) + behind
    g = _gen(seed)
    q, k, v, do = (torch.randn(n, heads, d, generator=g) for n, heads in ((nq, hq), (nk, hk), (nk, hk), (nq, hq)))
    q *= scale
    used_q, used_k = torch.zeros(nq, dtype=torch.bool), torch.zeros(nk, dtype=torch.bool)
    for b in range(len(lq)):
        used_q[off_q[b]:off_q[b] + lq[b]] = True
        used_k[off_k[b]:off_k[b] + lk[b]] = True
    q[~used_q], do[~used_q], k[~used_k], v[~used_k] = math.nan, math.nan, math.nan, math.nan
    q, k, v, do = (t.to(dtype) for t in (q, k, v, do))

    def place(t):
        if layout == "heads_first":
            return t.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
        if layout == "odd_start":
            z = torch.empty(t.shape[0], t.shape[1] * d + 3, dtype=dtype, device=DEV)
            z[:, 1:1 + t.shape[1] * d] = t.to(DEV).flatten(1)
            return z[:, 1:1 + t.shape[1] * d].unflatten(1, (t.shape[1], d))
        if layout == "fused":
            z = torch.full((t.shape[0], t.shape[1] + 2, d), math.nan, dtype=dtype, device=DEV)
            z[:, 1:-1] = t.to(DEV)
            return z[:, 1:-1]
        if layout == "last_strided":
            z = torch.empty(t.shape[0], t.shape[1], 2 * d, dtype=dtype, device=DEV)
            z[..., ::2] = t.to(DEV)
            return z[..., ::2]
        return t.to(DEV)

    m = PackedAttention(causal=causal, temperature=temperature)
    temp = temperature if temperature is not None else math.sqrt(d)
    qd, kd, vd = (place(t).detach().requires_grad_(train) for t in (q, k, v))
    k_len = torch.tensor(lk, dtype=torch.int32, device=DEV) if room is not None else None
    hint = {} if not hints else dict(max_q=max(lq), max_k=max(lk)) if hints is True else dict(max_q=hints[0], max_k=hints[1])
    out, lse = m(qd, kd, vd, off_q.to(DEV), off_k.to(DEV), k_len=k_len, return_lse=True, **hint)
    grads = torch.autograd.grad(out, (qd, kd, vd), place(do)) if train else ()
    want = {n: (torch.zeros(*sh, dtype=torch.float64), torch.zeros(*sh, dtype=torch.float64))
            for n, sh in dict(out=q.shape, dq=q.shape, dk=k.shape, dv=k.shape, lse=(nq, hq)).items()}
    want["lse"][0].fill_(-math.inf)
    G = hq // hk
    for b in range(len(lq)):
        rq, rk = slice(int(off_q[b]), int(off_q[b]) + lq[b]), slice(int(off_k[b]), int(off_k[b]) + lk[b])
        for c in range(hk):
            hs = slice(c * G, (c + 1) * G)
            ref = reference(q[rq, hs].double().transpose(0, 1), k[rk, c].double(), v[rk, c].double(), do[rq, hs].double().transpose(0, 1), causal,
                            temp, dtype)
            for i in (0, 1):
                want["out"][i][rq, hs], want["dq"][i][rq, hs] = ref["out"][i].transpose(0, 1), ref["dq"][i].transpose(0, 1)
                want["lse"][i][rq, hs] = ref["lse"][i].T
                want["dk"][i][rk, c], want["dv"][i][rk, c] = ref["dk"][i], ref["dv"][i]
    assert out.dtype == dtype and lse.dtype == torch.float32 and not lse.requires_grad
    _check("lse", lse, *want["lse"])
    _check("out", out, *want["out"])
    for name, t in zip(("dq", "dk", "dv"), grads):
        assert t.dtype == dtype
        _check(name, t, *want[name])
    return out


BOTH = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
MASK = pytest.mark.parametrize("causal", [False, True])


@gpu
@MASK
@BOTH
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257])
def test_one_sequence_lengths(n, dtype, causal):
    _run([n], [n], 2, 1, 32, causal, dtype)


@gpu
@MASK
@BOTH
@pytest.mark.parametrize("d", [1, 3, 4, 8, 16, 20, 33, 40, 64, 72, 96, 100, 128])
def test_head_sizes(d, dtype, causal):
    _run([70, 3, 131], [70, 3, 131], 4, 2, d, causal, dtype, seed=d)


@gpu
@MASK
@BOTH
@pytest.mark.parametrize("hq,hk", [(1, 1), (3, 1), (6, 2), (8, 8), (16, 2), (35, 5), (40, 1)])
def test_head_groups(hq, hk, dtype, causal):
    _run([45, 0, 7, 100], [45, 0, 7, 100], hq, hk, 64, causal, dtype, seed=hq)


@gpu
@MASK
@BOTH
def test_lengths_that_differ_between_queries_and_keys(dtype, causal):
    """More keys than queries (a cache), fewer (the first rows see nothing under the causal mask), none on either side."""
    _run([5, 40, 33, 0, 9, 70], [200, 10, 33, 8, 0, 65], 6, 3, 64, causal, dtype)


@gpu
@MASK
@BOTH
@pytest.mark.parametrize("d", [16, 128])
def test_rows_of_no_sequence_and_room_in_the_cache_are_never_read(d, dtype, causal):
    """NaN in front of, behind and between the sequences' used rows leaves no trace, in the gradients either."""
    _run([12, 1, 90], [50, 0, 77], 4, 2, d, causal, dtype, room=[64, 5, 80], front=3, behind=37)


@gpu
@BOTH
@pytest.mark.parametrize("layout", ["fused", "heads_first", "odd_start", "last_strided"])
@pytest.mark.parametrize("d", [32, 128])
def test_layouts(layout, d, dtype):
    _run([33, 80], [33, 80], 4, 2, d, True, dtype, layout=layout)


@gpu
@MASK
@BOTH
@pytest.mark.parametrize("batch", [64, 65, 700, 5000])
def test_many_short_sequences(batch, dtype, causal):
    lengths = torch.randint(0, 5, (batch,), generator=_gen(batch)).tolist()
    _run(lengths, lengths, 2, 1, 16, causal, dtype)


@gpu
@MASK
@BOTH
@pytest.mark.parametrize("d", [32, 64, 128])
def test_longer_sequences(d, dtype, causal):
    _run([1030, 517], [1030, 517], 4, 2, d, causal, dtype)


@gpu
@BOTH
@pytest.mark.parametrize("hq,hk", [(2, 2), (4, 1), (6, 2)])
def test_long_causal_sequences_of_very_different_lengths(hq, hk, dtype):
    """Tiles in descending order of work: every tile of every sequence once, whatever the lengths."""
    _run([700, 0, 1, 1300, 257, 512], [700, 0, 1, 1300, 257, 512], hq, hk, 32, True, dtype)
    _run([1400, 30, 900, 0], [600, 1100, 900, 300], hq, hk, 32, True, dtype, room=[640, 1500, 900, 640], front=5, behind=60)


@gpu
@BOTH
@pytest.mark.parametrize("lq,lk,hq,hk,d,bad", [([200], [200], 4, 2, 64, 150), ([700, 40], [700, 40], 2, 2, 32, 650), ([300], [300], 6, 2, 128, 3),
                                               ([5, 9], [100, 12], 4, 2, 40, 97), ([3], [3000], 2, 1, 20, 2998), ([20], [20], 2, 2, 16, 7)])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_later_keys_that_are_not_finite_leave_no_trace_in_earlier_rows(lq, lk, hq, hk, d, bad, value, dtype):
    """One key and value of the first sequence is not finite: rows in front of it are what they are without it, bit for bit where nothing has to be
    made again, and within both results' roundings otherwise: h |out| for each store, fp32 sums of n terms, and with bf16 the rounding of P to
    bf16 in the products (it is not rounded where sums are made again): sum_j h p_j |v_j| <= h max|v| because sum p = 1.  (This last term was
    missing at first: fp32 passed, bf16 differed by 4.9e-4 where h max|v| = 1.6e-2.)  Rows that see an infinite value are infinite."""
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention, pack_offsets
    q, k, v = (torch.randn(n, h, d, generator=_gen(n + h)).to(dtype).to(DEV) for n, h in ((sum(lq), hq), (sum(lk), hk), (sum(lk), hk)))
    off_q, off_k = pack_offsets(lq, DEV), pack_offsets(lk, DEV)
    m = PackedAttention(causal=True)
    for hints in ({}, dict(max_q=max(lq), max_k=max(lk))):
        clean = m(q, k, v, off_q, off_k, **hints).double()
        k2, v2 = k.clone(), v.clone()
        v2[bad, :, ::3] = value
        out = m(q, k, v2, off_q, off_k, **hints).double()
        first = bad - (lk[0] - lq[0])                       # the first row that sees the key
        n = (max(lk) * U * 4 + (_half_step(dtype) if dtype == torch.bfloat16 else 0.0)) * float(v.double().abs().max())
        for rows in (slice(0, max(first, 0)), slice(lq[0], sum(lq))):
            assert torch.isfinite(out[rows]).all()
            err = (out[rows] - clean[rows]).abs()
            assert (err <= n + 2 * _half_step(dtype) * clean[rows].abs()).all()
        seen = out[max(first, 0):lq[0], :, ::3]
        assert (seen.isnan() if math.isnan(value) else (seen == value) | seen.isnan()).all()
        k2[bad] = value
        out = m(q, k2, v2, off_q, off_k, **hints)
        assert torch.isfinite(out[:max(first, 0)]).all() and torch.isfinite(out[lq[0]:]).all()


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


@gpu
def test_caches_of_more_than_2_to_the_31_elements():
    """Rows that lie beyond 2^31 elements (and 2^32 bytes) of a cache; the rest of it is never touched."""
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention
    tokens, kv, d = 2_200_000, 8, 128
    k, v = (torch.empty(tokens, kv, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    small = [torch.randn(300, kv, d, generator=_gen(i)).to(torch.bfloat16).to(DEV) for i in range(2)]
    k[-300:], v[-300:] = small
    off_k = torch.tensor([tokens - 300, tokens - 40, tokens], dtype=torch.int32, device=DEV)
    near = torch.tensor([0, 260, 300], dtype=torch.int32, device=DEV)
    m = PackedAttention(causal=True)
    for lq in ([1, 1], [30, 17], [260, 40]):
        off_q = torch.tensor([0, lq[0], sum(lq)], dtype=torch.int32, device=DEV)
        q = torch.randn(sum(lq), 16, d, generator=_gen(9)).to(torch.bfloat16).to(DEV)
        hints = dict(max_q=max(lq), max_k=260)
        assert torch.equal(m(q, k, v, off_q, off_k, **hints), m(q, *small, off_q, near, **hints))


@gpu
@BOTH
def test_no_keys_and_no_queries(dtype):
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention
    m = PackedAttention(causal=True)
    q, none = torch.randn(6, 4, 16, device=DEV).to(dtype).requires_grad_(), torch.empty(0, 2, 16, device=DEV, dtype=dtype, requires_grad=True)
    off, zero = torch.tensor([0, 6], dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    out, lse = m(q, none, none, off, zero, return_lse=True)
    dq, dk = torch.autograd.grad(out, (q, none), torch.ones_like(out))
    assert (out == 0).all() and torch.isinf(lse).all() and (dq == 0).all() and dk.shape == none.shape
    kv = torch.randn(6, 2, 16, device=DEV).to(dtype).requires_grad_()
    empty = torch.empty(0, 4, 16, device=DEV, dtype=dtype, requires_grad=True)
    out = m(empty, kv, kv, zero, off)
    assert out.shape == empty.shape
    assert (torch.autograd.grad(out, kv, torch.empty_like(out))[0] == 0).all()


@gpu
@BOTH
def test_large_scores_and_a_temperature(dtype):
    """Scores of +-several hundred: the running maximum is passed by many powers of two from tile to tile."""
    _run([300], [300], 2, 2, 64, True, dtype, scale=40.0, temperature=2.0)


@gpu
@BOTH
@pytest.mark.parametrize("hq,hk,d", [(1, 1, 64), (8, 2, 128), (16, 1, 64), (40, 1, 32), (6, 2, 20), (12, 4, 4)])
@pytest.mark.parametrize("lens", [[1], [1000], [5, 1, 300, 64, 2000], [0, 129]])
def test_single_tokens_over_a_cache(lens, hq, hk, d, dtype):
    _run([1] * len(lens), lens, hq, hk, d, True, dtype, room=[n + 9 for n in lens], train=False)


@gpu
@BOTH
@pytest.mark.parametrize("hq,hk,d", [(8, 2, 128), (4, 4, 64), (2, 1, 16), (3, 3, 33)])
def test_single_tokens_over_long_caches(hq, hk, d, dtype):
    """Ranges of keys for blocks of their own, whose partial results are joined; sequences that end in the first range, or have no keys."""
    _run([1] * 5, [9000, 31, 0, 4097, 1025], hq, hk, d, True, dtype, room=[9001, 40, 3, 4097, 1030], train=False, front=1, behind=4)
    _run([3, 0, 2], [6000, 500, 2], hq, hk, d, True, dtype, room=[6000, 500, 8], train=False, hints=False)


@gpu
@MASK
@BOTH
@pytest.mark.parametrize("hq,hk,d", [(16, 16, 16), (4, 2, 32), (6, 1, 64), (2, 2, 5), (8, 4, 20)])
def test_short_sequences(hq, hk, d, dtype, causal):
    """A wave per sequence and key head, up to two tiles on either side."""
    lengths = [30, 2, 0, 1, 8, 31, 32, 33, 10, 5]
    _run(lengths, lengths, hq, hk, d, causal, dtype)
    _run([5, 10, 0, 7, 3], [60, 4, 9, 0, 33], hq, hk, d, causal, dtype, room=[64, 6, 9, 3, 64], front=4, behind=9)


@gpu
@BOTH
@pytest.mark.parametrize("lq", [[2, 3, 1], [1, 0, 9], [40, 1, 1]])
@pytest.mark.parametrize("hints", [True, False])
def test_a_few_tokens_over_a_cache(lq, hints, dtype):
    _run(lq, [700, 40, 1025], 8, 2, 64, True, dtype, room=[704, 41, 1030], train=False, front=2, behind=3, hints=hints)


@gpu
@BOTH
@pytest.mark.parametrize("hints", [(1, 1), (1, 4000), (1, 0), (300, 1)])
def test_wrong_hints_change_nothing(hints, dtype):
    """Any kernel gives the right result for any lengths, forward and backward."""
    _run([200, 100, 0, 33], [200, 100, 7, 500], 4, 2, 64, True, dtype, hints=hints)
    _run([200, 70], [130, 90], 3, 3, 16, False, dtype, hints=hints)


@gpu
def test_gradients_against_differences():
    """fp32: (f(x + t w) - f(x - t w)) / 2t along random directions, t = 1e-2, f summed in fp64.  The third-order term t^2 / 6 and the forward's
    noise 1e-6 / t = 1e-4 per value, both random over 97 x 4 x 32 values, stay far below 1e-2 of the slope's scale sqrt(values)."""
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention, pack_offsets
    off = pack_offsets([60, 37], DEV)
    x = [torch.randn(97, n, 32, generator=_gen(50 + n)).to(DEV) for n in (4, 2, 2)]
    w = [torch.randn(97, n, 32, generator=_gen(60 + n)).to(DEV) for n in (4, 2, 2)]
    g = torch.randn(97, 4, 32, generator=_gen(70)).to(DEV)
    for causal in (False, True):
        m = PackedAttention(causal=causal)
        f = lambda z: (m(*z, off).double() * g.double()).sum()
        leaves = [t.clone().requires_grad_() for t in x]
        grads = torch.autograd.grad(m(*leaves, off), leaves, g)
        for i in range(3):
            t = 1e-2
            up, dn = list(x), list(x)
            up[i], dn[i] = x[i] + t * w[i], x[i] - t * w[i]
            slope = float((grads[i].double() * w[i].double()).sum())
            assert abs(slope - float(f(up) - f(dn)) / (2 * t)) < 1e-2 * math.sqrt(97 * 4 * 32), (causal, i)


@gpu
@BOTH
def test_given_out_keeps_rows_of_no_sequence(dtype):
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention
    q = torch.randn(20, 4, 16, generator=_gen(1)).to(dtype).to(DEV)
    off = torch.tensor([3, 8, 15], dtype=torch.int32, device=DEV)
    m = PackedAttention()
    out = torch.full_like(q, 7.0)
    res = m(q, q, q, off, out=out)
    new = m(q, q, q, off)
    assert res.data_ptr() == out.data_ptr() and torch.equal(out[3:15], new[3:15])
    assert (out[:3] == 7).all() and (out[15:] == 7).all() and (new[:3] == 0).all() and (new[15:] == 0).all()


@gpu
@BOTH
def test_offsets_outside_the_tensors_are_clamped(dtype):
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention
    q = torch.randn(20, 2, 16, generator=_gen(1)).to(dtype).to(DEV)
    m = PackedAttention(causal=True)
    good = m(q, q, q, torch.tensor([0, 9, 20], dtype=torch.int32, device=DEV))
    bad = m(q, q, q, torch.tensor([-5, 9, 2 ** 31 - 1], dtype=torch.int32, device=DEV), k_len=torch.tensor([9, 2 ** 31 - 1], dtype=torch.int32, device=DEV))
    assert torch.equal(good, bad)
    x = q.clone().requires_grad_()
    for off in ([0, 15, 4], [30, 40, 50], [-9, -3, -1]):       # wrong rows at worst, nothing outside
        off = torch.tensor(off, dtype=torch.int32, device=DEV)
        y = m(x, x, x, off, k_len=torch.tensor([-4, 100], dtype=torch.int32, device=DEV))
        torch.autograd.grad(y, x, torch.ones_like(y))
    torch.cuda.synchronize()


@gpu
@BOTH
def test_results_do_not_depend_on_the_run(dtype):
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention, pack_offsets
    off = pack_offsets([500, 0, 900, 20], DEV)
    x = [torch.randn(1420, n, 64, generator=_gen(n)).to(dtype).to(DEV).requires_grad_() for n in (8, 2, 2)]
    g = torch.randn(1420, 8, 64, generator=_gen(9)).to(dtype).to(DEV)
    runs = []
    for _ in range(3):
        y = PackedAttention(causal=True)(*x, off)
        runs.append((y.detach(),) + torch.autograd.grad(y, x, g))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


@gpu
@BOTH
def test_whole_path_trains_serves_and_replays(dtype):
    """Projection -> norms and rotation -> attention, as a token stage uses them: the whole series at once, its last token over the cache, and
    both from a captured graph with other lengths and values put into the same buffers."""
    from uncrtaints_amd.src.backbones.packed_attention import HeadNormRotary, PackedAttention, pack_offsets
    from uncrtaints_amd.src.backbones.positional_encoding import RotaryAxes
    heads, kv, d, lengths, room = 8, 2, 32, [37, 64, 5], 70
    norms = HeadNormRotary(d, rotary=RotaryAxes(d, sections=(8, 12, 12), T=(10000.0, 100.0, 100.0))).to(DEV)
    attend = PackedAttention(causal=True)
    n = sum(lengths)
    qkv = torch.randn(n, heads + 2 * kv, d, generator=_gen(3)).to(dtype).to(DEV).requires_grad_()
    pos = torch.stack([torch.arange(n) // 8, torch.arange(n) % 8, torch.arange(n) % 5], 1).to(torch.int32).to(DEV)
    off = pack_offsets(lengths, DEV)
    g = torch.randn(n, heads, d, generator=_gen(4)).to(dtype).to(DEV)

    def step():
        q, k = norms(qkv[:, :heads], qkv[:, heads:heads + kv], pos)
        y = attend(q, k, qkv[:, heads + kv:], off, max_q=64)
        # detached: a captured graph's outputs do not keep an autograd graph of these leaves alive
        return (y.detach(), k.detach()) + torch.autograd.grad(y, (qkv, norms.q_weight, norms.k_weight), g)

    eager = [t.detach().clone() for t in step()]
    assert all(torch.isfinite(t).all() for t in eager)
    # serving: the last token of every series over a cache that holds the others
    cache_k = torch.full((3, room, kv, d), math.nan, dtype=dtype, device=DEV)
    cache_v = torch.full_like(cache_k, math.nan)
    for b, ln in enumerate(lengths):
        at = int(off[b])
        cache_k[b, :ln], cache_v[b, :ln] = eager[1][at:at + ln], qkv.detach()[at:at + ln, heads + kv:]
    last = off[1:].long() - 1
    one = torch.arange(4, device=DEV, dtype=torch.int32)
    with torch.no_grad():
        q1, _ = norms(qkv[last, :heads], qkv[last, heads:heads + kv], pos[last])
    k_len = torch.tensor(lengths, dtype=torch.int32, device=DEV)

    def serve():
        return attend(q1, cache_k.view(3 * room, kv, d), cache_v.view(3 * room, kv, d), one, one * room, k_len=k_len, max_q=1, max_k=64)

    served = serve()
    assert float((served.float() - eager[0][last].float()).abs().max()) < (0.05 if dtype == torch.bfloat16 else 1e-5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step() + (serve(),)
    for i in range(4):
        with torch.no_grad():
            if i == 2:
                qkv.mul_(-1.0)
                off.copy_(pack_offsets([1, 80, 25], DEV))
                k_len.copy_(torch.tensor([5, 9, 5], dtype=torch.int32, device=DEV))
        want = [t.detach().clone() for t in step()] + [serve().clone()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, held):
            assert torch.equal(a, b), i
        if i < 2:
            assert all(torch.equal(a, b) for a, b in zip(eager, want))


@gpu
def test_two_streams_at_once():
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention, pack_offsets
    m = PackedAttention(causal=True)
    off = [pack_offsets([1] * 4, DEV), pack_offsets([3000, 2000, 10, 400], DEV)]
    x = [torch.randn(5410, n, 64, generator=_gen(n)).to(torch.bfloat16).to(DEV) for n in (8, 2, 2)]
    qs = [torch.randn(4, 8, 64, generator=_gen(20 + i)).to(torch.bfloat16).to(DEV) for i in range(2)]
    want = [m(q, x[1], x[2], off[0], off[1], max_q=1) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(m(qs[i], x[1], x[2], off[0], off[1], max_q=1))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_packed_attention_refuses():
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention, pack_offsets
    for t in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            PackedAttention(temperature=t)
    with pytest.raises(ValueError):
        pack_offsets([3, -1], "cpu")
    m = PackedAttention()
    q, k, off = torch.zeros(6, 4, 8), torch.zeros(6, 2, 8), pack_offsets([2, 4], "cpu")
    assert off.tolist() == [0, 2, 6] and off.dtype == torch.int32
    for args, kw in (((q[0], k, k, off), {}), ((q, k, k[:5], off), {}), ((q, k, k[..., :4], off), {}), ((q[..., :4], k, k, off), {}),
                     ((torch.zeros(6, 4, 129), torch.zeros(6, 2, 129), torch.zeros(6, 2, 129), off), {}),
                     ((q[:, :3], k, k, off), {}), ((q, k[:, :0], k[:, :0], off), {}), ((q[:4], k, k, off), {}),
                     ((q, k, k, off.long()), {}), ((q, k, k, off.view(1, 3)), {}), ((q, k, k, off[::2]), {}), ((q, k, k, off, off[:2]), {}),
                     ((q, k, k, off[:1]), {}), ((q, k, k, off), dict(k_len=off)), ((q, k, k, off), dict(k_len=off[:2].float())),
                     ((q, k, k, off), dict(max_q=-1))):
        with pytest.raises(ValueError):
            m(*args, **kw)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        m(q.half(), k.half(), k.half(), off)
    with pytest.raises(RuntimeError, match="but q is"):
        m(q, k.bfloat16(), k, off)
    with pytest.raises(RuntimeError, match="cuda device"):
        m(q, k, k, off)


@gpu
def test_packed_attention_refuses_on_the_gpu():
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention, pack_offsets
    m = PackedAttention()
    q, off = torch.zeros(6, 4, 8, device=DEV), pack_offsets([2, 4], DEV)
    with pytest.raises(RuntimeError, match="offsets_q"):
        m(q, q, q, off.cpu())
    with pytest.raises(ValueError, match="without gradients"):
        m(q.clone().requires_grad_(), q, q, off, out=torch.empty_like(q))
    with pytest.raises(ValueError, match="contiguous"):
        m(q, q, q, off, out=torch.empty(6, 4, 16, device=DEV)[..., :8])
    with pytest.raises(RuntimeError, match="but q is"):
        m(q, q, q, off, out=torch.empty_like(q, dtype=torch.bfloat16))
    z = torch.zeros(12, 4, 8, device=DEV)
    with pytest.raises(ValueError, match="shares"):
        m(q, z[:6], z[6:], off, out=z[6:])


def test_entry_points_refuse_bad_sizes():
    """The C entries' own checks: no GPU is needed, nothing is enqueued."""
    from uncrtaints_amd import hip_backend as hb
    fwd = hb.lib().fn["uncr_packed_attn_fwd"]
    names = [n for _, n in hb.parse_header()["uncr_packed_attn_fwd"]]
    ok = dict.fromkeys(names, 0)
    ok.update(q=16, k=16, v=16, out=16, off_q=16, off_k=16, lse=None, k_len=None, temperature=1.0, B=1, Nq=0, Nk=4, Hq=4, Hk=2, D=8, stream=None)
    ok["work"] = None
    call = lambda **kw: fwd(*{**ok, **kw}.values())
    assert call() == 0
    for kw in (dict(B=0), dict(Nq=-1), dict(Nk=-1), dict(Hq=3), dict(Hk=0), dict(D=0), dict(D=129), dict(act=2), dict(temperature=0.0), dict(temperature=math.nan),
               dict(off_q=None), dict(off_k=None), dict(Nq=1 << 30, Hq=8), dict(Nq=2, q=None), dict(Nq=2, out=None), dict(Nq=2, k=None),
               dict(Nq=2, out=18), dict(Nq=2, Nk=40000, max_q=1, max_k=20000), dict(Nq=2, Nk=40000, max_q=1, max_k=20000, work=16, work_floats=99)):
        assert call(**kw) < 0, kw
    assert hb.query("uncr_packed_attn_work", 1, 20000, 1, 2, 40000, 4, 2, 8, 0) > 99 and hb.query("uncr_packed_attn_work", 1, 100, 1, 2, 200, 4, 2, 8, 0) == 0
    bwd = hb.lib().fn["uncr_packed_attn_bwd"]
    names = [n for _, n in hb.parse_header()["uncr_packed_attn_bwd"]]
    ok2 = dict.fromkeys(names, 0)
    ok2.update(q=16, k=16, v=16, out=16, dout=16, lse=16, dq=16, dk=16, dv=16, rowstat=16, off_q=16, off_k=16, k_len=None, temperature=1.0, B=1, Nq=2, Nk=2, Hq=4,
               Hk=2, D=8, stream=None)
    for kw in (dict(Hq=5), dict(D=200), dict(lse=None), dict(rowstat=None), dict(dq=None), dict(dk=None), dict(v=None), dict(dk=24 - 4), dict(act=-1)):
        assert bwd(*{**ok2, **kw}.values()) < 0, kw


@gpu
@BOTH
@pytest.mark.parametrize("lq, lk, hq, hk, d, hints", [
    ([1, 1, 1], [20000, 0, 4000], 4, 2, 8, True), ([1, 1], [300, 700], 4, 4, 64, True), ([40, 3], [40, 3], 4, 2, 16, True), ([5, 30], [5, 30], 2, 2, 16, True),
    ([100, 700], [600, 700], 2, 1, 32, False), ([300], [300], 2, 2, 128, False)])
def test_a_query_that_is_not_a_number_gives_a_row_that_is_none(lq, lk, hq, hk, d, hints, dtype):
    """In every kernel, the one that joins parts of a cache among them: NaN in the row's result and its lse, the other rows as they should be.
    A row that sees no key is 0 whatever its query holds."""
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention
    g = _gen(5)
    q, k, v = (torch.randn(n, h, d, generator=g).to(dtype) for n, h in ((sum(lq), hq), (sum(lk), hk), (sum(lk), hk)))
    off_q, off_k = _offsets(lq), _offsets(lk)
    bad = [(int(off_q[b]) + min(n - 1, b), (b + 1) % hq) for b, n in enumerate(lq)]
    for t, h in bad:
        q[t, h, d // 2] = math.nan
    out, lse = PackedAttention()(q.to(DEV), k.to(DEV), v.to(DEV), off_q.to(DEV), off_k.to(DEV), return_lse=True,
                                 **(dict(max_q=max(lq), max_k=max(lk)) if hints else {}))
    out, lse = out.cpu(), lse.cpu()
    for b, n in enumerate(lq):
        rq, rk = slice(int(off_q[b]), int(off_q[b]) + n), slice(int(off_k[b]), int(off_k[b]) + lk[b])
        for h in range(hq):
            c = h // (hq // hk)
            qs = q[rq, h].double()
            rows = torch.isfinite(qs).all(1)
            ref = reference(qs[rows][None], k[rk, c].double(), v[rk, c].double(), torch.zeros(1, int(rows.sum()), d, dtype=torch.float64), False,
                            math.sqrt(d), dtype)
            _check("out", out[rq, h][rows], *(t[0] for t in ref["out"]))
            _check("lse", lse[rq, h][rows], *(t[0] for t in ref["lse"]))
            if lk[b]:
                assert out[rq, h][~rows].isnan().all() and lse[rq, h][~rows].isnan().all()
            else:
                assert (out[rq, h] == 0).all() and (lse[rq, h] == -math.inf).all()


@gpu
def test_more_single_tokens_than_shared_blocks_hold():
    """1.1 million series of one date, 8 heads, nothing known of their lengths: one key each, so out is v -- the product with p, the reciprocal of
    l = p (2.5 units at most, 5 half steps) and the product with it: 7 u."""
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention
    n = 1_100_000
    g = torch.Generator(device=DEV).manual_seed(6)
    q, k, v = (torch.randn(n, 8, 4, generator=g, device=DEV) for _ in range(3))
    out = PackedAttention()(q, k, v, torch.arange(n + 1, dtype=torch.int32, device=DEV))
    assert bool(((out - v).abs() <= 7 * U * v.abs()).all())


@gpu
def test_out_counts_as_a_change_in_place():
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention, pack_offsets
    m, off = PackedAttention(), pack_offsets([2, 4], DEV)
    q, w = torch.randn(6, 4, 8, generator=_gen(7)).to(DEV), torch.ones(6, 4, 8, device=DEV, requires_grad=True)
    with pytest.raises(ValueError, match="requires one"):
        m(q, q, q, off, out=w)
    out = torch.zeros(6, 4, 8, device=DEV)
    loss = (out * w).sum()
    m(q, q, q, off, out=out)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


def test_scales_and_sizes_beyond_the_built_ones_are_refused():
    """Temperatures whose scale is no number in fp32, and launches of more threads than are counted: refused before anything is enqueued."""
    from uncrtaints_amd import engine as E
    from uncrtaints_amd import hip_backend as hb
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention
    for t in (1e-31, 1e-45, 1e31):
        with pytest.raises(ValueError, match="1e-30"):
            PackedAttention(temperature=t)
    with pytest.raises(RuntimeError, match="31 bits"):
        E.packed_attention_forward(torch.zeros(1, 1, 2).expand(2 ** 31, 1, 2), *(torch.zeros(4, 1, 2),) * 2, *(torch.zeros(2, dtype=torch.int32),) * 2, None, 1.0,
                                   False, False)
    args = lambda name: dict.fromkeys([n for _, n in hb.parse_header()[name]], 0)
    big = 1 << 22
    ok = {**args("uncr_packed_attn_fwd"), **dict(q=16, k=16, v=16, out=16, off_q=16, off_k=16, lse=None, k_len=None, work=None, temperature=1.0, B=big, Nq=big,
                                                 Nk=big, Hq=64, Hk=64, D=8, stream=None)}
    shape = hb.lib().fn["uncr_packed_attn_fwd"](*{**ok, "D": 0}.values())
    for kw in (dict(), dict(max_q=1, max_k=60), dict(D=128), dict(max_q=64, D=64)):
        assert hb.lib().fn["uncr_packed_attn_fwd"](*{**ok, **kw}.values()) == shape, kw
    for t in (1e-31, 1e31):
        assert hb.lib().fn["uncr_packed_attn_fwd"](*{**ok, "B": 1, "Nq": 0, "temperature": t}.values()) < 0
    ok = {**args("uncr_packed_attn_bwd"), **dict(q=16, k=16, v=16, out=16, dout=16, lse=16, dq=16, dk=16, dv=16, rowstat=16, off_q=16, off_k=16, k_len=None,
                                                 work=None, temperature=1.0, B=big, Nq=big, Nk=big, Hq=128, Hk=128, D=8, stream=None)}
    for kw in (dict(), dict(max_q=1, max_k=60), dict(Nq=0), dict(D=128)):
        assert hb.lib().fn["uncr_packed_attn_bwd"](*{**ok, **kw}.values()) == shape, kw


@gpu
@MASK
@BOTH
@pytest.mark.parametrize("hq, hk, d", [(3, 3, 16), (4, 2, 32), (2, 2, 64), (6, 2, 40), (2, 2, 128), (3, 1, 72), (2, 1, 127)])
def test_many_short_sequences_with_many_rows(hq, hk, d, dtype, causal):
    """Enough sequences for whole launches of the smaller blocks (up to 64 rows and 48 keys on average), some of them far longer"""
    g = _gen(70)
    lq = [int(n) for n in torch.randint(0, 45, (1100 // hk,), generator=g)] + [1, 150, 0, 64, 65]
    _run(lq, lq, hq, hk, d, causal, dtype, seed=71, hints=False, front=2, behind=3)


@gpu
@MASK
@BOTH
def test_many_short_sequences_over_other_keys(dtype, causal):
    g = _gen(72)
    lq = [int(n) for n in torch.randint(30, 45, (600,), generator=g)]
    lk = [int(n) for n in torch.randint(0, 80, (600,), generator=g)]
    _run(lq, lk, 4, 2, 128, causal, dtype, room=[n + 3 for n in lk], seed=73, hints=False)


def _compiles(tmp_path, body):
    """Does a kernel with this body, next to the attention kernels' header, compile? -> (status, messages)"""
    import os
    import subprocess
    from uncrtaints_amd import build
    src = tmp_path / "probe.hip"
    src.write_text('#include "packed_attn.h"\n__global__ void probe(float* out) {\n' + body + "\n}\n")
    r = subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "--offload-arch=gfx950", "-std=c++17", "-fsyntax-only", "-I" + build.CSRC, str(src)],
                       capture_output=True, text=True, timeout=100)
    return r.returncode, r.stdout + r.stderr


def test_the_sums_of_joining_waves_stay_inside_one_lds_object(tmp_path):
    """Forward and dQ blocks whose waves share the keys (half as many groups as waves) add their sums through the tiles' LDS: every built
    instance's sums lie inside the object they are addressed in, and a geometry whose sums do not is no program."""
    built = [("__bf16", 32, 64, 2), ("__bf16", 64, 64, 2), ("__bf16", 128, 64, 4), ("float", 32, 64, 2), ("float", 64, 64, 2), ("AttnThree", 32, 64, 2)]
    body = "".join(f"{{ __shared__ AttnBuffers<{t}, {dp}, {tk}> b; float* p = b.template join<{groups}>({groups} - 1);\n"
                   f"  static_assert(sizeof(b) == sizeof(b.k) + sizeof(b.v)); p[{max(dp, 32) // 32} * 1024 - 1] = 0.f; out[0] = p[0]; }}\n"
                   for t, dp, tk, groups in built)
    status, said = _compiles(tmp_path, body)
    assert status == 0, said
    status, said = _compiles(tmp_path, "__shared__ AttnBuffers<__bf16, 128, 32> b; out[0] = b.template join<4>(3)[0];")
    assert status != 0 and "do not hold the sums" in said


def test_extent_of_a_tensor():
    from uncrtaints_amd import engine as E
    z = torch.zeros(4, 6, 8)
    at = z.data_ptr()
    assert E.extent(z) == (at, at + 4 * 192) and E.extent(z[1:3]) == (at + 4 * 48, at + 4 * 144) and E.extent(z[:0]) == (z[:0].data_ptr(),) * 2
    assert E.extent(z[:, 1:3]) == (at + 4 * 8, at + 4 * (144 + 24)) and E.extent(z[..., ::2]) == (at, at + 4 * 191)
    assert E.extent(z[:1].expand(9, 6, 8)) == (at, at + 4 * 48) and E.extent(z.transpose(0, 2)) == E.extent(z)


@gpu
def test_out_beside_the_inputs_in_one_buffer():
    """A workspace that a program cuts up itself: rows that do not overlap are served, any that do are refused, the offsets' among them."""
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention, pack_offsets
    m = PackedAttention()
    z = torch.randn(4 * 6 + 1, 4, 8, generator=_gen(8)).to(DEV)
    q, k, v, out = (z[6 * i:6 * i + 6] for i in range(4))
    off = pack_offsets([2, 4], DEV)
    want = m(q, k, v, off)
    kept = z.clone()
    got = m(q, k, v, off, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out, want)
    kept[18:24] = want
    assert torch.equal(z, kept)
    z[24].view(-1)[:3] = off.view(torch.float32)
    inside = z[24].view(-1)[:3].view(torch.int32)
    assert torch.equal(m(q, k, v, inside, out=out), want)
    for bad in (z[17:23], z[1:7], z[11:17]):
        with pytest.raises(ValueError, match="shares"):
            m(q, k, v, off, out=bad)
    with pytest.raises(ValueError, match="shares"):
        m(q, k, v, inside, out=z[19:25])
    with pytest.raises(ValueError, match="shares"):
        m(q, k, v, off, offsets_k=off, k_len=inside[1:], out=z[19:25])
    with pytest.raises(ValueError, match="shares"):          # rows of a strided input around it
        m(z[::4][:6], k, v, off, out=out)
    assert torch.equal(z[:18], kept[:18])
    empty = torch.zeros(0, 4, 8, device=DEV)
    assert m(empty, k, v, torch.zeros(2, dtype=torch.int32, device=DEV), torch.tensor([0, 6], dtype=torch.int32, device=DEV), out=empty).shape == (0, 4, 8)


def _wide(lens, hk, G, d, dtype, aligned, causal):
    """Forward and backward with `hk` key heads that repeat three"""
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention
    n, g, base = sum(lens), _gen(80 + d), 3
    q, k, v, do = (torch.randn(n, h, d, generator=g).to(dtype) for h in (base * G, base, base, base * G))

    def repeat(t, per):          # [n, base * per, d] -> [n, hk * per, d], key head c repeating c % base
        idx = torch.cat([torch.arange(per) + c % base * per for c in range(hk)])
        t = t.to(DEV)[:, idx.to(DEV)]
        if aligned:
            return t
        z = torch.empty(n, t.shape[1] * d + 3, dtype=dtype, device=DEV)
        z[:, 1:1 + t.shape[1] * d] = t.flatten(1)
        return z[:, 1:1 + t.shape[1] * d].unflatten(1, (t.shape[1], d))

    leaves = [repeat(t, per).detach().requires_grad_() for t, per in ((q, G), (k, 1), (v, 1))]
    off = _offsets(lens)
    out, lse = PackedAttention(causal=causal)(*leaves, off.to(DEV), return_lse=True)
    got = dict(zip(("out", "lse", "dq", "dk", "dv"), (out.detach(), lse, *torch.autograd.grad(out, leaves, repeat(do, G)))))
    for name, t in got.items():          # the heads that repeat the first three are equal to them, bit for bit
        per = G if name in ("out", "lse", "dq") else 1
        for c in range(base, hk):
            assert torch.equal(t[:, c * per:(c + 1) * per], t[:, c % base * per:(c % base + 1) * per]), (name, c)
        got[name] = t[:, :base * per].cpu()
    for b, length in enumerate(lens):
        rows = slice(int(off[b]), int(off[b]) + length)
        for c in range(base):
            hs = slice(c * G, (c + 1) * G)
            ref = reference(q[rows, hs].double().transpose(0, 1), k[rows, c].double(), v[rows, c].double(), do[rows, hs].double().transpose(0, 1), causal,
                            math.sqrt(d), dtype)
            for name in ("out", "dq"):
                _check(name, got[name][rows, hs], *(t.transpose(0, 1) for t in ref[name]))
            _check("lse", got["lse"][rows, hs], *(t.T for t in ref["lse"]))
            for name in ("dk", "dv"):
                _check(name, got[name][rows, c], *ref[name])


# The instances that only launches of 1024 blocks and more take (whole blocks of rows, four pairs of waves in dK/dV, with and without tiles in
# descending order of work), over long sequences: many key heads that repeat three, so that the reference has only those to make.
WIDE = [   # lengths, key heads, queries per key head, d, types, aligned rows
    ([1700, 900, 1800], 64, 1, 128, (torch.bfloat16, torch.float32), True),
    ([1700, 900, 1800], 64, 1, 64, (torch.bfloat16, torch.float32), True),
    ([1700, 900, 1800], 64, 1, 32, (torch.bfloat16, torch.float32), True),
    ([1300, 0, 1500], 64, 1, 20, (torch.bfloat16, torch.float32), True),
    ([1700, 1, 1800], 64, 1, 72, (torch.bfloat16,), True),
    ([1100, 1300], 16, 8, 128, (torch.bfloat16,), True),
    ([1100, 1300], 64, 1, 32, (torch.float32, torch.bfloat16), False),
    ([1100, 1300], 64, 1, 64, (torch.float32, torch.bfloat16), False),
    ([1400, 1500], 64, 2, 127, (torch.bfloat16, torch.float32), False),
    ([400, 300, 500, 480], 64, 2, 64, (torch.float32,), True),
    ([400, 300, 500, 480], 64, 2, 32, (torch.float32,), True),
]


@gpu
@MASK
@pytest.mark.parametrize("lens,hk,G,d,dtype,aligned", [(*w[:4], t, w[5]) for w in WIDE for t in w[4]])
def test_launches_of_many_blocks_over_long_sequences(lens, hk, G, d, dtype, aligned, causal):
    _wide(lens, hk, G, d, dtype, aligned, causal)


@gpu
@MASK
@BOTH
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("G,d", [(1, 32), (1, 64), (1, 128), (3, 64), (2, 36), (1, 100)])
def test_many_sequences_of_up_to_64_rows(G, d, aligned, dtype, causal):
    """33 to 64 rows on average, enough sequences for 1024 blocks: blocks of two waves, forward and backward"""
    lens = [int(n) for n in torch.randint(33 // G, 60 // G, (64,), generator=_gen(90 + G))] + [0, 130, 1]
    _wide(lens, 24, G, d, dtype, aligned, causal)


@gpu
@BOTH
@pytest.mark.parametrize("d", [16, 32, 64, 128])
def test_wave_kernels_over_rows_that_start_at_no_vector_boundary(d, dtype):
    _run([1] * 3, [700, 0, 130], 4, 2, d, True, dtype, room=[704, 3, 130], train=False, layout="odd_start")
    _run([1, 2], [5000, 300], 8, 2, d, True, dtype, train=False, layout="odd_start", hints=False)
    _run([20, 3, 40, 0, 31], [20, 3, 40, 0, 31], 3, 3, d, True, dtype, layout="odd_start")
    _run([9, 3], [60, 33], 4, 2, d, False, dtype, layout="odd_start")
    _run([70, 3, 131], [70, 3, 131], 4, 2, d, True, dtype, layout="odd_start")
    _run([1] * 3, [700, 0, 130], 4, 2, d, True, dtype, room=[704, 3, 130], train=False)


@gpu
@BOTH
def test_two_captured_graphs_with_workspaces_replayed_at_once(dtype):
    """Ranges of a cache (partial results) and, in fp32, long sequences in three parts: each graph has a workspace of its own, so replays on two streams
    at once, and eager calls between them, leave each other alone."""
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention, pack_offsets
    m = PackedAttention(causal=True)
    one, lens = pack_offsets([1] * 3, DEV), pack_offsets([6000, 700, 30], DEV)
    k, v = (torch.randn(6730, 2, 64, generator=_gen(i)).to(dtype).to(DEV) for i in (1, 2))
    qs = [torch.randn(3, 8, 64, generator=_gen(10 + i)).to(dtype).to(DEV) for i in range(2)]
    long = [torch.randn(6730, 4, 64, generator=_gen(20 + i)).to(dtype).to(DEV) for i in range(2)]
    calls = [lambda i=i: (m(qs[i], k, v, one, lens, max_q=1, max_k=6000), m(long[i], k, v, lens)) for i in range(2)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    graphs, held = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g, c in zip(graphs, calls):
        with torch.cuda.graph(g):
            held.append(c())
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(4):
        for h in held:
            for t in h:
                t.fill_(7.0)
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            eager = calls[turn % 2]()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(held[i], want[i])), (turn, i)
        assert all(torch.equal(a, b) for a, b in zip(eager, want[turn % 2]))


@gpu
@BOTH
@pytest.mark.parametrize("lens,hints", [([30, 9, 64], True), ([30, 9, 64], False), ([700, 600], False)])
def test_broadcast_inputs_and_gradients(lens, hints, dtype):
    """Heads that share one row in memory, one query for all tokens, and an incoming gradient that is one number: as where each has memory of its own."""
    from uncrtaints_amd.src.backbones.packed_attention import PackedAttention, pack_offsets
    n, off, m = sum(lens), pack_offsets(lens, DEV), PackedAttention(causal=True)
    hints = dict(max_q=max(lens), max_k=max(lens)) if hints else {}
    q1, k1, v1 = (torch.randn(*s, generator=_gen(30 + i)).to(dtype).to(DEV) for i, s in enumerate(((1, 4, 32), (n, 1, 32), (n, 1, 32))))
    views = [q1.expand(n, 4, 32), k1.expand(n, 2, 32), v1.expand(n, 2, 32)]
    got, want = [], []
    for res, own in ((got, False), (want, True)):
        leaves = [(t.contiguous() if own else t).detach().requires_grad_() for t in views]
        y = m(*leaves, off, **hints)
        res += [y.detach(), *torch.autograd.grad(y, leaves, torch.full_like(y, 0.5) if own else torch.full((1, 1, 1), 0.5, dtype=dtype, device=DEV).expand_as(y))]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    base = [t.clone().requires_grad_() for t in (q1, k1, v1)]
    y = m(*(t.expand(n, h, 32) for t, h in zip(base, (4, 2, 2))), off, **hints)
    grads = torch.autograd.grad(y, base, torch.full_like(y, 0.5))
    for g, w, dim in zip(grads, want[1:], (0, 1, 1)):
        assert torch.equal(g, w.sum(dim, keepdim=True))


@gpu
@BOTH
def test_inference_mode(dtype):
    from uncrtaints_amd.src.backbones.packed_attention import HeadNormRotary, PackedAttention, pack_offsets
    from uncrtaints_amd.src.backbones.positional_encoding import RotaryAxes
    x, pos, off = torch.randn(20, 2, 16, generator=_gen(40)).to(dtype).to(DEV), torch.arange(20, device=DEV)[:, None], pack_offsets([11, 9], DEV)
    norm, m = HeadNormRotary(16, rotary=RotaryAxes(16)).to(DEV), PackedAttention()

    def path(**kw):
        q, k = norm(x, x, pos)
        return m(q, k, x, off, **kw).detach()

    want = path()
    with torch.inference_mode():
        out = torch.empty_like(x)
        assert torch.equal(path(), want) and torch.equal(path(out=out), want) and torch.equal(out, want)
    with torch.no_grad():
        assert torch.equal(path(out=out), want)
