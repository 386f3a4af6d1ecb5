"""The rotation by positions with several axes and the norms of queries and keys per head (positional_encoding.RotaryAxes,
packed_attention.HeadNormRotary) against their definition in 64 bits.

Tolerances, fixed before the first run.  u = 2^-24 (fp32 half step), h = finfo(storage).eps / 2 (the one rounding of a store):
  rotation   a c - b s: (cos, sin) are off by at most 8u (angle reduced in 64 bits, rounded to fp32 half turns: pi * u; sincospi 2 ulp
             <= 4u), each product and the sum by 1u of |a| + |b|  ->  (12u) (|a| + |b|) + h |y|
  norms      r = 1/sqrt(mean x^2 + eps): the sum of D <= 256 squares in fp32 by lanes and a tree is off by less than 24u relatively, rsqrt and
             the products by 4u  ->  y as above with another 16u (half of 24u under the root, + 4u) of |a| + |b|
  gradients  dx = r w u - x r^3 / D sum(w u x): every term carries at most 64u of the terms' absolute sum, + h |dx|
             dw = sum over n terms u x r: 64u per term and at most n_seq = 512 fp32 additions in a row -> (64 + 512) u sum |terms|"""
import math

import pytest
import torch

U = 2.0 ** -24
DEV = "cuda"
gpu = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _positions(n, axes, dtype, seed, far=1000):
    p = torch.randint(-far, far, (n, axes), generator=_gen(seed), dtype=torch.int64)
    return (p.double() + 0.25).to(dtype) if dtype.is_floating_point else p.to(dtype)


def _places(d, sections, pairs):
    first, second, axis, freq, at = [], [], [], [], 0
    for a, (n, base) in enumerate(sections):
        for i in range(n // 2):
            first.append(at + (i if pairs == "halves" else 2 * i))
            second.append(at + (i + n // 2 if pairs == "halves" else 2 * i + 1))
            axis.append(a)
            freq.append(base ** (-2.0 * i / n))
        at += n
    return torch.tensor(first), torch.tensor(second), torch.tensor(axis), torch.tensor(freq, dtype=torch.float64)


def _rotate64(x, pos, places, sign=1.0):
    first, second, axis, freq = places
    ang = (pos.double()[:, axis] * freq)[:, None] * sign
    a, b = x[..., first], x[..., second]
    return x.index_copy(-1, first, a * ang.cos() - b * ang.sin()).index_copy(-1, second, a * ang.sin() + b * ang.cos())


def _pair_size(x, places):
    """|a| + |b| of every element's pair (an element that passes through: 0)"""
    s = x[..., places[0]].abs() + x[..., places[1]].abs()
    return torch.zeros_like(x).index_copy(-1, places[0], s).index_copy(-1, places[1], s)


def _norm64(x, w, eps):
    return x * w / (x.square().mean(-1, keepdim=True) + eps).sqrt()


def _check(name, got, ref, bound):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    bad = ((got - ref).abs() > bound) | ~torch.isfinite(got)
    assert not bad.any(), (name, int(bad.sum()), float(((got - ref).abs() - bound).max()))


def _half(dtype):
    return torch.finfo(dtype).eps / 2


SHAPES = [   # d, sections with their bases, pairs
    (64, ((16, 10000.0), (24, 100.0), (24, 100.0)), "halves"),
    (128, ((32, 10000.0), (48, 100.0), (48, 100.0)), "neighbours"),
    (16, ((16, 1000.0),), "halves"),
    (4, ((4, 1000.0),), "neighbours"),
    (2, ((2, 10.0),), "halves"),
    (40, ((8, 10000.0), (12, 50.0)), "halves"),                       # 20 elements pass through
    (18, ((4, 300.0), (6, 20.0), (2, 7.0), (6, 5.0)), "halves"),       # four axes, odd halves
    (18, ((4, 300.0), (6, 20.0), (8, 7.0)), "neighbours"),
    (256, ((64, 10000.0), (96, 100.0), (96, 100.0)), "halves"),
    (202, ((66, 10000.0), (70, 100.0), (66, 100.0)), "halves"),        # more pairs than a wave has lanes, one at a time
]


def _module(d, sections, pairs):
    from uncrtaints_amd.src.backbones.positional_encoding import RotaryAxes
    return RotaryAxes(d, sections=tuple(n for n, _ in sections), T=tuple(b for _, b in sections), pairs=pairs)


@gpu
@pytest.mark.parametrize("d,sections,pairs", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,heads", [(1, 1), (37, 5), (300, 24)])
def test_rotary_axes(d, sections, pairs, dtype, n, heads):
    x = torch.randn(n, heads, d, generator=_gen(1)).to(dtype)
    g = torch.randn(n, heads, d, generator=_gen(2)).to(dtype)
    pos = _positions(n, len(sections), torch.float32, 3)
    places = _places(d, sections, pairs)
    m = _module(d, sections, pairs).to(DEV)
    xd = x.to(DEV).requires_grad_()
    y = m(xd, pos.to(DEV))
    assert y.dtype == dtype and y.is_contiguous()
    ref = _rotate64(x.double(), pos, places)
    _check("y", y, ref, 12 * U * _pair_size(x.double(), places) + _half(dtype) * ref.abs())
    dx, = torch.autograd.grad(y, xd, g.to(DEV))
    ref = _rotate64(g.double(), pos, places, -1.0)
    _check("dx", dx, ref, 12 * U * _pair_size(g.double(), places) + _half(dtype) * ref.abs())


@gpu
@pytest.mark.parametrize("pos_dtype,far", [(torch.float32, 2 ** 20), (torch.float64, 2 ** 40), (torch.int32, 2 ** 31 - 1), (torch.int64, 2 ** 45)])
def test_rotary_far_positions(pos_dtype, far):
    """Angles of 10^6 ... 10^13 radians.  The 64-bit product pos * turns is off by 2^-53 of its value: 2^45 / 2 pi turns * 2^-53 * 2 pi rad
    = 2^-8 / 1 at the fastest pair, so the bound takes 3 * 2^-53 * |angle| radians for either side's rounding beside the usual one."""
    d, sections = 32, ((16, 10000.0), (16, 3.0))
    x = torch.randn(50, 3, d, generator=_gen(4))
    pos = _positions(50, 2, pos_dtype, 5, far)
    places = _places(d, sections, "halves")
    y = _module(d, sections, "halves").to(DEV)(x.to(DEV), pos.to(DEV))
    ref = _rotate64(x.double(), pos, places)
    ang = (pos.double()[:, places[2]] * places[3]).abs()[:, None]
    slack = torch.zeros(50, 1, d, dtype=torch.float64).index_copy(-1, places[0], ang).index_copy(-1, places[1], ang) * 3 * 2.0 ** -53
    _check("y", y, ref, (12 * U + slack) * _pair_size(x.double(), places) + U * ref.abs())


def _views(kind, n, hq, hk, d, dtype, seed):
    """Queries and keys in the layouts a program has them in."""
    if kind == "fused":                                   # slices of one projection
        z = torch.randn(n, hq + 2 * hk, d, generator=_gen(seed)).to(dtype).to(DEV)
        return z[:, :hq], z[:, hq:hq + hk]
    if kind == "heads_first":                             # [heads, tokens, d]
        z = torch.randn(hq + hk, n, d, generator=_gen(seed)).to(dtype).to(DEV).transpose(0, 1)
        return z[:, :hq], z[:, hq:]
    if kind == "odd_start":                               # rows that start at no vector boundary
        z = torch.randn(n, (hq + hk) * d + 3, generator=_gen(seed)).to(dtype).to(DEV)
        return z[:, 1:1 + hq * d].unflatten(1, (hq, d)), z[:, 1 + hq * d:1 + (hq + hk) * d].unflatten(1, (hk, d))
    if kind == "last_strided":                            # d is not the contiguous dimension
        z = torch.randn(n, hq + hk, 2 * d, generator=_gen(seed)).to(dtype).to(DEV)[..., ::2]
        return z[:, :hq], z[:, hq:]
    q = torch.randn(n, hq, d, generator=_gen(seed)).to(dtype).to(DEV)
    return q, torch.randn(n, hk, d, generator=_gen(seed + 1)).to(dtype).to(DEV)


@gpu
@pytest.mark.parametrize("kind", ["plain", "fused", "heads_first", "odd_start", "last_strided"])
@pytest.mark.parametrize("d,sections,pairs", SHAPES)
@pytest.mark.parametrize("dtype,n,hq,hk", [(torch.float32, 53, 6, 2), (torch.bfloat16, 211, 16, 4), (torch.float32, 1, 1, 1), (torch.bfloat16, 2, 3, 9)])
def test_head_norm_rotary(kind, d, sections, pairs, dtype, n, hq, hk):
    from uncrtaints_amd.src.backbones.packed_attention import HeadNormRotary
    q, k = (t.detach().requires_grad_() for t in _views(kind, n, hq, hk, d, dtype, 7))
    pos = _positions(n, len(sections), torch.int32, 8)
    places = _places(d, sections, pairs)
    m = HeadNormRotary(d, rotary=_module(d, sections, pairs), eps=1e-5).to(DEV)
    with torch.no_grad():
        m.q_weight.copy_(1 + 0.2 * torch.randn(d, generator=_gen(9)))
        m.k_weight.copy_(1 + 0.2 * torch.randn(d, generator=_gen(10)))
    gq, gk = _views(kind, n, hq, hk, d, dtype, 11)
    yq, yk = m(q, k, pos.to(DEV))
    dq, dk, dwq, dwk = torch.autograd.grad((yq, yk), (q, k, m.q_weight, m.k_weight), (gq, gk))
    for name, x, w, y, g, dx, dw in (("q", q, m.q_weight, yq, gq, dq, dwq), ("k", k, m.k_weight, yk, gk, dk, dwk)):
        x64, w64 = x.detach().cpu().double().requires_grad_(), w.detach().cpu().double().requires_grad_()
        z = _norm64(x64, w64, 1e-5)
        ref = _rotate64(z, pos, places)
        assert y.dtype == dtype and dx.dtype == dtype and dw.dtype == torch.float32
        size = _pair_size(z.detach(), places) + z.detach().abs()
        _check(name, y, ref.detach(), 28 * U * size + _half(dtype) * ref.detach().abs())
        g64 = g.cpu().double()
        rx, rw = torch.autograd.grad(ref, (x64, w64), g64)
        u = _rotate64(g64, pos, places, -1.0)
        usize = _pair_size(g64, places) + g64.abs()
        with torch.no_grad():
            r = 1.0 / (x64.square().mean(-1, keepdim=True) + 1e-5).sqrt()
            terms = r * w64.abs() * usize + x64.abs() * r ** 3 * (w64 * x64).abs().mul(usize).mean(-1, keepdim=True)
            _check("d" + name, dx, rx, 64 * U * terms + _half(dtype) * rx.abs())
            _check("dw" + name, dw, rw, (64 + 512) * U * (usize * x64.abs() * r).sum((0, 1)) + U * rw.abs())
        del u


@gpu
def test_head_norm_rotary_many_tokens_and_differences():
    """Several tiles per block in the gradient, and the gradient against differences of the kernel's own forward along one direction:
    (f(x + t v) - f(x - t v)) / 2t with t = 1e-2 is off by t^2 / 6 |f'''| ~ 2e-5 and by the forward's noise 28u sum |g y| / t; the sums run
    over 5000 x 6 x 32 values, so both stay below 2e-4 of sqrt(sum) -- held to 1e-3 of the slope's scale."""
    from uncrtaints_amd.src.backbones.packed_attention import HeadNormRotary
    n, d = 5000, 32
    m = HeadNormRotary(d, rotary=_module(d, ((16, 1000.0), (16, 50.0)), "halves")).to(DEV)
    x = torch.randn(n, 6, d, generator=_gen(20)).to(DEV)
    g, v = torch.randn(n, 6, d, generator=_gen(21)).to(DEV), torch.randn(n, 6, d, generator=_gen(22)).to(DEV)
    pos = _positions(n, 2, torch.int32, 23).to(DEV)

    def f(z, wq, wk):
        with torch.no_grad():
            m.q_weight.copy_(wq), m.k_weight.copy_(wk)
            yq, yk = m(z[:, :4], z[:, 4:], pos)
        return (yq.double() * g[:, :4].double()).sum() + (yk.double() * g[:, 4:].double()).sum()

    w0, vw = torch.ones(2, d, device=DEV), torch.randn(2, d, generator=_gen(24)).to(DEV)
    xr = x.clone().requires_grad_()
    yq, yk = m(xr[:, :4], xr[:, 4:], pos)
    dx, dwq, dwk = torch.autograd.grad((yq, yk), (xr, m.q_weight, m.k_weight), (g[:, :4], g[:, 4:]))
    t = 1e-2
    for slope, diff in (((dx.double() * v.double()).sum(), f(x + t * v, *w0) - f(x - t * v, *w0)),
                        ((dwq.double() * vw[0].double()).sum() + (dwk.double() * vw[1].double()).sum(),
                         f(x, *(w0 + t * vw)) - f(x, *(w0 - t * vw)))):
        assert abs(float(slope - diff / (2 * t))) < 1e-3 * math.sqrt(n * 6 * d), (float(slope), float(diff / (2 * t)))


@gpu
def test_head_norm_without_rotary_zero_rows_and_no_tokens():
    from uncrtaints_amd.src.backbones.packed_attention import HeadNormRotary
    m = HeadNormRotary(24, eps=1e-6).to(DEV)
    q = torch.randn(5, 2, 24, generator=_gen(30))
    q[1] = 0.0                                                # a row of zeros: 0 * 1/sqrt(eps), finite gradient
    qd = q.to(DEV).requires_grad_()
    y, yk = m(qd, qd[:, :1])
    ref = _norm64(q.double(), 1.0, 1e-6)
    _check("q", y, ref, 29 * U * ref.abs())
    dx, = torch.autograd.grad(y, qd, torch.ones_like(y))
    assert torch.isfinite(dx).all() and float((dx[1].cpu() - 1e3).abs().max()) < 1e3 * 64 * U
    e = torch.empty(0, 2, 24, device=DEV, requires_grad=True)
    y, yk = m(e, e[:, :1])
    assert y.shape == (0, 2, 24)
    grads = torch.autograd.grad((y, yk), (e, m.q_weight, m.k_weight), (torch.empty_like(y), torch.empty_like(yk)))
    assert grads[0].shape == (0, 2, 24) and float(grads[1].abs().max()) == 0.0 and float(grads[2].abs().max()) == 0.0


@gpu
def test_rotary_and_norms_replay_from_a_graph_and_run_on_a_side_stream():
    from uncrtaints_amd.src.backbones.packed_attention import HeadNormRotary
    m = HeadNormRotary(64, rotary=_module(64, SHAPES[0][1], "halves")).to(DEV)
    q, pos = torch.randn(40, 6, 64, generator=_gen(40)).to(DEV).to(torch.bfloat16), _positions(40, 3, torch.int32, 41).to(DEV)
    g = torch.randn(40, 6, 64, generator=_gen(42)).to(DEV).to(torch.bfloat16)
    qr = q.clone().requires_grad_()

    def step():
        a, b = m(qr[:, :4], qr[:, 4:], pos)
        return (a.detach(), b.detach()) + torch.autograd.grad((a, b), (qr, m.q_weight, m.k_weight), (g[:, :4], g[:, 4:]))

    eager = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [t.detach().clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        with torch.no_grad():
            qr.copy_(q if i != 1 else -q)
        graph.replay()
        torch.cuda.synchronize()
        if i != 1:
            for a, b, c in zip(eager, other, held):
                assert torch.equal(a, b) and torch.equal(a, c)
        else:
            assert torch.equal(held[0], -eager[0])


def test_rotary_and_norms_refuse():
    from uncrtaints_amd.src.backbones.packed_attention import HeadNormRotary
    from uncrtaints_amd.src.backbones.positional_encoding import RotaryAxes
    for kw in (dict(d=7), dict(d=258), dict(d=8, sections=(3, 5)), dict(d=8, sections=(6, 4)), dict(d=16, sections=(2,) * 5),
               dict(d=8, pairs="thirds"), dict(d=8, T=0.0), dict(d=8, sections=(4, 4), T=(1.0,)), dict(d=8, T=float("nan"))):
        with pytest.raises(ValueError):
            RotaryAxes(**kw)
    r = RotaryAxes(8, sections=(4, 4))
    x, pos = torch.zeros(3, 2, 8), torch.zeros(3, 2)
    with pytest.raises(ValueError):
        r(torch.zeros(3, 2, 10), pos)
    with pytest.raises(RuntimeError, match="cuda device"):
        r(x, pos)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        r(x.half(), pos)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        r.plan(pos.half(), (3,), pos.device)
    with pytest.raises(ValueError, match="expected"):
        r.plan(torch.zeros(4, 2), (3,), pos.device)
    with pytest.raises(ValueError, match="no gradient"):
        r.plan(torch.zeros(3, 2, requires_grad=True), (3,), pos.device)
    for kw in (dict(d=7), dict(d=16, rotary=r), dict(d=8, eps=-1.0), dict(d=8, eps=float("nan"))):
        with pytest.raises(ValueError):
            HeadNormRotary(**kw)
    m = HeadNormRotary(8, rotary=r)
    with pytest.raises(ValueError, match="positions"):
        m(x, x)
    with pytest.raises(ValueError, match="tokens"):
        m(x, torch.zeros(4, 2, 8), pos)
    with pytest.raises(RuntimeError, match="float32"):
        HeadNormRotary(8).bfloat16()(x, x)
    with pytest.raises(RuntimeError, match="but q is"):
        m(x, x.bfloat16(), pos)
    with pytest.raises(RuntimeError, match="cuda device"):
        m(x, x, pos)


def test_rotary_entry_points_refuse_bad_geometry():
    """The C entries return their error codes for arguments no launch may see (nothing is enqueued: there is no GPU here)."""
    from uncrtaints_amd import hip_backend as hb
    fn = hb.lib().fn["uncr_rotary_axes"]
    ok = dict(x=16, x_ts=16, x_hs=8, y=16, y_ts=16, y_hs=8, pos=16, pos_dt=0, n_axes=2, s0=4, s1=4, s2=0, s3=0, turns=16, nb=0, inv=0, N=0, H=2,
              D=8, act=0, stream=None)
    call = lambda **kw: fn(*{**ok, **kw}.values())
    assert call() == 0                                         # no tokens: nothing to launch
    for kw in (dict(D=7), dict(D=258), dict(D=0), dict(N=-1), dict(H=0), dict(s0=3), dict(s0=-2), dict(s1=8), dict(s2=2), dict(n_axes=5),
               dict(n_axes=-1), dict(pos_dt=4), dict(act=2), dict(N=3, pos=None), dict(N=3, turns=None), dict(N=3, x=None), dict(N=3, y=None)):
        assert call(**kw) < 0, kw


@gpu
def test_positions_changed_before_the_backward_are_an_error():
    from uncrtaints_amd.src.backbones.packed_attention import HeadNormRotary
    r = _module(64, SHAPES[0][1], "halves").to(DEV)
    m = HeadNormRotary(64, rotary=r).to(DEV)
    x, pos = torch.randn(5, 6, 64, generator=_gen(50)).to(DEV).requires_grad_(), _positions(5, 3, torch.int32, 51).to(DEV)
    ys = r(x, pos), m(x, x, pos)[0]
    pos += 1
    for y in ys:
        with pytest.raises(RuntimeError, match="inplace"):
            y.sum().backward()


def test_more_tokens_than_are_counted_are_refused():
    from uncrtaints_amd import engine as E
    from uncrtaints_amd import hip_backend as hb
    with pytest.raises(RuntimeError, match="31 bits"):
        E.rotary_axes(torch.zeros(1, 1, 2).expand(2 ** 31, 1, 2), E.RotaryPlan())
    ok = dict(x=16, x_ts=256, x_hs=256, y=16, y_ts=256, y_hs=256, pos=16, pos_dt=0, n_axes=1, s0=256, s1=0, s2=0, s3=0, turns=16, nb=0, inv=0, N=2 ** 31 - 1,
              H=1, D=256, act=0, stream=None)
    fn = hb.lib().fn["uncr_rotary_axes"]
    assert fn(*ok.values()) == fn(*{**ok, "H": 0}.values()) < 0


def _norm_gradients(q, k, m, eps):
    """The norms' gradients (no rotation) against the formula's in 64 bits, within this file's bounds: u is dy itself here."""
    gq, gk = torch.randn(q.shape, generator=_gen(61)).to(q.dtype), torch.randn(k.shape, generator=_gen(62)).to(k.dtype)
    qd, kd = q.to(DEV).requires_grad_(), k.to(DEV).requires_grad_()
    grads = torch.autograd.grad(m(qd, kd), (qd, kd, m.q_weight, m.k_weight), (gq.to(DEV), gk.to(DEV)))
    for name, x, g, w, dx, dw in (("q", q, gq, m.q_weight, grads[0], grads[2]), ("k", k, gk, m.k_weight, grads[1], grads[3])):
        x, g, w = x.double(), g.double(), w.detach().cpu().double()
        r = 1.0 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
        xh = x * r
        ref = r * (w * g - xh * (w * g * xh).mean(-1, keepdim=True))
        _check("d" + name, dx, ref, 64 * U * r * ((w * g).abs() + xh.abs() * (w * g * xh).abs().mean(-1, keepdim=True)) + _half(q.dtype) * ref.abs())
        _check("dw" + name, dw, (g * xh).sum((0, 1)), (64 + 512) * U * (g * xh).abs().sum((0, 1)))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 3, 53])
@pytest.mark.parametrize("d,hq,hk", [(128, 8, 2), (16, 1, 1), (64, 3, 2), (6, 2, 1)])
def test_norm_gradients_without_eps_where_the_last_tokens_fill_no_wave(d, hq, hk, n, dtype):
    from uncrtaints_amd.src.backbones.packed_attention import HeadNormRotary
    q, k = (torch.randn(n, h, d, generator=_gen(70 + h)).to(dtype) for h in (hq, hk))
    _norm_gradients(q, k, HeadNormRotary(d, eps=0.0).to(DEV), 0.0)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,hq,hk", [(64, 4, 2), (40, 3, 1), (202, 2, 2), (256, 8, 1)])
def test_norm_gradients_of_very_large_and_very_small_rows(d, hq, hk, dtype):
    from uncrtaints_amd.src.backbones.packed_attention import HeadNormRotary
    scale = torch.tensor([1.0, 1e15, 1e16, 1e17, 1e-6, 1e-10, 1e-13, 1e-17]).view(8, 1, 1)
    q, k = (scale * torch.randn(8, h, d, generator=_gen(60 + h))  for h in (hq, hk))
    q, k = q.to(dtype), k.to(dtype)
    m = HeadNormRotary(d, eps=0.0).to(DEV)
    _norm_gradients(q, k, m, 0.0)
    m = HeadNormRotary(d, eps=1e-30).to(DEV)
    q[2] = 0.0
    _norm_gradients(q, k, m, 1e-30)


@gpu
def test_norm_gradients_of_the_most_tokens_that_are_counted():
    """Close to 2^31 rows of one head of 2 values, all the same row; a lane adds the weights' terms of 2^31 / (64 tokens x 4096 waves) = 8192 of them
    one after the other in fp32."""
    from uncrtaints_amd import engine as E
    n = 2 ** 31 - 1
    x, g = (torch.tensor(v, dtype=torch.bfloat16, device=DEV).view(1, 1, 2).expand(n, 1, 2) for v in ([3.0, 4.0], [1.0, -2.0]))
    w = torch.tensor([1.0, 0.5], device=DEV)
    dq, dk, dwq, dwk = E.headnorm_rotary_backward(g, g, x, x, w, w, 0.0, E.RotaryPlan())
    x64, g64, w64 = (t.double().cpu() for t in (x[0, 0], g[0, 0], w))
    r = 1.0 / x64.square().mean().sqrt()
    xh = x64 * r
    ref = r * (w64 * g64 - xh * (w64 * g64 * xh).mean())
    for dx in (dq, dk):
        _check("dx", dx[0, 0], ref, 64 * U * r * 10 + _half(torch.bfloat16) * ref.abs())
        rows = dx.view(-1).view(torch.int32)
        assert bool((rows == rows[0]).all())
    for dw in (dwq, dwk):
        assert bool(((dw.double().cpu() / n - g64 * xh).abs() <= (64 + 8192) * U * (g64 * xh).abs()).all())


def test_norm_gradients_refuse_tiles_that_are_not_counted():
    from uncrtaints_amd import hip_backend as hb
    name = "uncr_headnorm_rotary_bwd"
    ok = dict.fromkeys([n for _, n in hb.parse_header()[name]], 0)
    ok.update(q=20, k=20, gq=20, gk=20, dq=20, dk=20, wq=16, wk=16, part=16, dwq=16, dwk=16, pos=None, turns=None, eps=1.0, N=2 ** 31 - 1, Hq=1, Hk=1, D=256,
              stream=None)          # rows that start at no vector boundary: a wave takes one token at a time
    fn = hb.lib().fn[name]
    assert fn(*ok.values()) == fn(*{**ok, "Hq": 0}.values()) < 0


def test_forward_mode_tangents_are_refused():
    """A result without a tangent would pass for one whose derivative is 0.  Refused before anything is launched (no GPU here), through dual tensors
    and through functional transforms, in the forward and in a backward whose incoming gradient is dual."""
    import torch.autograd.forward_ad as fw
    from uncrtaints_amd import engine as E
    from uncrtaints_amd.src.backbones.packed_attention import HeadNormRotary, PackedAttention, pack_offsets
    from uncrtaints_amd.src.backbones.positional_encoding import RotaryAxes
    x, pos, off, w = torch.ones(3, 2, 8), torch.zeros(3, 2), pack_offsets([3], "cpu"), torch.ones(8)
    r = RotaryAxes(8, sections=(4, 4))
    norm, plain, attend = HeadNormRotary(8, rotary=r), HeadNormRotary(8), PackedAttention()
    calls = [lambda t: r(t, pos), lambda t: norm(t, x, pos), lambda t: norm(x, t, pos), lambda t: plain(x, t), lambda t: attend(t, x, x, off),
             lambda t: attend(x, t, x, off), lambda t: attend(x, x, t, off), lambda t: E.rotary_axes(t, E.RotaryPlan(), inverse=True),
             lambda t: E.headnorm_rotary_backward(t, x, x, x, w, w, 1e-6, E.RotaryPlan()),
             lambda t: E.headnorm_rotary_backward(x, t, x, x, w, w, 1e-6, E.RotaryPlan()),
             lambda t: E.packed_attention_backward(t, x, x, x, x, w, off, off, None, 1.0, False)]
    for call in calls:
        for grad in (True, False):
            with torch.set_grad_enabled(grad), fw.dual_level(), pytest.raises(NotImplementedError, match="tangent"):
                call(fw.make_dual(x, x))
            with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="tangent"):
                torch.func.jvp(call, (x,), (x,))
    with fw.dual_level():
        with pytest.raises(NotImplementedError, match="positions"):
            r.plan(fw.make_dual(pos, pos), (3,), pos.device)
        with pytest.raises(RuntimeError, match="cuda device"):          # a level without tangents refuses nothing
            r(x, pos)


@gpu
def test_forward_mode_tangents_are_refused_on_the_gpu():
    import torch.autograd.forward_ad as fw
    from uncrtaints_amd.src.backbones.packed_attention import HeadNormRotary, PackedAttention, pack_offsets
    x, off = torch.ones(3, 2, 8, device=DEV), pack_offsets([3], DEV)
    leaf = x.clone().requires_grad_()
    r = _module(8, ((8, 100.0),), "halves").to(DEV)
    pos = torch.ones(3, 1, device=DEV)
    attend, norm = PackedAttention(), HeadNormRotary(8, rotary=r).to(DEV)
    with fw.dual_level():
        dual = fw.make_dual(x, x)
        for call in (lambda t: r(t, pos), lambda t: norm(t, x, pos), lambda t: attend(x, x, t, off)):
            with pytest.raises(NotImplementedError, match="tangent"):
                call(dual)
        for y in (r(leaf, pos), norm(leaf, x, pos)[0], attend(leaf, x, x, off)):
            with pytest.raises(NotImplementedError, match="tangent"):
                torch.autograd.grad(y, leaf, dual)
        del norm.k_weight
        norm.k_weight = fw.make_dual(torch.ones(8, device=DEV), torch.ones(8, device=DEV))
        with pytest.raises(NotImplementedError, match="k_weight"):
            norm(x, x, pos)


def test_norm_weights_of_another_size_are_refused():
    """A replaced parameter: the kernels read d values of each."""
    from uncrtaints_amd.src.backbones.packed_attention import HeadNormRotary
    x = torch.zeros(3, 2, 8)
    for name in ("q_weight", "k_weight"):
        for w in (torch.ones(7), torch.ones(1), torch.ones(()), torch.ones(9), torch.ones(2, 8), torch.ones(0)):
            m = HeadNormRotary(8)
            setattr(m, name, torch.nn.Parameter(w))
            with pytest.raises(ValueError, match=name):
                m(x, x)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,sections,pairs", [(202, ((66, 10000.0), (70, 100.0), (66, 100.0)), "neighbours"), (250, ((100, 10000.0), (90, 20.0)), "neighbours"),
                                              (44, ((12, 100.0), (20, 50.0)), "halves"), (44, ((12, 100.0), (20, 50.0)), "neighbours")])
def test_pairs_that_fill_no_vector(d, sections, pairs, dtype):
    """More neighbours than a wave has lanes, one at a time; two pairs per lane"""
    test_rotary_axes(d, sections, pairs, dtype, 37, 5)
    for kind in ("plain", "odd_start"):
        test_head_norm_rotary(kind, d, sections, pairs, dtype, 53, 6, 2)
