"""Rotary positions over several axes and differential attention on a real MI355X, against their definitions in 64 bits.

Tolerances are worst cases, worked out element by element from the roundings the kernels make (``_reference`` carries them along with
the values): U = 2^-8 of the value for one rounding to bf16 -- of P (forward), dS and A = P1 - lam P2 (gradient), of the saved o, o2, of dO
behind the norm, of every bf16 result -- and F = 2^-14 for everything held in 32 bits (sums of at most a few thousand terms, exp2 and the
score in its exponent: |score| <= 60 at 2^-23 a step).  They are a few times what random rounding gives, so well-conditioned cases are held to
a 2-norm as well: five independent roundings of at most U / sqrt(3) each are 0.9 %, doubled for the difference of two maps = 2 %."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
U, F = 2.0 ** -8, 2.0 ** -14
EPS = 1e-5


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from mofo_amd import _lib
    _lib.load()
    return torch.device("cuda:0")


def _rand(shape, dev, seed, scale=1.0, dtype=BF16):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(dev)


def _rel(a, b):
    a, b = a.double().flatten(), b.double().flatten()
    return float((a - b).norm() / (b.norm() + 1e-300))


def _within(got, want, tol, what):
    d = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all(), f"{what}: not finite"
    bad = d > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / tol.clamp_min(1e-300)).max()):.3g} times its bound"


# ------------------------------------------------------------------------------------------------ rotary positions
def _rope64(x, heads, hd, sections, place, base, interleaved, sign=1.0):
    M = x.shape[0]
    P = sum(sections)
    cols = [place[:, a].double() * (base ** (-i / n)) for a, n in enumerate(sections) for i in range(n)]
    ang = torch.stack(cols, 1)[:, None] * sign
    v = x.double().reshape(M, heads, hd)
    y = v.clone()
    i = torch.arange(P, device=x.device)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + P)
    a, b = v[..., lo], v[..., hi]
    y[..., lo], y[..., hi] = a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()
    size = v.abs()
    size[..., lo] = size[..., hi] = (a.abs() + b.abs())
    return y.reshape(M, heads * hd), size.reshape(M, heads * hd)


ROPE = [  # M, heads, head_dim, sections, interleaved, token ids?, dtype
    (1, 1, 16, (3, 2, 3), False, True, BF16), (1, 24, 64, (8, 12, 12), False, True, BF16), (160, 24, 64, (8, 12, 12), False, True, BF16),
    (157, 12, 64, (4, 10, 10), True, True, BF16), (2049, 3, 80, (1, 18, 21), False, False, BF16), (8195, 2, 128, (38, 14, 12), True, False, BF16),
    (333, 5, 160, (40, 18, 6), True, False, F32), (2050, 2, 96, (39, 2, 7), False, False, F32), (77, 1, 256, (128,), False, False, F32),
    (77, 2, 64, (8, 8, 8, 8), False, False, BF16), (31, 2, 64, (0, 16, 0), True, True, BF16)]


@pytest.mark.parametrize("M,heads,hd,sections,interleaved,tokens,dtype", ROPE)
def test_rope_axes_forward_and_gradient(dev, M, heads, hd, sections, interleaved, tokens, dtype):
    from mofo_amd import ops
    W, P = heads * hd, sum(sections)
    extra = 40 if dtype == BF16 else 20                               # columns right of the view: not to be touched
    buf = _rand((M, W + extra), dev, 1, 1.0, dtype)
    x = buf[:, :W]
    g = torch.Generator().manual_seed(3)
    if tokens:
        tok = torch.randint(0, 1568, (M,), generator=g).to(I32).to(dev)
        place = torch.stack([tok // 196, tok // 14 % 14, tok % 14], 1)
        where = dict(tok_idx=tok, grid=(8, 14, 14))
    else:
        place = torch.randint(-50, 5000, (M, len(sections)), generator=g).to(I32).to(dev)
        where = dict(pos=place.contiguous())
    freqs = ops.rope_freqs(sections, 10000.0, dev)
    obuf = torch.full((M + 2, W + extra), 7.0, dtype=dtype, device=dev)
    before = buf.clone()
    ops.rope_axes_fwd(x, heads, hd, sections, freqs, obuf[:M, :W], interleaved=interleaved, **where)
    want, size = _rope64(x, heads, hd, sections, place, 10000.0, interleaved)
    tol = size * 2.0 ** -20 + (U * want.abs() if dtype == BF16 else 0)    # cos, sin and two products in f32: 8 units of 2^-23
    _within(obuf[:M, :W], want, tol + 1e-30, "rope")
    assert torch.equal(buf, before) and bool((obuf[M:] == 7).all()) and bool((obuf[:, W:] == 7).all())
    cover = torch.arange(hd, device=dev).expand(heads, hd).reshape(-1) >= 2 * P
    assert torch.equal(obuf[:M, :W][:, cover], x[:, cover])              # columns that no pair covers: copied
    # in place, the same bits
    y = buf[:, :W]
    ops.rope_axes_fwd(y, heads, hd, sections, freqs, y, interleaved=interleaved, **where)
    assert torch.equal(buf[:, :W], obuf[:M, :W]) and torch.equal(buf[:, W:], before[:, W:])
    # gradient: the formula's, and <dout, R x> = <R' dout, x> through differences of a linear map
    dout = _rand((M, W), dev, 5, 1.0, dtype)
    dx = torch.empty_like(dout)
    ops.rope_axes_bwd(dout, heads, hd, sections, freqs, dx, interleaved=interleaved, **where)
    want, size = _rope64(dout, heads, hd, sections, place, 10000.0, interleaved, -1.0)
    _within(dx, want, size * 2.0 ** -20 + (U * want.abs() if dtype == BF16 else 0) + 1e-30, "rope gradient")
    step, h = _rand((M, W), dev, 6, 1.0, F64), 1e-3
    diff = (_rope64(before[:, :W].double() + h * step, heads, hd, sections, place, 10000.0, interleaved)[0]
            - _rope64(before[:, :W].double() - h * step, heads, hd, sections, place, 10000.0, interleaved)[0]) / (2 * h)
    lhs, rhs = (dout.double() * diff).sum(), (dx.double() * step).sum()
    assert abs(float(lhs - rhs)) <= float((step.abs() * (size * 2.0 ** -20 + U * want.abs())).sum())


def test_rope_axes_far_positions(dev):
    """angles are formed in 64 bits: f32 products would be off by radians at these places"""
    from mofo_amd import ops
    place = torch.tensor([[2 ** 31 - 1, 0, 0], [-2 ** 31, 1, 2], [123456789, 7, 9], [1 << 24, 13, 13]], dtype=I32, device=dev)
    x = _rand((4, 64), dev, 2, 1.0, F32)
    out = torch.empty_like(x)
    ops.rope_axes_fwd(x, 1, 64, (8, 12, 12), ops.rope_freqs((8, 12, 12), 10000.0, dev), out, pos=place)
    want, size = _rope64(x, 1, 64, (8, 12, 12), place, 10000.0, False)
    _within(out, want, size * (2.0 ** -20 + 2.0 ** 31 * 2.0 ** -51), "far")   # the f64 angle itself: 2^31 at 2^-52 a side


def test_rope_axes_offsets_beyond_32_bits(dev):
    """rows 2^20 elements apart: the last ones start behind element 2^31; in place the same bits"""
    from mofo_amd import ops
    M, big = 2200, torch.empty(2200, 1 << 20, dtype=BF16, device=dev)
    x = _rand((M, 128), dev, 3)
    big[:, 64:192] = x
    pos, freqs = torch.arange(3 * M, dtype=I32, device=dev).reshape(M, 3), ops.rope_freqs((8, 12, 12), device=dev)
    want, out = torch.empty_like(x), torch.empty_like(x)
    ops.rope_axes_fwd(x, 2, 64, (8, 12, 12), freqs, want, pos=pos)
    ops.rope_axes_fwd(big[:, 64:192], 2, 64, (8, 12, 12), freqs, out, pos=pos)
    assert torch.equal(out, want)
    ops.rope_axes_fwd(big[:, 64:192], 2, 64, (8, 12, 12), freqs, big[:, 64:192], pos=pos)
    assert torch.equal(big[:, 64:192], want)


def test_rope_axes_no_rows(dev):
    from mofo_amd import ops
    x = torch.empty(0, 64, dtype=BF16, device=dev)
    ops.rope_axes_fwd(x, 1, 64, (8, 12, 12), ops.rope_freqs((8, 12, 12), device=dev), torch.empty_like(x), pos=torch.empty(0, 3, dtype=I32, device=dev))


def test_rope_axes_refusals(dev):
    from mofo_amd import ops
    x, f = _rand((6, 128), dev, 1), ops.rope_freqs((8, 12, 12), device=dev)
    tok = torch.zeros(6, dtype=I32, device=dev)
    ok = dict(tok_idx=tok, grid=(8, 14, 14))
    out = torch.empty_like(x)
    for bad, err in [
            (lambda: ops.rope_axes_fwd(x.half(), 2, 64, (8, 12, 12), f, out, **ok), TypeError),
            (lambda: ops.rope_axes_fwd(x, 2, 64, (8, 12, 12), f, out.float(), **ok), TypeError),
            (lambda: ops.rope_axes_fwd(x, 2, 64, (8, 12, 12), f.float(), out, **ok), TypeError),
            (lambda: ops.rope_axes_fwd(x, 3, 64, (8, 12, 12), f, out, **ok), ValueError),
            (lambda: ops.rope_axes_fwd(x, 2, 64, (8, 12, 13), f, out, **ok), ValueError),
            (lambda: ops.rope_axes_fwd(x, 4, 32, (8, 12, 12), f, out, **ok), ValueError),
            (lambda: ops.rope_axes_fwd(x, 2, 64, (8, 12, 12), f, out), ValueError),
            (lambda: ops.rope_axes_fwd(x, 2, 64, (8, 12, 12), f, out, pos=torch.zeros(6, 2, dtype=I32, device=dev)), ValueError),
            (lambda: ops.rope_axes_fwd(x, 2, 64, (8, 12, 12), f, out, tok_idx=tok), ValueError),
            (lambda: ops.rope_axes_fwd(x, 2, 64, (16, 16), f, out, **ok), ValueError),
            (lambda: ops.rope_axes_fwd(x, 2, 64, (8, 12, 12), f, out, tok_idx=tok[:5], grid=(8, 14, 14)), ValueError),
            (lambda: ops.rope_axes_fwd(x[:, 1:65], 1, 64, (8, 12, 12), f, out[:, :64], **ok), RuntimeError),
            (lambda: ops.rope_axes_fwd(x[:, :64], 1, 64, (8, 12, 12), f, x[:, 16:80], **ok), RuntimeError),
            (lambda: ops.rope_axes_fwd(x.cpu(), 2, 64, (8, 12, 12), f, out, **ok), ValueError)]:
        with pytest.raises(err):
            bad()
    # column ranges of one buffer that do not meet are two tensors
    ops.rope_axes_fwd(x[:, :64], 1, 64, (8, 12, 12), f, x[:, 64:], **ok)


# ------------------------------------------------------------------------------------------------ differential attention
def _heads(t, B, n, parts):
    return t.double().reshape(B, -1, n, parts, t.shape[1] // (n * parts)).permute(0, 2, 3, 1, 4)


def _limits(B, Nq, Nk, kv_len, causal, dev):
    ln = (torch.full((B,), Nk, device=dev) if kv_len is None else kv_len.long().clamp(0, Nk))[:, None].expand(B, Nq)
    i = torch.arange(Nq, device=dev)[None]
    return ln if causal == 0 else torch.minimum(ln, (i + 1 if causal == 1 else i + 1 + ln - Nq).clamp_min(0))


def _mean_sq(t):
    return t.square().mean(-1, keepdim=True).sqrt()


def _reference(q, k, v, B, H, Hkv, scale, lam, lam_init, gamma, out_scale, kv_len, causal, dout=None, grad_u=U):
    """{name: (value, bound)} in 64 bits, by the formulas (no autograd)"""
    dev = q.device
    Nq, Nk, G = q.shape[0] // B, k.shape[0] // B, H // Hkv
    Q, K, V = _heads(q, B, H, 2), _heads(k, B, Hkv, 2).repeat_interleave(G, 1), _heads(v, B, Hkv, 1).squeeze(2).repeat_interleave(G, 1)
    lim = _limits(B, Nq, Nk, kv_len, causal, dev)
    see = (torch.arange(Nk, device=dev) < lim[..., None])[:, None, None]
    ln = torch.full((B,), Nk, device=dev) if kv_len is None else kv_len.long().clamp(0, Nk)
    there = (torch.arange(Nk, device=dev) < ln[:, None])[:, None, :, None]
    K, V = torch.where(there[:, :, None], K, 0.0), torch.where(there, V, 0.0)
    Q = torch.where((lim > 0)[:, None, None, :, None], Q, 0.0)
    S = torch.where(see, Q @ K.transpose(-1, -2) * scale, -math.inf)
    top = S.amax(-1, keepdim=True).clamp_min(-1e300)
    E = (S - top).exp()
    Z = E.sum(-1, keepdim=True)
    P = E / torch.where(Z > 0, Z, 1.0)
    l = lam.double()
    e1, e2 = (l[0] * l[1]).sum(-1).exp(), (l[2] * l[3]).sum(-1).exp()
    w = (e1 - e2 + lam_init).expand(H)[None, :, None, None]
    A = P[:, :, 0] - w * P[:, :, 1]
    o1, o2 = P[:, :, 0] @ V, P[:, :, 1] @ V
    b1, b2 = (U + F) * (P[:, :, 0] @ V.abs()), (U + F) * (P[:, :, 1] @ V.abs())
    o, bo = o1 - w * o2, b1 + w.abs() * b2
    rows = lambda t: t.transpose(1, 2).reshape(B * t.shape[2], -1)  # noqa: E731
    if gamma is None:
        y, by = o, bo
    else:
        r = (o.square().mean(-1, keepdim=True) + EPS).rsqrt()
        gs = gamma.double() * out_scale
        y, by = o * r * gs, gs.abs() * (bo * r + o.abs() * r * r * _mean_sq(bo))
    res = {"out": (rows(y), rows(by + U * (y.abs() + by) + F * y.abs())), "o": (rows(o), rows(bo + U * (o.abs() + bo))),
           "o2": (rows(o2), rows(b2 + U * (o2.abs() + b2)))}
    lse = (top + Z.log()).squeeze(-1).permute(2, 0, 1, 3) / math.log(2.0)
    res["lse2"] = (lse, F * (1 + lse.abs()))
    if dout is None:
        return res
    dy = torch.where((lim > 0)[:, None, :, None], _heads(dout, B, H, 1).squeeze(2), 0.0)
    so, so2 = bo + U * (o.abs() + bo), b2 + U * (o2.abs() + b2)             # bounds of the saved o, o2
    if gamma is None:
        d, bd = dy, torch.zeros_like(dy)
        br = bd
    else:
        x, g = o * r, dy * gs
        m = (g * x).mean(-1, keepdim=True)
        rel = _mean_sq(so) * r
        bx = so * r + x.abs() * rel
        d = r * (g - x * m)
        bd = rel * d.abs() + r * (bx * m.abs() + x.abs() * (g.abs() * bx).mean(-1, keepdim=True)) + F * r * (g.abs() + (x * m).abs())
        br = bd + U * (d.abs() + bd)
        dg = (dy * x * out_scale).sum((0, 1, 2))
        res["dgamma"] = (dg, (dy.abs() * bx * out_scale).sum((0, 1, 2)) + grad_u * dg.abs() + F * (dy * x).abs().sum((0, 1, 2)))
    dA, bA = d @ V.transpose(-1, -2), br @ V.abs().transpose(-1, -2) + F * (d.abs() @ V.abs().transpose(-1, -2))
    dv = A.transpose(-1, -2) @ d
    bdv = (U * A.abs() + F * (P[:, :, 0] + w.abs() * P[:, :, 1])).transpose(-1, -2) @ (d.abs() + br) + A.abs().transpose(-1, -2) @ br
    s1 = so + w.abs() * so2                                                  # bound of o1 = o + lam o2
    dS, bS = [], []
    for n, (on, sn, wt) in enumerate(((o1, s1, torch.ones_like(w)), (o2, so2, -w))):
        dn = (d * on).sum(-1, keepdim=True)
        bn = (br * on.abs() + (d.abs() + br) * sn).sum(-1, keepdim=True) + F * (d * on).abs().sum(-1, keepdim=True)
        t = P[:, :, n] * (dA - dn) * wt
        bt = P[:, :, n] * (bA + bn) * wt.abs() + F * P[:, :, n] * (dA.abs() + dn.abs()) * wt.abs()
        dS.append(t)
        bS.append(bt + U * (t.abs() + bt))
        if n == 1:
            dl = -dn.squeeze(-1).sum((0, 2))
            bl = (bd * on.abs() + (d.abs() + bd) * sn).sum((0, 2, 3)) + F * (d * on).abs().sum((0, 2, 3))
    dS, bS = torch.stack(dS, 2), torch.stack(bS, 2)
    dq, bq = dS @ K * scale, bS @ K.abs() * scale
    dk, bk = dS.transpose(-1, -2) @ Q * scale, bS.transpose(-1, -2) @ Q.abs() * scale
    share = lambda t: t.reshape(B, Hkv, G, *t.shape[2:]).sum(2)  # noqa: E731
    flat = lambda t: rows(t.transpose(2, 3).flatten(3))  # noqa: E731
    for n, t, bt in (("dq", flat(dq), flat(bq)), ("dk", flat(share(dk)), flat(share(bk))), ("dv", rows(share(dv)), rows(share(bdv)))):
        res[n] = (t, bt + U * (t.abs() + bt) + F * t.abs())
    if lam.shape[1] == 1:
        dl, bl = dl.sum(0, keepdim=True), bl.sum(0, keepdim=True)
    d1, d2, c1, c2 = dl * e1, -dl * e2, bl * e1, bl * e2
    dlam = torch.stack([d1[:, None] * l[1], d1[:, None] * l[0], d2[:, None] * l[3], d2[:, None] * l[2]])
    blam = torch.stack([c1[:, None] * l[1].abs(), c1[:, None] * l[0].abs(), c2[:, None] * l[3].abs(), c2[:, None] * l[2].abs()])
    res["dlam"] = (dlam, blam + (grad_u + F) * dlam.abs())
    return res


TINY = 2.0 ** -126


def _case(dev, B, Nq, Nk, H, Hkv, norm, lam_heads=None, params=BF16, seed=0, sharp=1.0, lam_scale=0.1):
    """inputs as column ranges of wider buffers with guard columns; (q, k, v, lam, gamma, dout)"""
    qb, kvb = _rand((B * Nq, H * 128 + 8), dev, seed + 1, sharp), _rand((B * Nk, 2 * Hkv * 128 + 24), dev, seed + 2)
    lam = _rand((4, lam_heads or H, 64), dev, seed + 3, lam_scale, params)
    gamma = (1 + _rand((128,), dev, seed + 4, 0.2, F32)).to(params) if norm else None
    return qb[:, :H * 128], kvb[:, :Hkv * 128], kvb[:, Hkv * 128 + 16:2 * Hkv * 128 + 16], lam, gamma, _rand((B * Nq, H * 128), dev, seed + 5)


def _call(q, k, v, B, H, Hkv, scale, lam, lam_init, gamma, out_scale, kv_len, causal, dout=None, grads=BF16):
    """forward (and gradient) into guarded buffers -> {name: tensor}"""
    from mofo_amd import ops
    dev, Nq, Nk = q.device, q.shape[0] // B, k.shape[0] // B
    wide = lambda t: torch.full((t.shape[0] + 1, t.shape[1] + 8), 3.0, dtype=BF16, device=dev)  # noqa: E731
    view = lambda w, t: w[:t.shape[0], :t.shape[1]]  # noqa: E731
    ob = wide(q)
    ws = torch.full((ops.diff_attention_fwd_ws(B, Nq, Nk, H, Hkv) + 64,), math.nan, dtype=F32, device=dev)
    form = dict(gamma=gamma, eps=EPS, out_scale=out_scale, kv_len=kv_len, causal=causal)
    saved = None
    if dout is not None:
        saved = (torch.empty(B * Nq, H * 128, dtype=BF16, device=dev), torch.empty(B * Nq, H * 128, dtype=BF16, device=dev),
                 torch.empty(2, B, H, Nq, dtype=F32, device=dev))
    ops.diff_attention_fwd(q, k, v, B, H, Hkv, scale, lam, lam_init, view(ob, q), saved=saved, ws=ws, **form)
    got, guards = {"out": view(ob, q)}, [(ob, q)]
    if dout is not None:
        dqb, dkb, dvb = wide(q), wide(k), wide(v)
        dlam = torch.full(lam.shape, math.nan, dtype=grads, device=dev)
        dgamma = torch.full((128,), math.nan, dtype=grads, device=dev) if gamma is not None else None
        ws = torch.full((ops.diff_attention_bwd_ws(B, Nq, Nk, H, Hkv, gamma is not None) + 4,), math.nan, dtype=F32, device=dev)
        ops.diff_attention_bwd(q, k, v, B, H, Hkv, scale, lam, lam_init, saved, dout, view(dqb, q), view(dkb, k), view(dvb, v), dlam, ws, dgamma=dgamma, **form)
        assert bool(torch.isnan(ws[-4:]).all())
        got.update(o=saved[0], o2=saved[1], lse2=saved[2], dq=view(dqb, q), dk=view(dkb, k), dv=view(dvb, v), dlam=dlam)
        if gamma is not None:
            got["dgamma"] = dgamma
        guards += [(dqb, q), (dkb, k), (dvb, v)]
    for w, t in guards:
        assert bool((w[t.shape[0]:] == 3).all()) and bool((w[:, t.shape[1]:] == 3).all()), "rows behind the last one, columns beside the view"
    return got


def _check(got, want, rel=None):
    for n, t in got.items():
        value, tol = want[n]
        if n == "lse2":
            keep = value > -1e290
            assert bool((t.double()[~keep] > 1e29).all())
            t, value, tol = t.double()[keep], value[keep], tol[keep]
        _within(t, value, tol * 1.01 + TINY, n)
        if rel and n != "lse2":
            assert _rel(t, value) < rel, (n, _rel(t, value))


LENS = "lens"
DIFF = [  # B, Nq, Nk, H, Hkv, causal, kv_len, norm, lam_heads, parameters' type
    (1, 1, 1, 1, 1, 0, None, True, None, BF16), (1, 1, 1, 2, 1, 2, None, False, 1, F32), (2, 3, 3, 2, 2, 1, None, True, None, F32),
    (1, 31, 31, 3, 3, 0, None, True, None, BF16), (2, 33, 33, 2, 1, 1, None, True, 1, BF16), (1, 32, 64, 2, 2, 0, None, False, None, BF16),
    (2, 64, 32, 4, 2, 2, None, True, None, F32), (2, 160, 160, 6, 6, 0, None, True, None, BF16), (1, 257, 257, 3, 3, 1, None, False, None, F32),
    (5, 45, 45, 6, 2, 0, (0, 45, 1, 33, 200), True, None, BF16), (4, 70, 70, 8, 2, 1, (0, 70, -3, 65), False, None, BF16),
    (4, 40, 100, 4, 2, 2, (100, 39, 0, 41), True, None, BF16), (3, 129, 130, 2, 2, 2, (130, 64, 1), False, 1, F32),
    (1, 500, 700, 2, 1, 0, None, True, None, BF16), (2, 391, 391, 3, 1, 1, (391, 250), True, None, BF16),
    (9, 1, 1, 2, 2, 0, (1, 0, 1, 0, 1, 1, 1, 0, 1), True, None, BF16)]


@pytest.mark.parametrize("B,Nq,Nk,H,Hkv,causal,lens,norm,lam_heads,params", DIFF)
def test_diff_attention_forward_and_gradients(dev, B, Nq, Nk, H, Hkv, causal, lens, norm, lam_heads, params):
    q, k, v, lam, gamma, dout = _case(dev, B, Nq, Nk, H, Hkv, norm, lam_heads, params)
    kv_len = None if lens is None else torch.tensor(lens, dtype=I32, device=dev)
    args = (q, k, v, B, H, Hkv, 0.125, lam, 0.45, gamma, 0.55 if norm else 1.0, kv_len, causal)
    want = _reference(*args, dout=dout, grad_u=U if params == BF16 else 0.0)
    _check(_call(*args, dout=dout, grads=params), want, 0.02 if Nk >= 31 and not norm else None)
    _check(_call(*args), want)


MANY = [  # enough (clip, key head) pairs for blocks of 128 rows (keys) in every kernel, or long rows for many four-way blocks; as DIFF
    (24, 140, 140, 12, 12, 0, None, True, None, BF16),                        # eighths of 288 heads an XCD
    (257, 130, 130, 1, 1, 0, None, False, 1, F32),                            # 257 of them: the last eighth is short
    (67, 100, 100, 8, 4, 1, None, True, None, BF16),                          # two heads a key head, causal from the start
    (10, 500, 500, 8, 4, 2, (0, 500, 1, 499, 33, 128, 257, 500, 64, 129), True, None, BF16),          # ragged: one list over all XCDs
    (70, 50, 170, 4, 4, 2, tuple((b * 37) % 172 for b in range(70)), False, None, BF16),
    (110, 544, 544, 1, 1, 0, None, True, None, BF16),                         # whole rounds of 128-row blocks, the last rows in four-way ones
    (28, 272, 272, 8, 4, 0, tuple((b * 61) % 280 for b in range(28)), False, None, F32),
    (20000, 1, 3, 4, 1, 2, None, True, 1, BF16), (3, 5, 77, 64, 1, 2, (77, 4, 0), True, None, F32),   # many clips of one token, many heads on one
    (1, 2150, 2150, 8, 8, 1, None, True, 1, BF16)]                            # four-way, more blocks than the card holds at a time


@pytest.mark.parametrize("B,Nq,Nk,H,Hkv,causal,lens,norm,lam_heads,params", MANY)
def test_diff_attention_many_blocks(dev, B, Nq, Nk, H, Hkv, causal, lens, norm, lam_heads, params):
    test_diff_attention_forward_and_gradients(dev, B, Nq, Nk, H, Hkv, causal, lens, norm, lam_heads, params)


def test_diff_attention_two_streams_at_once(dev):
    """calls of two streams with workspaces of their own overlap and keep their bits"""
    from mofo_amd import ops
    states = []
    for seed, (B, Nq, Nk, H, Hkv) in enumerate(((2, 300, 300, 6, 2), (3, 3, 2500, 4, 2))):
        q, k, v, lam, gamma, dout = _case(dev, B, Nq, Nk, H, Hkv, True, seed=10 * seed)
        want = _call(q, k, v, B, H, Hkv, 0.125, lam, 0.4, gamma, 0.6, None, 2, dout=dout)
        new = lambda t: torch.full(t.shape, 9.0, dtype=BF16, device=dev)  # noqa: E731
        need = max(ops.diff_attention_fwd_ws(B, Nq, Nk, H, Hkv), ops.diff_attention_bwd_ws(B, Nq, Nk, H, Hkv, True))
        states.append((torch.cuda.Stream(), (q, k, v, B, H, Hkv, 0.125, lam, 0.4), dict(gamma=gamma, eps=EPS, out_scale=0.6, causal=2), dout, want,
                       (new(q), new(q), torch.empty(2, B, H, Nq, dtype=F32, device=dev)), [new(q), new(q), new(k), new(v)], torch.empty_like(lam),
                       torch.empty_like(gamma), torch.empty(need, dtype=F32, device=dev)))
    torch.cuda.synchronize()
    for _ in range(4):
        for stream, args, form, dout, _, saved, (out, dq, dk, dv), dlam, dgamma, ws in states:
            with torch.cuda.stream(stream):
                ops.diff_attention_fwd(*args, out, saved=saved, ws=ws, **form)
                ops.diff_attention_bwd(*args, saved, dout, dq, dk, dv, dlam, ws, dgamma=dgamma, **form)
    torch.cuda.synchronize()
    for _, _, _, _, want, saved, (out, dq, dk, dv), dlam, dgamma, _ in states:
        for n, t in dict(out=out, o=saved[0], o2=saved[1], lse2=saved[2], dq=dq, dk=dk, dv=dv, dlam=dlam, dgamma=dgamma).items():
            assert torch.equal(t, want[n]), n


TOKEN = [  # B, Nq, Nk, H, Hkv, kv_len, norm
    (1, 1, 257, 6, 6, None, True), (1, 1, 31, 1, 1, None, False), (2, 1, 1000, 8, 2, None, True), (3, 2, 777, 4, 1, (777, 2, 500), True),
    (4, 5, 90, 4, 4, (90, 5, 0, 33), False), (16, 1, 2048, 8, 2, tuple(1 + 136 * b for b in range(16)), True), (1, 1, 30000, 2, 1, (29999,), True),
    (2, 17, 640, 6, 3, (640, 17), True), (1, 40, 5000, 2, 2, None, False)]


@pytest.mark.parametrize("B,Nq,Nk,H,Hkv,lens,norm", TOKEN)
def test_diff_attention_few_tokens_against_a_cache(dev, B, Nq, Nk, H, Hkv, lens, norm):
    """new tokens at the end of a cache whose rows behind kv_len hold NaN: the split over the keys, and the same with the gradient's o, o2, lse2"""
    q, k, v, lam, gamma, dout = _case(dev, B, Nq, Nk, H, Hkv, norm)
    kv_len = None if lens is None else torch.tensor(lens, dtype=I32, device=dev)
    if lens is not None:
        behind = (torch.arange(Nk, device=dev)[None] >= kv_len[:, None]).reshape(-1)
        k[behind] = math.nan
        v[behind] = math.inf
    args = (q, k, v, B, H, Hkv, 0.125, lam, 0.2, gamma, 0.8 if norm else 1.0, kv_len, 2)
    clean = (q, torch.nan_to_num(k, 0.0), torch.nan_to_num(v, 0.0, 0.0, 0.0)) + args[3:]
    want = _reference(*clean, dout=dout)
    _check(_call(*args), want)
    _check(_call(*args, dout=dout), want)


@pytest.mark.parametrize("B,N,H,Hkv,lens", [(3, 70, 4, 2, (70, 33, 0)), (40, 140, 8, 8, tuple((b * 29) % 141 for b in range(40))), (12, 1111, 8, 2, tuple(range(0, 1200, 100)))])
def test_diff_attention_masked_places_may_hold_anything(dev, B, N, H, Hkv, lens):
    """NaN and infinities behind kv_len in k and v, and in q and dout of rows that see nothing, reach no output and no gradient"""
    q, k, v, lam, gamma, dout = _case(dev, B, N, N, H, Hkv, True)
    kv_len = torch.tensor(lens, dtype=I32, device=dev)
    for causal in (0, 2):
        lim = _limits(B, N, N, kv_len, causal, dev).reshape(-1)
        behind = (torch.arange(N, device=dev)[None] >= kv_len[:, None]).reshape(-1)
        k2, v2, q2, d2 = k.clone(), v.clone(), q.clone(), dout.clone()
        k2[behind], v2[behind] = math.nan, -math.inf
        q2[lim == 0] = math.nan
        args = lambda *t: t + (B, H, Hkv, 0.125, lam, 0.45, gamma, 0.55, kv_len, causal)  # noqa: E731
        a, b = _call(*args(q, k, v), dout=dout), _call(*args(q2, k2, v2), dout=d2)
        for n in a:
            assert torch.equal(a[n], b[n]), n
        for n in ("out", "dq"):
            assert not a[n][lim == 0].any(), n
        for n in ("dk", "dv"):
            assert not a[n][behind].any(), n


@pytest.mark.parametrize("sharp", [0.0, 30.0])
def test_diff_attention_flat_and_sharp_maps(dev, sharp):
    """all scores equal, and scores of some hundred log2 units that grow along the keys (the running maximum moves many times)"""
    B, N, H = 1, 300, 2
    q, k, v, lam, _, dout = _case(dev, B, N, N, H, H, False, sharp=max(sharp / 8, 1e-3))
    if sharp == 0.0:
        q.zero_()
    else:
        k.mul_(torch.linspace(0.1, 4.0, N, device=dev)[:, None].to(BF16))
    args = (q, k, v, B, H, H, 0.125, lam, 0.45, None, 1.0, None, 0)
    got, want = _call(*args, dout=dout), _reference(*args, dout=dout)
    # scores of hundreds: 32-bit scores are off by 2^-23 of their size in the exponent, four times what F allows for
    slack = 1.0 if sharp == 0.0 else 4.0
    _check(got, {n: (a, b * slack) for n, (a, b) in want.items()})


@pytest.mark.parametrize("lam_init", [-0.6, 0.0, 0.9])
def test_diff_attention_signs_of_lambda(dev, lam_init):
    """negative, about zero (exactly zero with all-zero vectors) and large lambda, heads of both signs that share keys"""
    B, N, H, Hkv = 1, 77, 4, 2
    q, k, v, lam, gamma, dout = _case(dev, B, N, N, H, Hkv, True, params=F32, lam_scale=0.2)
    if lam_init == 0.0:
        lam[:, :2] = 0.0
    args = (q, k, v, B, H, Hkv, 0.125, lam, lam_init, gamma, 0.7, None, 0)
    _check(_call(*args, dout=dout, grads=F32), _reference(*args, dout=dout, grad_u=0.0))


@pytest.mark.parametrize("scale", [2.0 ** -24, 2.0 ** 24])
def test_diff_attention_ends_of_the_scale(dev, scale):
    """the smallest and the largest scale taken: uniform maps, and one key a row; rows that see nothing, and a head whose lambda is exactly zero"""
    B, N, H = 2, 70, 2
    q, k, v, lam, gamma, dout = _case(dev, B, N, N, H, H, True, params=F32)
    lam[:, 0] = 0.0
    args = (q, k, v, B, H, H, scale, lam, 0.0, gamma, 0.6, torch.tensor([70, 30], dtype=I32, device=dev), 2)
    got = _call(*args, dout=dout, grads=F32)
    if scale < 1:
        _check(got, _reference(*args, dout=dout, grad_u=0.0))
    for n, t in got.items():
        assert bool(torch.isfinite(t.float()).all()), n
    assert not got["out"][N:N + 40].any() and not got["dq"][N:N + 40].any() and not got["dk"][N + 30:].any() and not got["dv"][N + 30:].any()


@pytest.mark.parametrize("B,Nq,Nk,H,Hkv", [(2, 1, 4000, 4, 2), (1, 50, 50, 2, 1), (24, 140, 140, 12, 12)])
def test_diff_attention_a_bad_query_stays_in_its_row(dev, B, Nq, Nk, H, Hkv):
    """NaN in one visible query row of one head: that row is NaN in that head, in every form of the forward pass, and no other number moves"""
    q, k, v, lam, gamma, _ = _case(dev, B, Nq, Nk, H, Hkv, True)
    args = lambda t: (t, k, v, B, H, Hkv, 0.125, lam, 0.4, gamma, 0.6, None, 0)  # noqa: E731
    want = _call(*args(q))["out"]
    q2, row = q.clone(), Nq * B - 1
    q2[row, 128 + 70] = math.nan
    got = _call(*args(q2))["out"]
    assert bool(torch.isnan(got[row, 128:256]).all())
    same = torch.ones_like(got, dtype=torch.bool)
    same[row, 128:256] = False
    assert torch.equal(got[same], want[same])


def test_diff_attention_gradients_against_differences(dev):
    """the kernels' gradients along a direction against central differences of the definition in 64 bits"""
    B, N, H, Hkv = 2, 37, 4, 2
    q, k, v, lam, gamma, dout = _case(dev, B, N, N, H, Hkv, True, params=F32)
    kv_len = torch.tensor([37, 20], dtype=I32, device=dev)
    tail = (0.6, kv_len, 1)
    args = (q, k, v, B, H, Hkv, 0.125, lam, 0.4, gamma) + tail
    got, want = _call(*args, dout=dout, grads=F32), _reference(*args, dout=dout, grad_u=0.0)
    loss = lambda a, b, c, l, g: (_reference(a, b, c, B, H, Hkv, 0.125, l, 0.4, g, *tail)["out"][0] * dout.double()).sum()  # noqa: E731
    there = (torch.arange(N, device=dev)[None] < kv_len[:, None]).reshape(-1)[:, None]
    for at, (n, t) in enumerate((("dq", q), ("dk", k), ("dv", v), ("dlam", lam), ("dgamma", gamma))):
        step = torch.randn(t.shape, generator=torch.Generator().manual_seed(at), dtype=F64).to(dev)
        if n in ("dk", "dv"):
            step = step * there
        h = 1e-5
        ends = [[x.double() + (sgn * h * step if j == at else 0) for j, x in enumerate((q, k, v, lam, gamma))] for sgn in (1, -1)]
        slope = (loss(*ends[0]) - loss(*ends[1])) / (2 * h)
        bound = (want[n][1] * step.abs()).sum() + 1e-6 * slope.abs()
        assert abs(float(slope - (got[n].double() * step).sum())) <= float(bound), n


def test_diff_attention_same_bits_every_time(dev):
    B, N, H, Hkv = 3, 333, 6, 2
    q, k, v, lam, gamma, dout = _case(dev, B, N, N, H, Hkv, True)
    args = (q, k, v, B, H, Hkv, 0.125, lam, 0.45, gamma, 0.55, None, 1)
    a = _call(*args, dout=dout)
    for _ in range(3):
        b = _call(*args, dout=dout)
        assert all(torch.equal(a[n], b[n]) for n in a)


def test_diff_attention_rows_do_not_depend_on_their_neighbours(dev):
    """a clip's results are the same bits alone and inside a batch (nothing is shared between clips)"""
    B, N, H = 4, 200, 3
    q, k, v, lam, gamma, dout = _case(dev, B, N, N, H, H, True)
    tail = (H, H, 0.125, lam, 0.45, gamma, 0.55, None, 0)
    whole = _call(q, k, v, B, *tail, dout=dout)
    one = slice(2 * N, 3 * N)
    alone = _call(q[one], k[one], v[one], 1, *tail, dout=dout[one])
    for n in ("out", "dq", "dk", "dv"):
        assert _rel(whole[n][one], alone[n]) < 2 * U, n      # another split of the keys may round P against another reference


def test_diff_attention_offsets_beyond_32_bits(dev):
    """a cache whose rows lie 2^20 elements apart: its last rows start behind element 2^31"""
    B, Nk, H = 1, 2200, 1
    ld = 1 << 20
    big = torch.empty(Nk, ld, dtype=BF16, device=dev)
    big[:, :256] = _rand((Nk, 256), dev, 3)
    q, lam = _rand((1, 128), dev, 1), _rand((4, 1, 64), dev, 2, 0.1)
    args = (q, big[:, :128], big[:, 128:256], B, H, H, 0.125, lam, 0.45, None, 1.0, None, 2)
    _check(_call(*args), _reference(*args))
    small = (q, big[:, :128].clone(), big[:, 128:256].clone()) + args[3:]
    assert torch.equal(_call(*args)["out"], _call(*small)["out"])


def test_diff_attention_captured_and_replayed(dev):
    """forward and gradient in a graph, on a stream of its own, replayed between eager calls of other inputs; two graphs, two workspaces"""
    from mofo_amd import ops
    B, N, H, Hkv = 2, 150, 4, 2
    tail = dict(eps=EPS, out_scale=0.55, causal=1)

    def state(seed):
        q, k, v, lam, gamma, dout = (t.clone() for t in _case(dev, B, N, N, H, Hkv, True, seed=seed))
        s = dict(q=q, k=k, v=v, lam=lam, gamma=gamma, dout=dout, out=torch.empty_like(q), saved=(torch.empty_like(q), torch.empty_like(q),
                 torch.empty(2, B, H, N, dtype=F32, device=dev)), dq=torch.empty_like(q), dk=torch.empty_like(k), dv=torch.empty_like(v),
                 dlam=torch.empty_like(lam), dgamma=torch.empty_like(gamma), ws=torch.empty(ops.diff_attention_bwd_ws(B, N, N, H, Hkv, True), dtype=F32, device=dev),
                 ws_f=torch.empty(max(1, ops.diff_attention_fwd_ws(B, N, N, H, Hkv)), dtype=F32, device=dev))
        return s

    def step(s):
        ops.diff_attention_fwd(s["q"], s["k"], s["v"], B, H, Hkv, 0.125, s["lam"], 0.45, s["out"], gamma=s["gamma"], saved=s["saved"], ws=s["ws_f"], **tail)
        ops.diff_attention_bwd(s["q"], s["k"], s["v"], B, H, Hkv, 0.125, s["lam"], 0.45, s["saved"], s["dout"], s["dq"], s["dk"], s["dv"], s["dlam"], s["ws"],
                               gamma=s["gamma"], dgamma=s["dgamma"], **tail)

    names = ("out", "dq", "dk", "dv", "dlam", "dgamma")
    one, two, eager = state(1), state(50), state(99)
    want = []
    for s in (one, two):
        step(s)
        torch.cuda.synchronize()
        want.append({n: s[n].clone() for n in names})
    graphs = []
    for s in (one, two):
        g = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(s)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            step(s)
        graphs.append(g)
    for turn in range(4):
        for s, g, w in zip((one, two), graphs, want):
            for n in names:
                s[n].fill_(5.0)
            g.replay()
            step(eager)
            torch.cuda.synchronize()
            for n in names:
                assert torch.equal(s[n], w[n]), (turn, n)


def test_rope_and_diff_attention_as_a_block_uses_them(dev):
    """packed projection of the visible tokens -> rotary q, k -> differential attention -> its gradient -> the projection's gradient, against
    64 bits; the launches go to a stream of their own through ops.use_stream"""
    from mofo_amd import ops
    B, N, H, sections = 2, 160, 3, (8, 12, 12)
    M, D = B * N, H * 128
    packed = _rand((M, 3 * D), dev, 1)
    tok = torch.stack([torch.randperm(1568, generator=torch.Generator().manual_seed(b))[:N].sort().values for b in range(B)]).to(I32).to(dev)
    lam, gamma, dout = _rand((4, H, 64), dev, 2, 0.1), _rand((128,), dev, 3), _rand((M, D), dev, 4)
    freqs = ops.rope_freqs(sections, device=dev)
    qk, out, dqkv, dqk = torch.empty(M, 2 * D, dtype=BF16, device=dev), torch.empty(M, D, dtype=BF16, device=dev), torch.empty_like(packed), torch.empty(M, 2 * D, dtype=BF16, device=dev)
    saved = (torch.empty_like(out), torch.empty_like(out), torch.empty(2, B, H, N, dtype=F32, device=dev))
    dlam, dgamma = torch.empty_like(lam), torch.empty_like(gamma)
    ws = torch.empty(max(ops.diff_attention_fwd_ws(B, N, N, H, H), ops.diff_attention_bwd_ws(B, N, N, H, H, True)), dtype=F32, device=dev)
    where = dict(tok_idx=tok, grid=(8, 14, 14))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ops.use_stream(side)
    try:
        ops.rope_axes_fwd(packed[:, :2 * D], 4 * H, 64, sections, freqs, qk, **where)
        ops.diff_attention_fwd(qk[:, :D], qk[:, D:], packed[:, 2 * D:], B, H, H, 0.125, lam, 0.4, out, gamma=gamma, eps=EPS, out_scale=0.6, saved=saved, ws=ws)
        ops.diff_attention_bwd(qk[:, :D], qk[:, D:], packed[:, 2 * D:], B, H, H, 0.125, lam, 0.4, saved, dout, dqk[:, :D], dqk[:, D:], dqkv[:, 2 * D:], dlam, ws,
                               gamma=gamma, dgamma=dgamma, eps=EPS, out_scale=0.6)
        ops.rope_axes_bwd(dqk, 4 * H, 64, sections, freqs, dqkv[:, :2 * D], **where)
    finally:
        ops.use_stream(None)
    torch.cuda.current_stream().wait_stream(side)
    place = torch.stack([tok.reshape(-1) // 196, tok.reshape(-1) // 14 % 14, tok.reshape(-1) % 14], 1)
    turned, _ = _rope64(packed[:, :2 * D], 4 * H, 64, sections, place, 10000.0, False)
    # the roundings of q and k are the operator's inputs: the attention is held to its own bounds on the rotated values it was given
    _check(dict(out=out, dq=dqk[:, :D], dk=dqk[:, D:], dv=dqkv[:, 2 * D:], dlam=dlam, dgamma=dgamma),
           _reference(qk[:, :D], qk[:, D:], packed[:, 2 * D:], B, H, H, 0.125, lam, 0.4, gamma, 0.6, None, 0, dout=dout))
    # and end to end: one more rounding of q, k, dq, dk each
    want = _reference(turned[:, :D], turned[:, D:], packed[:, 2 * D:], B, H, H, 0.125, lam, 0.4, gamma, 0.6, None, 0, dout=dout)
    assert _rel(out, want["out"][0]) < 0.02 and _rel(dqkv[:, 2 * D:], want["dv"][0]) < 0.02
    back, _ = _rope64(torch.cat([want["dq"][0], want["dk"][0]], 1), 4 * H, 64, sections, place, 10000.0, False, -1.0)
    assert _rel(dqkv[:, :2 * D], back) < 0.02


def test_diff_attention_refusals(dev):
    from mofo_amd import ops
    B, N, H, Hkv = 2, 8, 4, 2
    q, k, v, lam, gamma, dout = (t.clone() for t in _case(dev, B, N, N, H, Hkv, True))
    out, z = torch.empty_like(q), torch.empty(2, B, H, N, dtype=F32, device=dev)
    saved = (torch.empty_like(q), torch.empty_like(q), z)
    ws = torch.empty(ops.diff_attention_bwd_ws(B, N, N, H, Hkv, True), dtype=F32, device=dev)
    ln = torch.full((B,), N, dtype=I32, device=dev)

    def fwd(**kw):
        a = dict(q=q, k=k, v=v, B=B, H=H, Hkv=Hkv, scale=0.125, lam=lam, lam_init=0.4, out=out, gamma=gamma)
        a.update(kw)
        return lambda: ops.diff_attention_fwd(**a)

    def bwd(**kw):
        a = dict(q=q, k=k, v=v, B=B, H=H, Hkv=Hkv, scale=0.125, lam=lam, lam_init=0.4, saved=saved, dout=dout, dq=torch.empty_like(q), dk=torch.empty_like(k),
                 dv=torch.empty_like(v), dlam=torch.empty_like(lam), dgamma=torch.empty_like(gamma), gamma=gamma, ws=ws)
        a.update(kw)
        return lambda: ops.diff_attention_bwd(**a)

    for bad in (fwd(q=q.float()), fwd(lam=lam.half()), fwd(gamma=gamma.float()), fwd(kv_len=ln.long()), fwd(out=out.float()), bwd(dlam=lam.half()), bwd(dgamma=gamma.float())):
        with pytest.raises(TypeError):
            bad()
    for bad in (fwd(B=3), fwd(Hkv=3), fwd(v=v[:8]), fwd(lam=lam[:3]), fwd(lam=lam[:, :3]), fwd(gamma=gamma[:64]), fwd(kv_len=ln[:1]), fwd(causal=3),
                fwd(out=out[:8]), fwd(saved=(saved[0], saved[1], z[:1])), fwd(q=q.cpu()), bwd(dgamma=None), bwd(dk=torch.empty_like(q)), bwd(dout=dout[:8]),
                bwd(ws=None)):
        with pytest.raises(ValueError):
            bad()
    for bad in (fwd(scale=-1.0), fwd(scale=0.0), fwd(scale=math.nan)):
        with pytest.raises(RuntimeError, match="scale"):
            bad()
    for bad in (fwd(out=q), fwd(saved=(saved[0], saved[0], z)), fwd(saved=(out, saved[1], z)), bwd(dq=q), bwd(dq=dout)):
        with pytest.raises(RuntimeError, match="overlaps"):
            bad()
    shifted = torch.empty(B * N, H * 128 + 4, dtype=BF16, device=dev)
    for bad in (fwd(q=shifted[:, 4:]), bwd(ws=ws[:-1]), bwd(ws=torch.empty(ws.numel() + 1, dtype=F32, device=dev)[1:])):
        with pytest.raises(RuntimeError):
            bad()
    fwd()(), bwd()()


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("B,Nq,Nk,H,Hkv,lens,causal", [
    (3, 70, 70, 4, 2, (70, 33, 0), 0), (3, 70, 70, 4, 2, (0, 70, 5), 1), (3, 70, 70, 4, 2, (70, 33, 0), 2), (2, 64, 32, 4, 2, (32, 7), 2),
    (40, 140, 140, 8, 8, tuple((b * 29) % 141 for b in range(40)), 2)])
def test_diff_attention_gradients_of_rows_that_see_nothing_are_not_taken(dev, norm, B, Nq, Nk, H, Hkv, lens, causal):
    """NaN and infinities in dout, and in q, of rows that see no key: every output and every gradient, dgamma among them, keeps its bits"""
    q, k, v, lam, gamma, dout = _case(dev, B, Nq, Nk, H, Hkv, norm)
    kv_len = torch.tensor(lens, dtype=I32, device=dev)
    nothing = (_limits(B, Nq, Nk, kv_len, causal, dev) == 0).reshape(-1)
    assert bool(nothing.any()) and not bool(nothing.all())
    args = lambda t: (t, k, v, B, H, Hkv, 0.125, lam, 0.45, gamma, 0.55 if norm else 1.0, kv_len, causal)  # noqa: E731
    want = _call(*args(q), dout=dout)
    for bad in (math.nan, math.inf):
        q2, d2 = q.clone(), dout.clone()
        q2[nothing], d2[nothing] = bad, bad
        got = _call(*args(q2), dout=d2)
        for n in want:
            assert torch.equal(got[n], want[n]), (n, bad)


def test_row_pitches_and_counts_that_do_not_fit_the_entries_are_refused(dev):
    """two rows 2^32 + 512 elements apart (a pitch whose low 32 bits would do), a grid and a number of rows beyond 32 bits"""
    from mofo_amd import ops
    big = torch.zeros((1 << 32) + 1024, dtype=BF16, device=dev)
    far = lambda n: big.as_strided((2, n), ((1 << 32) + 512, 1))  # noqa: E731
    x, lam = _rand((2, 128), dev, 1), _rand((4, 1, 64), dev, 2, 0.1)
    f, pos, tok = ops.rope_freqs((8, 12, 12), device=dev), torch.zeros(2, 3, dtype=I32, device=dev), torch.zeros(2, dtype=I32, device=dev)
    out, ws = torch.empty_like(x), torch.empty(1 << 16, dtype=F32, device=dev)
    saved = (torch.empty_like(x), torch.empty_like(x), torch.empty(2, 1, 1, 2, dtype=F32, device=dev))
    attend = lambda **kw: ops.diff_attention_fwd(**{**dict(q=x, k=x, v=x, B=1, H=1, Hkv=1, scale=0.125, lam=lam, lam_init=0.4, out=out), **kw})  # noqa: E731
    back = lambda **kw: ops.diff_attention_bwd(**{**dict(q=x, k=x, v=x, B=1, H=1, Hkv=1, scale=0.125, lam=lam, lam_init=0.4, saved=saved, dout=x, dq=torch.empty_like(x),  # noqa: E731
                                                         dk=torch.empty_like(x), dv=torch.empty_like(x), dlam=torch.empty_like(lam), ws=ws), **kw})
    for bad in (lambda: ops.rope_axes_fwd(far(128), 2, 64, (8, 12, 12), f, out, pos=pos), lambda: ops.rope_axes_bwd(x, 2, 64, (8, 12, 12), f, far(128), pos=pos),
                lambda: attend(q=far(128)), lambda: attend(k=far(128)), lambda: attend(v=far(128)), lambda: attend(out=far(128)), lambda: back(dout=far(128)),
                lambda: back(dq=far(128)), lambda: back(dk=far(128)), lambda: back(dv=far(128)),
                lambda: ops.rope_axes_fwd(x, 2, 64, (8, 12, 12), f, out, tok_idx=tok, grid=(8, (1 << 32) + 14, 14))):
        with pytest.raises(ValueError):
            bad()
    rows = torch.zeros(16, dtype=BF16, device=dev).expand((1 << 32) + 1, 16)
    with pytest.raises(ValueError, match="rows"):
        ops.rope_axes_fwd(rows, 1, 16, (8,), ops.rope_freqs((8,), device=dev), rows, tok_idx=tok, grid=(8, 14, 14))


def _far_scores(dev, B, Nq, Nk, H, Hkv, offset, seed=0):
    """whole-numbered inputs whose scores are ``offset`` + small whole numbers, exact in 32 bits in any order of the sums (all below 2^24 in size);
    the offset's sign is the query row's and the map's own"""
    g = torch.Generator().manual_seed(seed)
    whole = lambda *s: torch.randint(-2, 3, s, generator=g).to(F32)  # noqa: E731
    a = 2.0 ** (math.frexp(offset)[1] // 2)
    q, k, v = whole(B * Nq, H, 2, 64), whole(B * Nk, Hkv, 2, 64), torch.randn(B * Nk, Hkv * 128, generator=g)
    sign = torch.randint(0, 2, (B * Nq, H, 2), generator=g) * 2.0 - 1
    q[..., 0], k[..., 0] = sign * a, offset / a
    lam = (torch.randn(4, H, 64, generator=g) * 0.1).to(F32).to(dev)
    return q.reshape(B * Nq, -1).to(BF16).to(dev), k.reshape(B * Nk, -1).to(BF16).to(dev), v.to(BF16).to(dev), lam


FAR = [  # B, Nq, Nk, H, Hkv, causal: ranges of keys, four-way blocks, 128-row blocks, 128-row blocks with a causal mask
    (2, 1, 4000, 4, 2, 2), (1, 3, 2500, 2, 2, 0), (1, 300, 300, 2, 1, 1), (24, 140, 140, 12, 12, 0), (67, 100, 100, 8, 4, 1)]


@pytest.mark.parametrize("offset", [2.0 ** 12, 2.0 ** 16, 2.0 ** 22])
@pytest.mark.parametrize("B,Nq,Nk,H,Hkv,causal", FAR)
def test_diff_attention_scores_far_from_zero(dev, B, Nq, Nk, H, Hkv, causal, offset):
    """soft maps whose scores all lie far from zero: exponents are differences, so the size of the scores costs the outputs nothing.  (The scores
    themselves are exact here; lse2 is one 32-bit number of the scores' size.)  With and without what the gradient wants."""
    q, k, v, lam = _far_scores(dev, B, Nq, Nk, H, Hkv, offset)
    args = (q, k, v, B, H, Hkv, 0.125, lam, 0.45, None, 1.0, None, causal)
    want = _reference(*args)
    _check(_call(*args), want, 0.01)
    from mofo_amd import ops
    saved = (torch.empty_like(q), torch.empty_like(q), torch.empty(2, B, H, Nq, dtype=F32, device=dev))
    out, ws = torch.empty_like(q), torch.empty(ops.diff_attention_fwd_ws(B, Nq, Nk, H, Hkv), dtype=F32, device=dev)
    ops.diff_attention_fwd(q, k, v, B, H, Hkv, 0.125, lam, 0.45, out, saved=saved, ws=ws, causal=causal)
    _check(dict(out=out, o=saved[0], o2=saved[1], lse2=saved[2]), want, 0.01)


@pytest.mark.parametrize("B,Nq,Nk,H,Hkv,causal", FAR)
def test_diff_attention_scores_of_any_size(dev, B, Nq, Nk, H, Hkv, causal):
    """every score the same number, 1.4 * 2^106 (times the scale), of either sign: the maps are uniform"""
    q, k, v, lam = _far_scores(dev, B, Nq, Nk, H, Hkv, 181 * 2.0 ** 99)
    q.view(-1, 64)[:, 1:] = 0
    args = (q, k, v, B, H, Hkv, 0.125, lam, 0.45, None, 1.0, None, causal)
    _check(_call(*args), _reference(*args), 0.01)


@pytest.mark.parametrize("B,Nq,Nk,H,Hkv,causal", FAR)
def test_diff_attention_scores_that_come_near(dev, B, Nq, Nk, H, Hkv, causal):
    """the keys' scores lie 2^16 (times the scale) from zero at the start and near it from a third of the keys on: on either side of it by the row,
    and below it in every row, so that no row's reference stays far"""
    q, k, v, lam = _far_scores(dev, B, Nq, Nk, H, Hkv, 2.0 ** 16)
    k.view(B, Nk, -1, 64)[:, Nk // 3:, :, 0] = 1.0 / 256
    for below in (False, True):
        if below:
            q.view(-1, 64)[:, 0] = -q.view(-1, 64)[:, 0].abs()
        args = (q, k, v, B, H, Hkv, 0.125, lam, 0.45, None, 1.0, None, causal)
        _check(_call(*args), _reference(*args), 0.01)


@pytest.mark.parametrize("B,Nq,Nk,H,Hkv,causal", FAR)
def test_diff_attention_gradients_of_scores_far_from_zero(dev, B, Nq, Nk, H, Hkv, causal):
    """scores about +-2^12, the size up to which the gradient's probabilities are promised to 2^-9 of their value: that in the place of F,
    2^-14, is 32 times F.  2-norms: the usual 2 %, and twice 2^-9 for the difference of two maps; without the columns of the offset, where dq
    and dk are sums that cancel to nothing."""
    q, k, v, lam = _far_scores(dev, B, Nq, Nk, H, Hkv, 2.0 ** 15)
    dout = _rand((B * Nq, H * 128), dev, 5)
    args = (q, k, v, B, H, Hkv, 0.125, lam, 0.45, None, 1.0, None, causal)
    got, want = _call(*args, dout=dout, grads=F32), _reference(*args, dout=dout, grad_u=0.0)
    _check(got, {n: (t, b * (32.0 if n.startswith("d") else 1.0)) for n, (t, b) in want.items()})
    for n in ("dq", "dk", "dv"):
        a, b = (t.double().reshape(t.shape[0], -1, 64)[..., 1 if n != "dv" else 0:] for t in (got[n], want[n][0]))
        assert _rel(a, b) < 0.02 + 2 * 2.0 ** -9, (n, _rel(a, b))


@pytest.mark.parametrize("power", [-21, 27])
@pytest.mark.parametrize("B,Nq,Nk,H,Hkv,causal", FAR)
def test_diff_attention_same_bits_at_any_scale(dev, B, Nq, Nk, H, Hkv, causal, power):
    """the ends of the scale, 2^-24 and 2^24, with the same scores: powers of two move from q and k into the scale, and back out of dq and dk"""
    q, k, v, lam, gamma, dout = _case(dev, B, Nq, Nk, H, Hkv, True)
    half, rest = 2.0 ** -(power // 2), 2.0 ** -(power - power // 2)
    form = (lam, 0.45, gamma, 0.55, None, causal)
    want = _call(q, k, v, B, H, Hkv, 0.125, *form, dout=dout)
    got = _call(q * half, k * rest, v, B, H, Hkv, 0.125 * 2.0 ** power, *form, dout=dout)
    for n in want:
        scaled = {"dq": 1 / half, "dk": 1 / rest}.get(n, 1.0)
        assert torch.equal(got[n], want[n] * scaled), n


@pytest.mark.parametrize("B,Nq,Nk,H,Hkv,causal", FAR)
def test_diff_attention_far_and_bad_rows_leave_their_neighbours_alone(dev, B, Nq, Nk, H, Hkv, causal):
    """one visible query row with scores of 2^40, and another whose scores are NaN: no bit of any other row moves, with near and with far scores of
    the others"""
    for offset in (0.0, 2.0 ** 16):
        q, k, v, lam = _far_scores(dev, B, Nq, Nk, H, Hkv, offset or 1.0)
        args = lambda t: (t, k, v, B, H, Hkv, 0.125, lam, 0.4, None, 1.0, None, causal)  # noqa: E731
        want = _call(*args(q))["out"]
        q2, far, bad = q.clone(), Nq * B - 1, Nq * B - (2 if Nq * B > 1 else 1)
        q2[far, :128] *= 2.0 ** 40
        q2[bad, (H - 1) * 128 + 70] = math.nan
        got = _call(*args(q2))["out"]
        assert bool(torch.isfinite(got[far, :128].float()).all()) and bool(torch.isnan(got[bad, (H - 1) * 128:]).all())
        same = torch.ones_like(got, dtype=torch.bool)
        same[far, :128] = same[bad, (H - 1) * 128:] = False
        assert torch.equal(got[same], want[same])


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("B,Nq,Nk,H,Hkv,causal", FAR)
def test_diff_attention_far_scores_and_rows_that_see_nothing(dev, norm, B, Nq, Nk, H, Hkv, causal):
    """lengths from none to all with scores far from zero: rows that see nothing give zeros, whatever they hold"""
    q, k, v, lam = _far_scores(dev, B, Nq, Nk, H, Hkv, 2.0 ** 16)
    gamma = _rand((128,), dev, 9, 1.0, F32) if norm else None
    for lens in ([(b * 37) % (Nk + 1) for b in range(B)], [Nk - (b * 11) % (Nk + 1) for b in range(B)]):
        kv_len = torch.tensor(lens, dtype=I32, device=dev)
        args = lambda t: (t, k, v, B, H, Hkv, 0.125, lam, 0.4, gamma, 0.6 if norm else 1.0, kv_len, causal)  # noqa: E731
        want = _reference(*args(q))
        got = _call(*args(q))
        _check(got, want)
        q2 = q.clone()
        q2[(_limits(B, Nq, Nk, kv_len, causal, dev) == 0).reshape(-1)] = math.nan
        assert torch.equal(_call(*args(q2))["out"], got["out"])
