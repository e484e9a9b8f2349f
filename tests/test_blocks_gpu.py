"""The block operators and the choice head against plain 64-bit forms.

Tolerances are elementwise and derived, not fitted.  u(t) = finfo(t).eps / 2 is
the rounding of one output.  A sum of f32 terms in any order is within
2^-24 * (number of additions) of the sum of magnitudes; the tensor cores add 16
(8-bit: 32) products at a time into an f32 accumulator that they may truncate,
so a product over k is within (k / 16 + 16) * 2^-22 of sum |x| |w|.  What a
kernel rounds on the way (dz, dg, du to 16 bits) adds u(t) times the sum of the
magnitudes that it enters.
"""
import math

import numpy as np
import pytest
import torch

import browsergnn_b200 as bg

pytestmark = pytest.mark.gpu

F32, BF, F16, F8 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn
U = {t: torch.finfo(t).eps / 2 for t in (F32, BF, F16)}
TINY = {F32: 1e-38, BF: 1e-38, F16: 2.0 ** -25}  # half a subnormal step


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, t=F32, std=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(t)


def within(got, want, tol, what):
    got = got.double()
    assert got.shape == want.shape, what
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~(((got - want).abs() <= tol) | same)
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; first at {i}: got "
                             f"{got[i].item()!r} want {want[i].item()!r} tol "
                             f"{(tol.expand_as(want)[i].item() if hasattr(tol, 'expand_as') else tol)!r}")


def wide(x, how):
    """x as a view with other strides: 'plain', 'rows' apart, 'odd' (rows that
    start off every vector) or 'vector' (rows that start on one, NaN behind)."""
    if how == "plain":
        return x
    if how == "vector":
        big = torch.full((x.shape[0], (x.shape[1] + 7) // 8 * 8 + 8), math.nan, dtype=x.dtype,
                         device=x.device)
        big[:, :x.shape[1]] = x
        return big[:, :x.shape[1]]
    pad = 8 if how == "rows" else 3
    big = torch.full((x.shape[0], x.shape[1] + 2 * pad), math.nan, dtype=x.dtype, device=x.device)
    big[:, pad:-pad] = x
    return big[:, pad:-pad]


# ---------------------------------------------------------------------------
# norm
# ---------------------------------------------------------------------------
NORMS = [  # rows, cols, x, residual, out
    (1, 1, F32, None, F32), (1, 1024, BF, BF, F8), (3, 8, F16, F32, F16), (7, 47, F32, F32, BF),
    (129, 256, F32, F32, BF), (33, 1433, F16, F16, F16), (5, 2056, BF, F32, F8),
    (300, 16, BF, None, BF), (2, 8192, F32, None, F8), (2, 16392, BF, BF, BF),
    (2, 8200, F16, None, F32), (3, 20001, F32, F32, F8), (2, 33000, BF, F32, BF),
    (70000, 24, F32, None, F16), (9, 100, BF, BF, F8),
]


@pytest.mark.parametrize("how", ["plain", "rows", "odd"])
@pytest.mark.parametrize("rows,cols,tx,tr,to", NORMS)
def test_rms_norm(rows, cols, tx, tr, to, how):
    g = gen(rows * 31 + cols)
    x = wide(normal(g, rows, cols, t=tx), how)
    r = None if tr is None else wide(normal(g, rows, cols, t=tr, std=3.0), how)
    w = normal(g, cols, t=F32 if tx == F32 else tx) + 1
    eps = 1e-5
    out, total, scale = bg.rmsNorm(x, w, residual=r, eps=eps, outType=to)
    t = x.double()
    if r is not None:
        want = x.double() + r.double()
        assert total.dtype == tr
        # the sum rounded to f32, then to its type
        within(total, want, (U[tr] + U[F32]) * want.abs() + TINY[tr], "total")
        t = total.double()
    else:
        assert total is x
    s = (t.pow(2).mean(1, keepdim=True) + eps).rsqrt()
    y = t * s * w.double()
    slop = (cols + 16) * 2.0 ** -24  # the mean square; halved by the root, doubled for safety
    if to == F8:
        amax = y.abs().amax(1)
        within(scale, amax / 448, amax / 448 * (slop + 4 * U[F32]), "scale")
        got = out.double() * scale.double()[:, None]
        tol = y.abs() * (2.0 ** -4 + slop) + scale.double()[:, None] * 2.0 ** -10
        within(got, y, tol, "out")
    else:
        assert scale is None and out.dtype == to
        within(out, y, y.abs() * (U[to] + slop + 4 * U[F32]) + TINY[to], "out")


def test_rms_norm_one_row_and_empty():
    g = gen(1)
    x, w = normal(g, 64, t=BF), normal(g, 64)
    a, total, _ = bg.rmsNorm(x, w, residual=x)
    b, _, _ = bg.rmsNorm(x[None], w, residual=x[None])
    assert a.shape == (64,) and total.shape == (64,) and torch.equal(a, b[0])
    out, total, scale = bg.rmsNorm(torch.empty(0, 64, device="cuda"), w, outType=F8)
    assert out.shape == (0, 64) and scale.shape == (0,)
    none = torch.empty(3, 0, device="cuda")
    out, _, scale = bg.rmsNorm(none, torch.empty(0, device="cuda"), outType=F8)
    assert out.shape == (3, 0) and (scale == 0).all()
    gx, gw = bg.rmsNormBackward(torch.empty(0, 64, device="cuda"),
                                torch.empty(0, 64, device="cuda"), w)
    assert gx.shape == (0, 64) and torch.equal(gw, torch.zeros_like(w))


def test_rms_norm_rows_of_zeros_tiny_and_not_finite():
    w = torch.ones(40, device="cuda")
    x = torch.zeros(5, 40, device="cuda")
    x[1] = 1e-30
    x[2, 3] = math.nan
    x[3, 5] = math.inf
    x[4] = 2.0
    out, _, scale = bg.rmsNorm(x, w, eps=0.25, outType=F8)
    assert torch.equal(out[0].float(), torch.zeros(40, device="cuda")) and scale[0] == 1
    assert torch.allclose(out[1].float() * scale[1], x[1] * 2, rtol=2.0 ** -4, atol=0)
    assert scale[2].isnan() and out[2].float().isnan().all()
    assert torch.isfinite(scale[4]) and torch.isfinite(out[4].float()).all()
    y, _, _ = bg.rmsNorm(x, w, eps=0.25)
    assert y[2].isnan().all() and y[3, 5].isnan() and torch.isfinite(y[[0, 1, 4]]).all()


@pytest.mark.parametrize("how", ["plain", "odd"])
@pytest.mark.parametrize("rows,cols,tt,tg,stream", [
    (1, 1, F32, F32, False), (1, 1024, BF, BF, True), (257, 256, F32, BF, True),
    (40, 1433, F16, F16, True), (3000, 16, F32, F32, False), (6, 8192, BF, BF, True),
    (5, 8200, F32, F16, False), (4, 4100, F16, F16, True), (7, 5001, F32, F32, True),
    (3, 20000, BF, BF, False), (100, 47, F32, F32, True), (5000, 100, BF, BF, False)])
def test_rms_norm_backward(rows, cols, tt, tg, stream, how):
    g = gen(rows + 7 * cols)
    t = wide(normal(g, rows, cols, t=tt, std=2.0), how)
    gy = wide(normal(g, rows, cols, t=tg), how)
    gt = wide(normal(g, rows, cols, t=tt), how) if stream else None
    w = normal(g, cols) + 1
    gx, gw = bg.rmsNormBackward(gy, t, w, eps=1e-5, gradTotal=gt)
    T, G, W = t.double(), gy.double(), w.double()
    s = (T.pow(2).mean(1, keepdim=True) + 1e-5).rsqrt()
    xh = T * s
    c = (G * W * xh).mean(1, keepdim=True)
    want = s * (G * W - xh * c)
    mag = s * ((G * W).abs() + xh.abs() * (G * W * xh).abs().mean(1, keepdim=True))
    if stream:
        want = want + gt.double()
        mag = mag + gt.double().abs()
    within(gx, want, U[tt] * want.abs() + (2 * cols + 32) * 2.0 ** -24 * mag + TINY[tt], "x")
    prod = (G * xh).abs().sum(0)
    within(gw, (G * xh).sum(0), (rows + cols + 32) * 2.0 ** -24 * prod, "weight")
    assert gx.dtype == tt and gw.dtype == w.dtype
    again = bg.rmsNormBackward(gy, t, w, eps=1e-5, gradTotal=gt)
    assert torch.equal(again[0], gx) and torch.equal(again[1], gw)


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------
def act64(z, act):
    """(act, act') in 64 bits."""
    p = 1 / (1 + torch.exp(-z))
    one = torch.ones_like(z)
    if act is None:
        return z, one
    if isinstance(act, tuple):
        name, a = act
        if name == "leaky_relu":
            return torch.where(z > 0, z, a * z), torch.where(z > 0, one, a * one)
        return torch.where(z > 0, z, a * torch.expm1(z)), torch.where(z > 0, one, a * torch.exp(z))
    if act == "relu":
        return z.clamp_min(0), (z > 0).double()
    if act == "sigmoid":
        return p, p * (1 - p)
    if act == "tanh":
        return torch.tanh(z), 1 - torch.tanh(z) ** 2
    if act == "silu":
        return z * p, p * (1 + z * (1 - p))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 0.134145 * z * z)


SLOPE = 1.2     # |act'| of every activation above
BEND = 1.2      # |act''| where it exists
ACT_F32 = 24 * 2.0 ** -24  # an f32 activation: a few roundings and exp's two ulps


def acc(k):
    return (k / 16 + 16) * 2.0 ** -22


def eight(g, rows, cols, std):
    x = normal(g, rows, cols, std=std)
    s = x.abs().amax(1).clamp_min(1e-6) / 448 if cols else torch.ones(rows, device="cuda")
    return (x / s[:, None]).to(F8), s


def operand(g, rows, cols, t, std=1.0):
    if t == F8:
        q, s = eight(g, rows, cols, std)
        return q, s, q.double() * s.double()[:, None]
    x = normal(g, rows, cols, t=t, std=std)
    return x, None, x.double()


PRODUCTS = [  # m, k, n, type, act, bias, residual, out
    (1, 16, 16, BF, None, None, None, BF), (1, 1024, 300, F16, "silu", F16, F32, F32),
    (5, 64, 47, BF, "gelu", BF, None, BF), (130, 100, 256, F16, "relu", F32, F16, F16),
    (257, 256, 513, BF, "tanh", None, BF, F32), (64, 1433, 16, BF, ("elu", 1.0), BF, None, F32),
    (1000, 72, 1000, F16, ("leaky_relu", 0.2), None, F32, F16),
    (300, 4096, 264, BF, None, None, F32, F32), (3, 7, 5, BF, "sigmoid", F32, None, BF),
    (200, 160, 96, F8, "gelu", BF, BF, BF), (129, 1040, 300, F8, None, None, F32, F32),
    (40, 250, 33, F8, "silu", None, None, BF), (20000, 64, 640, BF, "relu", BF, None, BF),
    (2, 1, 1, F16, None, None, None, F32), (9, 0, 20, BF, "silu", BF, F32, F32),
    # few rows, and the first past them
    (2, 1040, 70, F8, "gelu", BF, F32, BF), (4, 2050, 33, BF, "relu", F32, BF, F32),
    (3, 75, 130, F8, None, None, None, F32), (4, 0, 9, F16, "sigmoid", F16, None, F16),
    (5, 2050, 33, BF, "relu", F32, BF, F32), (1, 4096, 4100, BF, "silu", None, None, BF),
    (8, 300, 64, F16, "tanh", None, F16, F16), (9, 300, 64, F16, "tanh", None, F16, F16),
    # small enough for the rows' kernel, and just not
    (1001, 40, 32, BF, "silu", BF, F32, F32), (1025, 40, 32, BF, "silu", BF, F32, F32),
    (21, 9000, 88, F16, None, None, None, F32), (21, 9100, 88, F16, None, None, None, F32),
    (700, 130, 120, F8, "gelu", BF, BF, BF),
    (5, 3501, 2700, BF, None, None, None, BF), (7, 301, 271, F8, "silu", BF, None, BF),
]


@pytest.mark.parametrize("how", ["plain", "rows", "odd", "vector"])
@pytest.mark.parametrize("m,k,n,t,act,tb,tr,to", PRODUCTS)
def test_linear_fused(m, k, n, t, act, tb, tr, to, how):
    g = gen(m + 3 * k + 5 * n)
    std = math.sqrt(2 / (k + n))
    x, xs, X = operand(g, m, k, t)
    w, ws, W = operand(g, n, k, t, std)
    if t != F8:
        x, w = wide(x, how), wide(w, how)
    b = None if tb is None else normal(g, n, t=tb, std=0.1)
    r = None if tr is None else wide(normal(g, m, n, t=tr), how)
    got = bg.linearFused(x, w, bias=b, act=act, residual=r, outType=to, xScale=xs, weightScale=ws)
    z = X @ W.t() + (0 if b is None else b.double())
    ez = acc(k) * (X.abs() @ W.abs().t()) + 2.0 ** -22 * z.abs()
    want = act64(z, act)[0]
    tol = SLOPE * ez + ACT_F32 * (want.abs() + z.abs())
    if r is not None:
        want = want + r.double()
    within(got, want, tol + (U[to] + U[F32]) * want.abs() + TINY[to], "out")
    assert got.dtype == to


@pytest.mark.parametrize("how", ["plain", "odd", "vector"])
@pytest.mark.parametrize("m,k,n,t,act,tb", [
    (1, 1024, 512, BF, "silu", None), (1, 16, 16, F16, "gelu", F16), (130, 100, 47, BF, "silu", F32),
    (257, 256, 513, F16, "sigmoid", None), (40, 250, 33, BF, None, BF),
    (64, 1433, 160, BF, "relu", None), (300, 160, 96, F8, "silu", BF), (129, 1040, 300, F8, "gelu",
                                                                        None),
    (20000, 64, 320, BF, "tanh", None), (3, 5, 7, F16, ("elu", 1.0), None), (4, 0, 9, BF, "silu", BF),
    (1, 1040, 70, F8, "gelu", BF), (2, 300, 40, F8, "silu", None), (4, 2050, 33, F16, "relu", F32),
    (5, 2050, 33, F16, "relu", F32), (8, 1040, 70, F8, "gelu", BF), (9, 1040, 70, F8, "gelu", BF)])
def test_gated_linear(m, k, n, t, act, tb, how):
    g = gen(m + 3 * k + 5 * n)
    std = math.sqrt(2 / (k + n))
    x, xs, X = operand(g, m, k, t)
    wg, gs, WG = operand(g, n, k, t, std)
    wu, us, WU = operand(g, n, k, t, std)
    if t != F8:
        x, wg, wu = wide(x, how), wide(wg, how), wide(wu, how)
    bg_ = None if tb is None else normal(g, n, t=tb, std=0.1)
    bu = None if tb is None else normal(g, n, t=tb, std=0.1)
    got = bg.gatedLinear(x, wg, wu, biasGate=bg_, biasUp=bu, act=act, xScale=xs, gateScale=gs,
                         upScale=us)
    zg = X @ WG.t() + (0 if bg_ is None else bg_.double())
    zu = X @ WU.t() + (0 if bu is None else bu.double())
    eg = acc(k) * (X.abs() @ WG.abs().t()) + 2.0 ** -22 * zg.abs()
    eu = acc(k) * (X.abs() @ WU.abs().t()) + 2.0 ** -22 * zu.abs()
    a = act64(zg, act)[0]
    want = a * zu
    to = BF if t == F8 else t
    tol = (SLOPE * eg + ACT_F32 * (a.abs() + zg.abs())) * (zu.abs() + eu) + a.abs() * eu
    within(got, want, tol + (U[to] + U[F32]) * want.abs() + TINY[to], "out")
    assert got.dtype == to


@pytest.mark.parametrize("how", ["plain", "odd", "vector"])
@pytest.mark.parametrize("m,k,n,t,act,tb", [
    (1, 16, 16, BF, None, None), (1, 1024, 300, F16, "silu", F16), (5, 64, 47, BF, "gelu", BF),
    (130, 100, 256, F16, None, F32), (257, 256, 513, BF, "tanh", None),
    (3000, 256, 47, F16, "gelu", F16), (64, 1433, 16, BF, ("elu", 1.0), BF),
    (20011, 64, 640, BF, None, BF), (3, 7, 5, BF, "sigmoid", F32), (0, 8, 8, BF, "silu", BF),
    (6, 0, 9, BF, "silu", BF)])
def test_linear_fused_backward(m, k, n, t, act, tb, how):
    g = gen(m + 3 * k + 5 * n)
    std = math.sqrt(2 / (k + n))
    x, w = wide(normal(g, m, k, t=t), how), wide(normal(g, n, k, t=t, std=std), how)
    b = None if tb is None else normal(g, n, t=tb, std=0.1)
    go = wide(normal(g, m, n, t=t), how)
    gx, gw, gb = bg.linearFusedBackward(go, x, w, bias=b, act=act)
    X, W, G = x.double(), w.double(), go.double()
    z = X @ W.t() + (0 if b is None else b.double())
    ez = acc(k) * (X.abs() @ W.abs().t()) + 2.0 ** -22 * z.abs()
    d = act64(z, act)[1]
    dz = G * d
    # dz's own rounding, and what z's error does to it
    edz = torch.zeros_like(dz) if act is None else \
        U[t] * dz.abs() + G.abs() * (BEND * ez + ACT_F32 * (1 + z.abs())) + TINY[t]
    check_grads(t, X, [W], [dz], [edz], gx, [gw])
    if b is None:
        assert gb is None
    else:
        tol = edz.sum(0) + m * 2.0 ** -24 * dz.abs().sum(0) + U[tb] * dz.sum(0).abs() + TINY[tb]
        within(gb, dz.sum(0), tol, "bias")
    again = bg.linearFusedBackward(go, x, w, bias=b, act=act)
    assert torch.equal(again[0], gx) and torch.equal(again[1], gw)


def check_grads(t, X, W, dz, edz, gx, gw):
    m = X.shape[0]
    n = W[0].shape[0]
    want = sum(z @ w for z, w in zip(dz, W))
    tol = sum((e + acc(len(W) * n) * (z.abs() + e)) @ w.abs() for z, e, w in zip(dz, edz, W))
    within(gx, want, tol + (U[t] + U[F32]) * want.abs() + TINY[t], "x")
    for i, (z, e, g) in enumerate(zip(dz, edz, gw)):
        want = z.t() @ X
        tol = (e + acc(m) * (z.abs() + e)).t() @ X.abs()
        within(g, want, tol + (U[t] + U[F32]) * want.abs() + TINY[t], f"weight {i}")
        assert g.dtype == t


@pytest.mark.parametrize("how", ["plain", "odd", "vector"])
@pytest.mark.parametrize("m,k,n,t,act,tb", [
    (1, 64, 64, BF, "silu", None), (5, 100, 47, F16, "gelu", F16), (130, 256, 300, BF, "silu", F32),
    (2500, 128, 257, F16, "sigmoid", F16), (33, 1433, 24, BF, None, BF),
    (20011, 64, 128, BF, "silu", BF), (0, 8, 8, BF, "silu", BF), (6, 0, 9, BF, "silu", BF)])
def test_gated_linear_backward(m, k, n, t, act, tb, how):
    g = gen(m + 3 * k + 5 * n)
    std = math.sqrt(2 / (k + n))
    x = wide(normal(g, m, k, t=t), how)
    wg, wu = wide(normal(g, n, k, t=t, std=std), how), wide(normal(g, n, k, t=t, std=std), how)
    b0 = None if tb is None else normal(g, n, t=tb, std=0.1)
    b1 = None if tb is None else normal(g, n, t=tb, std=0.1)
    go = wide(normal(g, m, n, t=t), how)
    gx, gwg, gwu, g0, g1 = bg.gatedLinearBackward(go, x, wg, wu, biasGate=b0, biasUp=b1, act=act)
    X, WG, WU, G = x.double(), wg.double(), wu.double(), go.double()
    zg = X @ WG.t() + (0 if b0 is None else b0.double())
    zu = X @ WU.t() + (0 if b1 is None else b1.double())
    eg = acc(k) * (X.abs() @ WG.abs().t()) + 2.0 ** -22 * zg.abs()
    eu = acc(k) * (X.abs() @ WU.abs().t()) + 2.0 ** -22 * zu.abs()
    a, d = act64(zg, act)
    dg, du = G * zu * d, G * a
    edg = U[t] * dg.abs() + TINY[t] + G.abs() * (
        eu * SLOPE + (zu.abs() + eu) * (BEND * eg + ACT_F32 * (1 + zg.abs())))
    edu = U[t] * du.abs() + TINY[t] + G.abs() * (SLOPE * eg + ACT_F32 * (a.abs() + zg.abs()))
    check_grads(t, X, [WG, WU], [dg, du], [edg, edu], gx, [gwg, gwu])
    for got, z, e in ((g0, dg, edg), (g1, du, edu)):
        if tb is None:
            assert got is None
        else:
            tol = e.sum(0) + m * 2.0 ** -24 * z.abs().sum(0) + U[tb] * z.sum(0).abs() + TINY[tb]
            within(got, z.sum(0), tol, "bias")


def test_gated_gradient_against_differences():
    """The gradient along a direction against central differences of the
    forward itself, from inputs on a grid that bf16 holds."""
    g = gen(8)
    m, k, n, h = 24, 72, 40, 2.0 ** -5
    def grid(*s):
        return torch.randint(-32, 33, s, device="cuda", generator=g).double() / 32
    x, dx = grid(m, k), torch.sign(grid(m, k)) * 1.0
    wg, wu = grid(n, k) / 8, grid(n, k) / 8
    c = normal(g, m, n, t=BF)

    def f64(v):
        return (c.double() * act64(v @ wg.t(), "silu")[0] * (v @ wu.t())).sum()

    def own(v):
        assert torch.equal(v.to(BF).double(), v)
        out = bg.gatedLinear(v.to(BF), wg.to(BF), wu.to(BF), outType=F32)
        return (c.double() * out.double()).sum()

    grad = bg.gatedLinearBackward(c, x.to(BF), wg.to(BF), wu.to(BF))[0].double()
    diff = (own(x + h * dx) - own(x - h * dx)) / (2 * h)
    true = (f64(x + h * dx) - f64(x - h * dx)) / (2 * h)
    e = 1e-4
    exact = (f64(x + e * dx) - f64(x - e * dx)) / (2 * e)  # 64 bits: error of order e^2
    # forward noise over h, the curvature that the wide difference sees, the
    # gradient's roundings (dg, du, dx: three halves of a step, added up)
    a, u = act64(x @ wg.t(), "silu")[0], x @ wu.t()
    noise = (c.double().abs() * (a.abs() + 1) * (u.abs() + 1)).sum() * acc(k) * 8 / h
    rough = 3 * U[BF] * (c.double().abs() * (u.abs() * SLOPE) @ wg.abs() +
                         c.double().abs() * a.abs() @ wu.abs()).sum()
    assert abs((diff - true).item()) <= noise.item()
    assert abs((grad * dx).sum().item() - exact.item()) <= rough.item() + 1e-4 * abs(exact.item())


# ---------------------------------------------------------------------------
# choice head
# ---------------------------------------------------------------------------
def choices(g, rows, cols, t, mask):
    x = normal(g, rows, cols, t=t, std=3.0)
    m = None
    if mask == "columns":
        m = torch.rand(cols, device="cuda", generator=g) < 0.3
    elif mask == "rows":
        m = torch.rand(rows, cols, device="cuda", generator=g) < 0.5
        m[rows // 2] = True  # nothing left
        m = m.to(torch.uint8)
    tg = torch.randint(0, cols, (rows,), device="cuda", generator=g)
    if rows > 2:
        tg[1] = -1
    return x, m, tg


def left64(x, m):
    v = x.double()
    return v if m is None else v.masked_fill(m.bool().expand(v.shape), -math.inf)


def head64(x, m, tg, top):
    v = left64(x, m)
    lse = torch.logsumexp(v, 1)
    some = lse > -math.inf
    lp = torch.where(v > -math.inf, v - lse.masked_fill(~some, 0)[:, None], -math.inf)
    p = torch.where(v > -math.inf, lp.exp(), 0)
    ent = -(p * lp.masked_fill(p == 0, 0)).sum(1)
    t = tg.long()
    logp = lp.gather(1, t.clamp_min(0)[:, None])[:, 0].masked_fill(t < 0, 0)
    vv = v.cpu().numpy()
    ids = np.full((v.shape[0], top), -1, np.int64)
    tl = np.full((v.shape[0], top), -np.inf)
    for r in range(v.shape[0]):
        order = np.lexsort((np.arange(v.shape[1]), -vv[r]))[:top]
        order = order[vv[r][order] > -np.inf]
        ids[r, :order.size] = order
        tl[r, :order.size] = lp[r].cpu().numpy()[order]
    return lp, p, lse, logp, ent, ids, torch.from_numpy(tl).cuda()


HEADS = [(1, 1, F32, 1), (3, 2, BF, 5), (100, 47, F32, 3), (9, 1000, F16, 32), (4, 1025, BF, 20),
         (5, 5001, F16, 20), (2, 40000, F32, 7), (1, 300007, BF, 32), (700, 3001, F32, 0),
         (3, 200, BF, 32), (1, 20000, F32, 20), (513, 8, F16, 8)]


@pytest.mark.parametrize("how", ["plain", "odd"])
@pytest.mark.parametrize("mask", [None, "columns", "rows"])
@pytest.mark.parametrize("rows,cols,t,top", HEADS)
def test_log_probs(rows, cols, t, top, mask, how):
    g = gen(rows + cols)
    x, m, tg = choices(g, rows, cols, t, mask)
    x = wide(x, how)
    if m is not None and m.dim() == 2 and how == "odd":
        big = torch.ones(rows, cols + 5, dtype=m.dtype, device="cuda")
        big[:, 2:-3] = m
        m = big[:, 2:-3]
    logp, ent, lse, ids, tl = bg.logProbs(x, tg, mask=m, topK=top)
    lp, p, lse_w, logp_w, ent_w, ids_w, tl_w = head64(x, m, tg, top)
    # f32 sums of cols terms, each exp within a few ulps of its argument's
    # size (arguments to 40 or so below the maximum carry their weight)
    tol = (math.log2(cols + 1) * 8 + 64) * 2.0 ** -24
    big = x.double().abs().amax().clamp_min(1)
    within(lse, lse_w, tol * (1 + big), "lse")
    within(logp, logp_w, tol * (1 + 2 * big), "logp")
    within(ent, ent_w, tol * (1 + ent_w.abs() + math.log(cols + 1)), "entropy")
    if top:
        assert np.array_equal(ids.cpu().numpy(), ids_w)
        within(tl, tl_w, tol * (1 + 2 * big), "top")
    else:
        assert ids is None and tl is None
    gl, gh = normal(g, rows), normal(g, rows)
    got = bg.logProbsBackward(x, tg, lse, ent, gl, gradEntropy=gh, mask=m)
    G, H = gl.double()[:, None], gh.double()[:, None]
    hit = torch.zeros_like(lp)
    at = tg.long()
    rows_on = (at >= 0).nonzero()[:, 0]
    hit[rows_on, at[rows_on]] = 1
    G = torch.where(at[:, None] >= 0, G, 0)
    safe = lp.masked_fill(p == 0, 0)
    leftm = (left64(x, m) > -math.inf).double()
    want = p * (-G - H * (safe + ent_w[:, None])) + G * hit * leftm
    mag = p * (G.abs() + H.abs() * (safe.abs() + ent_w[:, None] + 1)) * (1 + safe.abs())
    tolg = U[t] * want.abs() + tol * (2 + 4 * big) * mag + U[F32] * (G * hit).abs() + TINY[t]
    within(got, want, tolg, "logits")
    assert got.dtype == t
    only = bg.logProbsBackward(x, tg, lse, ent, gl, mask=m)
    within(only, -p * G + G * hit * leftm,
           U[t] * (p * G.abs() + (G * hit).abs()) + tol * (2 + 4 * big) * mag + TINY[t], "no entropy")


def test_log_probs_ties_lowest_values_and_not_finite():
    low = torch.finfo(BF).min
    x = torch.full((8, 3000), 1.0, device="cuda", dtype=BF)  # all equal: lowest index first
    x[1] = low                     # every choice at the type's lowest value
    x[2, :] = low
    x[2, 17] = 100.0               # ... beside an ordinary one
    x[3, 5] = math.nan
    x[4, :] = -math.inf            # nothing left
    x[5, 2999] = 2.0
    x[6, 0] = math.inf
    x[7, 7::2] = -math.inf
    t = torch.tensor([0, 1, 17, 1, 2, 2999, 3, 9], device="cuda")
    mask = torch.zeros(8, 3000, dtype=torch.bool, device="cuda")
    x[0, 100] = math.nan           # a NaN under a mask is not looked at
    x[0, 101] = math.inf
    mask[0, 100] = mask[0, 101] = True
    logp, ent, lse, ids, top = bg.logProbs(x, t, mask=mask, topK=4)
    n = math.log(2998)
    assert abs(logp[0].item() + n) < 1e-5 and abs(ent[0].item() - n) < 1e-5
    assert ids[0].tolist() == [0, 1, 2, 3]
    assert abs(logp[1].item() + math.log(3000)) < 1e-5 and abs(ent[1].item() - math.log(3000)) < 1e-5
    assert ids[1].tolist() == [0, 1, 2, 3]
    assert logp[2] == 0 and ent[2] == 0 and ids[2].tolist() == [17, 0, 1, 2]
    assert logp[3].isnan() and ent[3].isnan() and lse[3].isnan()
    assert ids[3].tolist() == [0, 1, 2, 3] and top[3].isnan().all()
    assert logp[4] == -math.inf and ent[4] == 0 and lse[4] == -math.inf
    assert ids[4].tolist() == [-1] * 4 and (top[4] == -math.inf).all()
    assert ids[5].tolist() == [2999, 0, 1, 2]
    assert logp[6].isnan() and ids[6].tolist() == [0, 1, 2, 3]
    assert logp[7] == -math.inf and torch.isfinite(ent[7])
    g = bg.logProbsBackward(x, t, lse, ent, torch.ones(8, device="cuda"), mask=mask)
    assert torch.equal(g[4], torch.zeros_like(g[4])) and g[0, 100] == 0 and g[0, 101] == 0
    assert torch.isfinite(g[[0, 1, 2, 4, 5, 7]].float()).all() and g[3].isnan().any()
    # p = 1/3000 each, though the lse of this row cannot hold log 3000
    p = 1 / 3000
    assert abs(g[1, 0].item() + p) < 2 * U[BF] * p and abs(g[1, 1].item() - 1 + p) < 2 * U[BF]
    # no columns at all
    logp, ent, lse, ids, top = bg.logProbs(torch.empty(2, 0, device="cuda"),
                                           torch.full((2,), -1, device="cuda"), topK=2)
    assert logp.tolist() == [0, 0] and ent.tolist() == [0, 0] and (ids == -1).all()


@pytest.mark.parametrize("cols", [40, 700, 3000])
@pytest.mark.parametrize("at", [500.0, -3e4])
def test_log_probs_far_from_zero(cols, at):
    """Rows whose log-sum-exp is large, masks among them: the gradient does not
    lean on its last bits."""
    g = gen(cols)
    x = normal(g, 6, cols) + at
    m = torch.rand(6, cols, device="cuda", generator=g) < 0.4
    m[5] = True
    t = torch.zeros(6, device="cuda", dtype=torch.int64)
    logp, ent, lse, _, _ = bg.logProbs(x, t, mask=m)
    lp, p, lse_w, logp_w, ent_w, _, _ = head64(x, m, t, 1)
    within(logp, logp_w, 2.0 ** -18 * (1 + logp_w.abs().nan_to_num(posinf=0)), "logp")
    within(ent, ent_w, 2.0 ** -18 * (1 + ent_w), "entropy")
    gl = torch.ones(6, device="cuda")
    d = bg.logProbsBackward(x, t, lse, ent, gl, mask=m)
    hit = torch.zeros_like(p)
    hit[:, 0] = (left64(x, m)[:, 0] > -math.inf).double()
    # p from m and S summed again in f32: 2^-18 of it is more than their error
    within(d, hit - p, 2.0 ** -18 * p + 2.0 ** -23, "logits")


def test_gated_with_one_bias():
    g = gen(77)
    x, wg, wu = normal(g, 40, 64, t=BF), normal(g, 48, 64, t=BF), normal(g, 48, 64, t=BF)
    b, zero = normal(g, 48, t=BF), torch.zeros(48, device="cuda", dtype=BF)
    go = normal(g, 40, 48, t=BF)
    for rows in (1, 40):
        xs, gs = x[:rows], go[:rows]
        assert torch.equal(bg.gatedLinear(xs, wg, wu, biasGate=b),
                           bg.gatedLinear(xs, wg, wu, biasGate=b, biasUp=zero))
        assert torch.equal(bg.gatedLinear(xs, wg, wu, biasUp=b),
                           bg.gatedLinear(xs, wg, wu, biasGate=zero, biasUp=b))
        one = bg.gatedLinearBackward(gs, xs, wg, wu, biasUp=b)
        two = bg.gatedLinearBackward(gs, xs, wg, wu, biasGate=zero, biasUp=b)
        assert one[3] is None
        for i in (0, 1, 2, 4):
            assert torch.equal(one[i], two[i])


def test_long_contractions_take_the_wide_tiles():
    """512-column tiles (operands of both majors, ragged edges) against the
    64-bit product."""
    g = gen(5)
    # 18 x 16 tiles of 256 columns on 74 pairs: four rounds, two of 512 columns
    m, k, n = 4500, 4088, 4088
    x, w = normal(g, m, k, t=BF), normal(g, n, k, t=BF, std=k ** -0.5)
    go = normal(g, m, n, t=BF)
    out = bg.linearFused(x, w)
    want = x.double() @ w.double().t()
    S = x.double().abs() @ w.double().abs().t()
    within(out, want, acc(k) * S + (U[BF] + U[F32]) * want.abs(), "out")
    gx, gw, _ = bg.linearFusedBackward(go, x, w)
    G = go.double()
    want = G @ w.double()
    within(gx, want, acc(n) * (G.abs() @ w.double().abs()) + (U[BF] + U[F32]) * want.abs(), "x")
    want = G.t() @ x.double()
    within(gw, want, acc(m) * (G.abs().t() @ x.double().abs()) + (U[BF] + U[F32]) * want.abs(), "w")
    test_gated_linear(m, k, 2040, BF, "silu", BF, "plain")
    test_gated_linear(m, 8200, 2036, F8, "gelu", None, "plain")
    test_gated_linear_backward(m, k, 2040, F16, "gelu", F16, "plain")


def test_log_probs_target_out_of_range():
    ctx = bg.get_context()
    ctx.synchronize()
    x = torch.zeros(3, 50, device="cuda")
    for bad in (50, -2, 2 ** 32 + 5):
        t = torch.tensor([1, bad, 49], device="cuda")
        logp, ent, lse, _, _ = bg.logProbs(x, t)
        assert logp[1].isnan() and torch.isfinite(logp[[0, 2]]).all()
        with pytest.raises(bg.BGNNIndexError):
            ctx.synchronize()
        ctx.synchronize()
        bg.logProbsBackward(x, t, lse, ent, torch.ones(3, device="cuda"))
        with pytest.raises(bg.BGNNIndexError):
            ctx.synchronize()


def test_log_probs_gradient_against_differences():
    g = gen(3)
    x = normal(g, 5, 400)
    m = torch.rand(400, device="cuda", generator=g) < 0.2
    t = torch.arange(5, device="cuda") * 7
    m[t] = False
    gl, gh = normal(g, 5), normal(g, 5)
    d = torch.sign(normal(g, 5, 400))

    def f(v, own):
        if own:
            lp, h, _, _, _ = bg.logProbs(v.float(), t, mask=m)
        else:
            _, _, _, lp, h, _, _ = head64(v, m, t, 1)
        return (gl.double() * lp.double() + gh.double() * h.double()).sum()

    lp, h, lse, _, _ = bg.logProbs(x, t, mask=m)
    grad = bg.logProbsBackward(x, t, lse, h, gl, gradEntropy=gh, mask=m)
    e, X = 2.0 ** -6, x.double()
    own = (f((X + e * d).float(), True) - f((X - e * d).float(), True)) / (2 * e)
    ref = (f((X + e * d).float().double(), False) - f((X - e * d).float().double(), False)) / (2 * e)
    # f32 figures of size 10 to 2^-20 relative, over 2 e
    assert abs(own.item() - ref.item()) <= 5 * 2 * 10 * 2.0 ** -20 / (2 * e) * 2
    small = 1e-5
    ref = (f(X + small * d, False) - f(X - small * d, False)) / (2 * small)
    assert abs((grad.double() * d).sum().item() - ref.item()) <= 1e-4 * (1 + abs(ref.item()))


# ---------------------------------------------------------------------------
# together, on streams, in graphs
# ---------------------------------------------------------------------------
def block(stream_in, p, out8):
    """norm -> gated -> product back onto the f32 stream -> norm -> scores -> head."""
    y, total, s = bg.rmsNorm(stream_in["x"], p["w1"], residual=stream_in["r"],
                             outType=F8 if out8 else BF)
    if out8:
        h = bg.gatedLinear(y, p["g8"], p["u8"], xScale=s, gateScale=p["gs"], upScale=p["us"])
    else:
        h = bg.gatedLinear(y, p["g"], p["u"])
    stream = bg.linearFused(h, p["d"], residual=total, outType=F32)
    y, _, _ = bg.rmsNorm(stream, p["w2"], outType=BF)
    logits = bg.linearFused(y, p["c"], bias=p["b"])
    logp, ent, lse, ids, top = bg.logProbs(logits, stream_in["t"], topK=3)
    gl = bg.logProbsBackward(logits, stream_in["t"], lse, ent, stream_in["gl"])
    gy, gc, gb = bg.linearFusedBackward(gl, y, p["c"], bias=p["b"])
    gs, gw2 = bg.rmsNormBackward(gy.float(), stream, p["w2"])
    gh, gd, _ = bg.linearFusedBackward(gs.to(BF), h, p["d"])
    outs = [total, stream, logp, ent, ids, top, gc, gb, gw2, gd]
    if not out8:
        gy, gg, gu, _, _ = bg.gatedLinearBackward(gh, y := bg.rmsNorm(total, p["w1"], outType=BF)[0],
                                                  p["g"], p["u"])
        gx, gw1 = bg.rmsNormBackward(gy, total, p["w1"], gradTotal=gs)
        outs += [gg, gu, gx, gw1]
    return outs


def block_params(g, k, f, c):
    p = {"w1": normal(g, k) * 0.1 + 1, "w2": normal(g, k) * 0.1 + 1,
         "g": normal(g, f, k, t=BF, std=0.1), "u": normal(g, f, k, t=BF, std=0.1),
         "d": normal(g, k, f, t=BF, std=0.1), "c": normal(g, c, k, t=BF, std=0.1),
         "b": normal(g, c, t=BF)}
    p["g8"], p["gs"] = eight(g, f, k, 0.1)
    p["u8"], p["us"] = eight(g, f, k, 0.1)
    return p


def block_input(g, m, k, c):
    return {"x": normal(g, m, k), "r": normal(g, m, k),
            "t": torch.randint(0, c, (m,), device="cuda", generator=g),
            "gl": torch.full((m,), -1.0 / m, device="cuda")}


@pytest.mark.parametrize("out8", [False, True])
def test_block_together_on_streams_and_in_graphs(out8):
    g = gen(11)
    k, f, c = 72, 200, 47
    p = block_params(g, k, f, c)
    a, b = block_input(g, 333, k, c), block_input(g, 333, k, c)
    eager_a, eager_b = block(a, p, out8), block(b, p, out8)
    # plain 64-bit forward of the stream (bf16 chain: each rounding is 2^-9)
    if not out8:
        t = (a["x"] + a["r"]).double()
        y = t * (t.pow(2).mean(1, keepdim=True) + 1e-6).rsqrt() * p["w1"].double()
        h = act64(y @ p["g"].double().t(), "silu")[0] * (y @ p["u"].double().t())
        want = t + h @ p["d"].double().t()
        err = (eager_a[1].double() - want).norm() / want.norm()
        assert err < 4 * U[BF]
    # another stream
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = block(a, p, out8)
    torch.cuda.current_stream().wait_stream(side)
    for u, v in zip(eager_a, on_side):
        assert torch.equal(u, v)
    # two graphs of the same operators, replayed in turn and again on new inputs
    ga = bg.CapturedForward(lambda: block(a, p, out8))
    gb = bg.CapturedForward(lambda: block(b, p, out8))
    for _ in range(3):
        ra, rb = ga(), gb()
    torch.cuda.synchronize()
    for u, v in zip(eager_a + eager_b, ra + rb):
        assert torch.equal(u, v)
    a["x"].copy_(b["x"]), a["r"].copy_(b["r"]), a["t"].copy_(b["t"])
    ra = ga()
    for u, v in zip(eager_b, ra):
        assert torch.equal(u, v)
    # both at once
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    s1.wait_stream(torch.cuda.current_stream())
    s2.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(s1):
            ra = ga()
        with torch.cuda.stream(s2):
            rb = gb()
    torch.cuda.synchronize()
    for u, v in zip(eager_b + eager_b, ra + rb):
        assert torch.equal(u, v)
    ga.close(), gb.close()


def test_rows_behind_the_last_stay_as_they_were():
    """The C entry points write what they say and nothing behind it."""
    from browsergnn_b200.backend import ptr

    ctx = bg.get_context()
    g = gen(5)
    m, k, n, ld = 130, 40, 36, 48
    x, w = normal(g, m, k, t=BF), normal(g, n, k, t=BF)
    out = torch.full((m + 2, ld), 7.0, dtype=BF, device="cuda")
    ctx.call("bgnn_linear_fused", 1, ptr(x), k, None, ptr(w), k, None, m, k, n, 0, None, 0, 0.0, 0,
             None, 0, 1, ptr(out), ld)
    assert (out[m:] == 7).all() and (out[:, n:] == 7).all()
    assert torch.equal(out[:m, :n], bg.linearFused(x, w))
    # in place on the residual stream
    r = normal(g, m, n)
    want = bg.linearFused(x, w, residual=r, outType=F32)
    ctx.call("bgnn_linear_fused", 1, ptr(x), k, None, ptr(w), k, None, m, k, n, 0, None, 0, 0.0, 0,
             ptr(r), n, 0, ptr(r), n)
    assert torch.equal(r, want)
    with pytest.raises(bg.BGNNError, match="INVALID_ARG"):
        ctx.call("bgnn_linear_fused", 1, ptr(x), k - 1, None, ptr(w), k, None, m, k, n, 0, None, 0,
                 0.0, 0, None, 0, 1, ptr(out), ld)
    with pytest.raises(bg.BGNNError, match="e4m3"):
        ctx.call("bgnn_linear_fused", 0, ptr(x), k, None, ptr(w), k, None, m, k, n, 0, None, 0, 0.0,
                 0, None, 0, 1, ptr(out), ld)
