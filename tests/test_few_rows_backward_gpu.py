"""The products' gradients for few rows (four, or eight of up to 512 columns): dz
is not rounded on the way."""

import pytest
import torch

import browsergnn_b200 as bg
from tests.test_blocks_gpu import (ACT_F32, BEND, BF, F16, F32, SLOPE, TINY, U, acc, act64, gen, normal,
                                   wide, within)

pytestmark = pytest.mark.gpu


def check(t, X, W, dz, edz, gx, gw, tb, gb):
    """edz: dz's error, the activation's and z's; no rounding of dz."""
    n = X.shape[0], W[0].shape[0]
    want = sum(z @ w for z, w in zip(dz, W))
    # f32 sums over n (both products') in any order, and dz's error
    tol = sum((e + (2 * n[1] + 8) * 2.0 ** -24 * (z.abs() + e)) @ w.abs()
              for z, e, w in zip(dz, edz, W))
    within(gx, want, tol + U[t] * want.abs() + TINY[t], "x")
    for i in range(len(W)):
        want = dz[i].t() @ X
        tol = (edz[i] + (n[0] + 2) * 2.0 ** -24 * (dz[i].abs() + edz[i])).t() @ X.abs()
        within(gw[i], want, tol + U[t] * want.abs() + TINY[t], f"weight {i}")
        if tb is not None:
            want = dz[i].sum(0)
            within(gb[i], want, edz[i].sum(0) + 8 * 2.0 ** -24 * dz[i].abs().sum(0) +
                   U[tb] * want.abs() + TINY[tb], f"bias {i}")
        else:
            assert gb[i] is None


SHAPES = [(1, 1, 1), (1, 16, 16), (2, 85, 36), (3, 87, 71), (8, 60, 964), (1, 937, 203), (4, 64, 3000),
          (5, 264, 47), (6, 0, 9), (7, 500, 8), (8, 512, 520), (4, 4096, 520), (1, 1024, 4096)]


@pytest.mark.parametrize("how", ["plain", "odd", "vector"])
@pytest.mark.parametrize("t,act,tb", [(BF, "silu", None), (F16, "gelu", F16), (BF, "tanh", F32),
                                      (F16, ("elu", 1.0), BF)])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear(m, k, n, t, act, tb, how):
    g = gen(m + 3 * k + 5 * n)
    x, w = (wide(v, how) for v in (normal(g, m, k, t=t), normal(g, n, k, t=t, std=(2 / (k + n)) ** 0.5)))
    go = wide(normal(g, m, n, t=t), how)
    b = None if tb is None else normal(g, n, t=tb, std=0.1)
    gx, gw, gb = bg.linearFusedBackward(go, x, w, bias=b, act=act)
    X, W, G = x.double(), w.double(), go.double()
    z = X @ W.t() + (0 if b is None else b.double())
    ez = acc(k) * (X.abs() @ W.abs().t()) + 2.0 ** -22 * z.abs()
    dz = G * act64(z, act)[1]
    edz = G.abs() * (BEND * ez + ACT_F32 * (1 + z.abs())) + 2.0 ** -24 * dz.abs()
    check(t, X, [W], [dz], [edz], gx, [gw], tb, [gb])
    again = bg.linearFusedBackward(go, x, w, bias=b, act=act)
    assert torch.equal(again[0], gx) and torch.equal(again[1], gw)


@pytest.mark.parametrize("how", ["plain", "odd", "vector"])
@pytest.mark.parametrize("t,act,tb", [(BF, "silu", None), (F16, "sigmoid", F16), (BF, None, F32)])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_gated(m, k, n, t, act, tb, how):
    g = gen(m + 3 * k + 5 * n)
    std = (2 / (k + n)) ** 0.5
    x, wg, wu = (wide(v, how) for v in (normal(g, m, k, t=t), normal(g, n, k, t=t, std=std),
                                        normal(g, n, k, t=t, std=std)))
    go = wide(normal(g, m, n, t=t), how)
    b, c = (None, None) if tb is None else (normal(g, n, t=tb, std=0.1), normal(g, n, t=tb, std=0.1))
    gx, gwg, gwu, gbg, gbu = bg.gatedLinearBackward(go, x, wg, wu, biasGate=b, biasUp=c, act=act)
    X, P, Q, G = x.double(), wg.double(), wu.double(), go.double()
    z, u = X @ P.t(), X @ Q.t()
    if tb is not None:
        z, u = z + b.double(), u + c.double()
    ez, eu = (acc(k) * (X.abs() @ w.abs().t()) + 2.0 ** -22 * v.abs() for w, v in ((P, z), (Q, u)))
    a, d = act64(z, act)
    dg, du = G * u * d, G * a
    edg = G.abs() * (eu * SLOPE + (u.abs() + eu) * (BEND * ez + ACT_F32 * (1 + z.abs()))) + \
        2.0 ** -23 * dg.abs()
    edu = G.abs() * (SLOPE * ez + ACT_F32 * (a.abs() + z.abs())) + 2.0 ** -23 * du.abs()
    check(t, X, [P, Q], [dg, du], [edg, edu], gx, [gwg, gwu], tb, [gbg, gbu])


@pytest.mark.parametrize("t", [BF, F16])
def test_no_further_from_64_bits_than_its_rounding(t):
    """Norm-wise over one row at a time: with dz rounded to 16 bits a row's
    gradient was up to twice as far off as its own rounding.  A result rounded
    to nearest from f32 is off by its rounding and 2^-20 of the terms at most."""
    g = gen(5)
    for m, k, n in ((1, 58, 3614), (2, 51, 3075), (1, 42, 1455)):
        x, w = normal(g, m, k, t=t), normal(g, n, k, t=t, std=(2 / (k + n)) ** 0.5)
        u, go = normal(g, n, k, t=t, std=(2 / (k + n)) ** 0.5), normal(g, m, n, t=t)
        X, W, V, G = (v.double() for v in (x, w, u, go))
        z, y = X @ W.t(), X @ V.t()
        a, d = act64(z, "silu")
        for got, want in ((bg.linearFusedBackward(go, x, w, act="silu")[0], (G * d) @ W),
                          (bg.gatedLinearBackward(go, x, w, u)[0], (G * y * d) @ W + (G * a) @ V)):
            own = (want.to(t).double() - want).norm()
            assert (got.double() - want).norm() <= 1.02 * own


def test_results_that_are_not_asked_for():
    """NULL gradients through the C entry points."""
    g = gen(7)
    m, k, n = 3, 40, 24
    x, w, go = normal(g, m, k, t=BF), normal(g, n, k, t=BF), normal(g, m, n, t=BF)
    u = normal(g, n, k, t=BF)
    wx, ww, wb = bg.linearFusedBackward(go, x, w, bias=torch.zeros(n, device="cuda"), act="silu")
    ctx = bg.get_context()
    for only in range(3):
        out = [torch.full_like(v, 7.0) for v in (wx, ww, wb)]
        args = [out[i].data_ptr() if i == only else None for i in range(3)]
        ctx.call("bgnn_linear_fused_backward", 1, go.data_ptr(), n, x.data_ptr(), k, w.data_ptr(), k, m,
                 k, n, 0, None, 8, 0.0, *args)
        for i, (v, want) in enumerate(zip(out, (wx, ww, wb))):
            assert torch.equal(v, want) if i == only else (v == 7).all()
    b = torch.zeros(n, device="cuda")
    want = bg.gatedLinearBackward(go, x, w, u, biasGate=b, biasUp=b)
    for only in ((0,), (1, 2), (3,), (4,)):
        out = [torch.full_like(v, 7.0) for v in want]
        args = [out[i].data_ptr() if i in only else None for i in range(5)]
        ctx.call("bgnn_gated_linear_backward", 1, go.data_ptr(), n, x.data_ptr(), k, w.data_ptr(), k,
                 u.data_ptr(), k, m, k, n, 0, None, None, 8, 0.0, *args)
        for i, (v, e) in enumerate(zip(out, want)):
            assert torch.equal(v, e) if i in only else (v == 7).all()
