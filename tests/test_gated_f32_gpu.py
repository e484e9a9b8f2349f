"""gatedLinear with an f32 result over long contractions."""
import pytest
import torch

import browsergnn_b200 as bg
from tests.test_blocks_gpu import (ACT_F32, BF, F16, F32, SLOPE, U, acc, act64, eight, gen, normal, wide,
                                   within)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [BF, F16])
@pytest.mark.parametrize("m", [200, 20000])
def test_sums_do_not_lean_one_way(m, t):
    """Of positive terms, so that every addition that is cut short counts.

    Pieces of 512 products are summed by the tensor cores, 16 at a time: 32
    additions that may each lose up to a step, 2^-23 of the sum so far.  The 16
    pieces of 8,192 are added in f32, rounded to nearest: at most half a step
    each, 2^-24.  So a factor is within 32 * 2^-23 + 16 * 2^-24, their product
    within twice that and its own rounding.  (One accumulator over all 8,192
    would lose 512 steps' halves on average, 1.5e-5 a factor.)"""
    g = gen(m)
    k, n = 8192, 256

    def some(rows):
        return (torch.rand(rows, k, device="cuda", generator=g) / 2 + 0.5).to(t)

    x, wg, wu = some(m), some(n), some(n)
    got = bg.gatedLinear(x, wg, wu, act=None, outType=F32)
    want = (x.double() @ wg.double().t()) * (x.double() @ wu.double().t())
    within(got, want, want * (2 * (32 * 2.0 ** -23 + 16 * 2.0 ** -24) + U[F32]), "out")


@pytest.mark.parametrize("how", ["plain", "odd"])
@pytest.mark.parametrize("m,k,n,act,tb", [
    (1, 512, 40, "silu", None), (40, 24, 17, "gelu", F32), (300, 520, 130, "silu", BF),
    (257, 1433, 513, "tanh", None), (20000, 64, 640, "relu", F32), (129, 0, 300, "sigmoid", BF),
    (4500, 4104, 260, "silu", None), (1000, 512, 33, None, BF), (1000, 513, 65, "gelu", None)])
def test_shapes(m, k, n, act, tb, how):
    g = gen(m + k + n)
    std = (2 / (k + n)) ** 0.5
    x, wg, wu = (wide(v, how) for v in (normal(g, m, k, t=BF), normal(g, n, k, t=BF, std=std),
                                        normal(g, n, k, t=BF, std=std)))
    b, c = (None, None) if tb is None else (normal(g, n, t=tb), normal(g, n, t=tb))
    got = bg.gatedLinear(x, wg, wu, biasGate=b, biasUp=c, act=act, outType=F32)
    X, G, V = x.double(), wg.double(), wu.double()
    z, u = X @ G.t(), X @ V.t()
    if tb is not None:
        z, u = z + b.double(), u + c.double()
    ez, eu = (acc(k) * (X.abs() @ w.abs().t()) + 2.0 ** -22 * v.abs() for w, v in ((G, z), (V, u)))
    a = act64(z, act)[0]
    tol = (SLOPE * ez + ACT_F32 * (a.abs() + z.abs())) * (u.abs() + eu) + a.abs() * eu
    within(got, a * u, tol + 2 * U[F32] * (a * u).abs() + 1e-37, "out")


def test_eight_bits():
    g = gen(9)
    m, k, n = 700, 1500, 200
    (x, xs), (w, ws), (u, us) = eight(g, m, k, 1.0), eight(g, n, k, 0.05), eight(g, n, k, 0.05)
    got = bg.gatedLinear(x, w, u, act="silu", outType=F32, xScale=xs, gateScale=ws, upScale=us)
    X, W, V = (q.double() * s.double()[:, None] for q, s in ((x, xs), (w, ws), (u, us)))
    z, y = X @ W.t(), X @ V.t()
    ez, ey = (acc(k) * (X.abs() @ q.abs().t()) + 2.0 ** -22 * v.abs() for q, v in ((W, z), (V, y)))
    a = act64(z, "silu")[0]
    tol = (SLOPE * ez + ACT_F32 * (a.abs() + z.abs())) * (y.abs() + ey) + a.abs() * ey
    within(got, a * y, tol + 2 * U[F32] * (a * y).abs(), "out")
