"""The block operators where their operands lie in other ways than the other
tests have them: 8-bit rows with strides, results in the residual's buffer,
offsets past 32 bits, an SM budget, modules in a Sequential."""
import math

import pytest
import torch

import browsergnn_b200 as bg
from tests.test_blocks_gpu import (ACT_F32, BEND, BF, F16, F32, F8, SLOPE, TINY, U, acc, act64, eight,
                                   gen, normal, within)

pytestmark = pytest.mark.gpu


def wide8(x, how):
    """As wide, for 8 bits (whose fill is 448)."""
    pad = {"rows": 16, "odd": 3}[how]
    big = torch.full((x.shape[0], x.shape[1] + 2 * pad), 448.0, device="cuda").to(F8)
    big.view(torch.uint8)[:, pad:-pad] = x.view(torch.uint8)
    return big[:, pad:-pad]


@pytest.mark.parametrize("how", ["rows", "odd"])
@pytest.mark.parametrize("m,k,n", [(1, 40, 30), (3, 1040, 70), (9, 129, 600), (200, 160, 96),
                                   (700, 250, 513)])
def test_eight_bit_rows_apart(m, k, n, how):
    g = gen(m + k)
    x, xs = eight(g, m, k, 1.0)
    w, ws = eight(g, n, k, math.sqrt(2 / (k + n)))
    u, us = eight(g, n, k, math.sqrt(2 / (k + n)))
    X, W, V = (q.double() * s.double()[:, None] for q, s in ((x, xs), (w, ws), (u, us)))
    z, y = X @ W.t(), X @ V.t()
    ez, ey = (acc(k) * (X.abs() @ q.abs().t()) + 2.0 ** -22 * v.abs() for q, v in ((W, z), (V, y)))
    x, w, u = wide8(x, how), wide8(w, how), wide8(u, how)
    got = bg.linearFused(x, w, outType=F32, xScale=xs, weightScale=ws)
    within(got, z, ez + U[F32] * z.abs(), "linear")
    got = bg.gatedLinear(x, w, u, act="silu", xScale=xs, gateScale=ws, upScale=us)
    a = act64(z, "silu")[0]
    tol = (SLOPE * ez + ACT_F32 * (a.abs() + z.abs())) * (y.abs() + ey) + a.abs() * ey
    within(got, a * y, tol + (U[BF] + U[F32]) * (a * y).abs() + TINY[BF], "gated")


CODE = {F32: 0, BF: 1, F16: 2}


@pytest.mark.parametrize("t", [F32, BF])
@pytest.mark.parametrize("m,k,n", [(1, 64, 33), (5, 300, 70), (40, 24, 17), (300, 128, 257),
                                   (3000, 64, 520)])
@pytest.mark.parametrize("ld", [0, 1, 8])
def test_products_in_the_residuals_buffer(m, k, n, t, ld):
    g = gen(m + n)
    ld += n
    x, w = normal(g, m, k, t=BF), normal(g, n, k, t=BF)
    r = normal(g, m, ld, t=t)
    want = bg.linearFused(x, w, act="gelu", residual=r[:, :n], outType=t)
    behind = r[:, n:].clone()
    ctx = bg.get_context()
    ctx.call("bgnn_linear_fused", 1, x.data_ptr(), k, None, w.data_ptr(), k, None, m, k, n, 0, None,
             7, 0.0, CODE[t], r.data_ptr(), ld, CODE[t], r.data_ptr(), ld)
    assert torch.equal(r[:, :n], want) and torch.equal(r[:, n:], behind)


@pytest.mark.parametrize("tx,tr", [(F32, F32), (BF, BF), (F16, F32)])
@pytest.mark.parametrize("rows,cols", [(1, 5), (9, 3), (1000, 47), (300, 256), (33, 1433),
                                       (3, 20001)])
def test_sums_in_the_residuals_buffer(rows, cols, tx, tr):
    g = gen(rows + cols)
    x, r = normal(g, rows, cols, t=tx), normal(g, rows, cols, t=tr)
    w = normal(g, cols)
    want, total, _ = bg.rmsNorm(x, w, residual=r)
    out = torch.empty_like(x)
    bg.get_context().call("bgnn_rms_norm", CODE[tx], x.data_ptr(), cols, CODE[tr], r.data_ptr(), cols,
                          0, w.data_ptr(), rows, cols, 1e-6, r.data_ptr(), CODE[tx], out.data_ptr(),
                          None)
    assert torch.equal(r, total) and torch.equal(out, want)


def test_rows_two_to_the_31_elements_apart():
    g = gen(1)
    rows, cols, ld = 4, 520, 2 ** 30 + 8
    big = torch.empty(3 * ld + cols, dtype=BF, device="cuda")
    x = big.as_strided((rows, cols), (ld, 1))
    near = normal(g, rows, cols, t=BF)
    x.copy_(near)
    w = normal(g, cols)
    a, b = bg.rmsNorm(x, w, residual=x), bg.rmsNorm(near, w, residual=near)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    a, b = bg.rmsNormBackward(x, x, w, gradTotal=x), bg.rmsNormBackward(near, near, w, gradTotal=near)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    t = torch.tensor([0, 519, 3, 5], device="cuda")
    a, b = bg.logProbs(x, t, topK=4), bg.logProbs(near, t, topK=4)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    one = torch.ones(rows, device="cuda")
    assert torch.equal(bg.logProbsBackward(x, t, a[2], a[1], one),
                       bg.logProbsBackward(near, t, a[2], a[1], one))
    wt = normal(g, 96, cols, t=BF)
    assert torch.equal(bg.linearFused(x, wt), bg.linearFused(near, wt))  # streaming kernel
    assert torch.equal(bg.linearFused(wt, x, outType=F32), bg.linearFused(wt, near, outType=F32))
    go = normal(g, rows, 96, t=BF)
    for u, v in zip(bg.linearFusedBackward(go, x, wt, act="silu")[:2],
                    bg.linearFusedBackward(go, near, wt, act="silu")[:2]):
        assert torch.equal(u, v)
    many = normal(g, 20000, cols, t=BF)
    far = big.as_strided((3, cols), (ld, 1))
    assert torch.equal(bg.linearFused(many, far), bg.linearFused(many, near[:3]))  # by TMA


def test_results_past_two_to_the_32_elements():
    g = gen(2)
    m, k, n = 2100000, 64, 2056  # 4.3e9 outputs
    x = torch.randn(m, k, device="cuda", generator=g).to(BF)
    w = normal(g, n, k, t=BF, std=k ** -0.5)
    tail = slice(m - 300, m)
    X, W = x[tail].double(), w.double()
    z = X @ W.t()
    ez = acc(k) * (X.abs() @ W.abs().t()) + 2.0 ** -22 * z.abs()
    a, da = act64(z, "silu")
    ea = SLOPE * ez + ACT_F32 * (a.abs() + z.abs())
    out = bg.linearFused(x, w, act="silu")
    within(out[tail], a, ea + (U[BF] + U[F32]) * a.abs() + TINY[BF], "out")
    h = bg.gatedLinear(x, w, w)
    within(h[tail], a * z, ea * (z.abs() + ez) + a.abs() * ez + (U[BF] + U[F32]) * (a * z).abs() +
           TINY[BF], "gated")
    del h
    wn = normal(g, n)
    y, _, _ = bg.rmsNorm(out, wn)
    assert torch.equal(y[tail], bg.rmsNorm(out[tail], wn)[0])
    del y
    t = torch.zeros(m, device="cuda", dtype=torch.int32)
    p, q = bg.logProbs(out, t, topK=2), bg.logProbs(out[tail], t[tail], topK=2)
    assert all(torch.equal(u[tail], v) for u, v in zip(p, q))
    one = torch.ones(m, device="cuda")
    d = bg.logProbsBackward(out, t, p[2], p[1], one)
    assert torch.equal(d[tail], bg.logProbsBackward(out[tail], t[tail], p[2][tail], p[1][tail],
                                                    one[tail]))
    gx, _, _ = bg.linearFusedBackward(d, x, w, act="silu")
    G = d[tail].double()
    dz = G * da
    edz = U[BF] * dz.abs() + G.abs() * (BEND * ez + ACT_F32 * (1 + z.abs())) + TINY[BF]
    want = dz @ W
    within(gx[tail], want, (edz + acc(n) * (dz.abs() + edz)) @ W.abs() +
           (U[BF] + U[F32]) * want.abs() + TINY[BF], "x")


@pytest.mark.parametrize("sms", [1, 2, 3, 50])
def test_an_sm_budget(sms):
    g = gen(3)
    x, w, u = (normal(g, *s, t=BF) for s in ((1500, 200), (700, 200), (700, 200)))
    go = normal(g, 1500, 700, t=BF)
    ctx = bg.get_context()

    def run():
        return [bg.linearFused(x, w, outType=F32), bg.gatedLinear(x, w, u),
                *bg.gatedLinearBackward(go, x, w, u)[:3]]

    want = run()
    ctx.call("bgnn_ctx_set_sm_budget", sms)
    try:
        got = run()
    finally:
        ctx.call("bgnn_ctx_set_sm_budget", 0xffffffff)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_modules_in_a_sequential():
    g = gen(4)
    x = normal(g, 50, 24)
    m = bg.Sequential([bg.Linear(inFeatures=24, outFeatures=16), bg.ReLU(), bg.RMSNorm(features=16),
                       bg.GatedFeedForward(features=16, hiddenFeatures=40)])
    y = x
    for part in m._modules.values():
        y = part.forward(y)
    assert torch.equal(m.forward(x), y)


@pytest.mark.parametrize("type", ["bf16", "f16", "e4m3"])
def test_modules_captured(type):
    """Forward and gradients recorded once and replayed on other features."""
    g = gen(6)
    x, other, go = (normal(g, 300, 24) for _ in range(3))
    m = bg.Sequential([bg.RMSNorm(features=24),
                       bg.GatedFeedForward(features=24, hiddenFeatures=72, type=type)])
    ffn = m._modules["1"]

    def run():
        out = [m.forward(x)]
        if type != "e4m3":
            out += [v for _, v in sorted(ffn.backward(x, go).items())]
        return out

    calls = bg.CapturedForward(run)
    x.copy_(other)
    go.mul_(1e-6)
    got = [v.clone() for v in calls()]
    assert all(torch.equal(a, b) for a, b in zip(got, run()))
    calls.close()
