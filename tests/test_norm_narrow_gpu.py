"""The RMS norm and its gradient on rows narrower than a vector, a few and many
of them, contiguous and at every offset, against 64-bit forms."""
import pytest
import torch

import browsergnn_b200 as bg
from tests.test_blocks_gpu import BF, F8, F16, F32, TINY, U, gen, normal, wide, within

pytestmark = pytest.mark.gpu


def at_end(x, off):
    """x as a view whose last element is its storage's, `off` elements behind a
    vector's start."""
    flat = torch.empty(x.numel() + off, dtype=x.dtype, device=x.device)
    flat[off:] = x.reshape(-1)
    return flat[off:].view(x.shape)


@pytest.mark.parametrize("rows", [2, 3, 9, 1000])
@pytest.mark.parametrize("cols", list(range(1, 13)))
@pytest.mark.parametrize("tx,tr,to", [(F32, F32, BF), (F32, None, F32), (BF, BF, F8),
                                      (F16, F32, F16), (BF, None, BF)])
def test_rms_norm(rows, cols, tx, tr, to):
    g = gen(rows * 13 + cols)
    w = normal(g, cols) + 1
    base_x = normal(g, rows, cols, t=tx)
    base_r = None if tr is None else normal(g, rows, cols, t=tr, std=3.0)
    slop = (cols + 16) * 2.0 ** -24  # as in the norm's own tests
    for how in ("plain", "odd", 1, 6):
        place = (lambda v: at_end(v, how)) if isinstance(how, int) else (lambda v: wide(v, how))
        x, r = place(base_x), None if base_r is None else place(base_r)
        out, total, scale = bg.rmsNorm(x, w, residual=r, eps=1e-5, outType=to)
        if r is not None:
            want = base_x.double() + base_r.double()
            within(total, want, (U[tr] + U[F32]) * want.abs() + TINY[tr], "total")
        t = total.double()
        y = t * (t.pow(2).mean(1, keepdim=True) + 1e-5).rsqrt() * w.double()
        if to == F8:
            got = out.double() * scale.double()[:, None]
            tol = y.abs() * (2.0 ** -4 + slop) + scale.double()[:, None] * 2.0 ** -10
            within(got, y, tol, how)
        else:
            within(out, y, y.abs() * (U[to] + slop + 4 * U[F32]) + TINY[to], how)


@pytest.mark.parametrize("rows", [2, 3, 9, 1000])
@pytest.mark.parametrize("cols", list(range(1, 13)))
@pytest.mark.parametrize("tt,tg,stream", [(F32, F32, True), (F32, BF, False), (F16, F16, True)])
def test_rms_norm_backward(rows, cols, tt, tg, stream):
    g = gen(rows * 17 + cols)
    w = normal(g, cols) + 1
    T0, G0 = normal(g, rows, cols, t=tt, std=2.0), normal(g, rows, cols, t=tg)
    S0 = normal(g, rows, cols, t=tt) if stream else None
    T, G, W = T0.double(), G0.double(), w.double()
    s = (T.pow(2).mean(1, keepdim=True) + 1e-5).rsqrt()
    xh = T * s
    c = (G * W * xh).mean(1, keepdim=True)
    want = s * (G * W - xh * c)
    mag = s * ((G * W).abs() + xh.abs() * (G * W * xh).abs().mean(1, keepdim=True))
    if stream:
        want, mag = want + S0.double(), mag + S0.double().abs()
    tol = U[tt] * want.abs() + (2 * cols + 32) * 2.0 ** -24 * mag + TINY[tt]
    for how in ("plain", "odd", 1, 6):
        place = (lambda v: at_end(v, how)) if isinstance(how, int) else (lambda v: wide(v, how))
        gx, gw = bg.rmsNormBackward(place(G0), place(T0), w, eps=1e-5,
                                    gradTotal=place(S0) if stream else None)
        within(gx, want, tol, how)
        within(gw, (G * xh).sum(0), (rows + cols + 32) * 2.0 ** -24 * (G * xh).abs().sum(0), how)


def test_modules_of_one_to_four_features():
    for f in (1, 2, 3, 4):
        g = gen(f)
        x = normal(g, 600, f)
        n = bg.RMSNorm(features=f)
        t = x.double()
        y = t * (t.pow(2).mean(1, keepdim=True) + 1e-6).rsqrt()
        within(n.forward(x), y, y.abs() * (f + 21) * 2.0 ** -24, f)
        m = bg.GatedFeedForward(features=f, hiddenFeatures=8)
        out, grads = m.forward(x), m.backward(x, x)
        assert out.shape == x.shape and torch.isfinite(out).all()
        assert all(torch.isfinite(v).all() for v in grads.values())


@pytest.mark.parametrize("t", [BF, F16])
@pytest.mark.parametrize("cols", [1004, 1005, 1012, 1016, 1019, 1020, 1021, 1024])
def test_backward_at_the_shared_memory_of_a_launch(cols, t):
    """A block's column sums, its staged rows and its static shared memory come
    to 48 KB, the most that a launch has without asking, at about 1,020 columns."""
    g = gen(cols)
    w = normal(g, cols)
    T0, G0 = normal(g, 40, cols, t=t), normal(g, 40, cols, t=t)
    T, G, W = T0.double(), G0.double(), w.double()
    s = (T.pow(2).mean(1, keepdim=True) + 1e-6).rsqrt()
    xh = T * s
    for how in ("plain", "odd"):
        gx, gw = bg.rmsNormBackward(wide(G0, how), wide(T0, how), w)
        c = (G * W * xh).mean(1, keepdim=True)
        mag = s * ((G * W).abs() + xh.abs() * (G * W * xh).abs().mean(1, keepdim=True))
        want = s * (G * W - xh * c)
        within(gx, want, U[t] * want.abs() + (2 * cols + 32) * 2.0 ** -24 * mag + TINY[t], how)
        within(gw, (G * xh).sum(0), (40 + cols + 32) * 2.0 ** -24 * (G * xh).abs().sum(0), how)
