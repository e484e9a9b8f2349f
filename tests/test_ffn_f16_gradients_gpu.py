"""GatedFeedForward's gradients with f16 operands, whatever the size of the
upstream gradient."""
import pytest
import torch

import browsergnn_b200 as bg
from tests.test_blocks_gpu import gen, normal
from tests.test_blocks_modules_gpu import ffn64, rel

pytestmark = pytest.mark.gpu

U16 = 2.0 ** -11


def gradients(rows, f, h, go):
    g = gen(rows)
    m = bg.GatedFeedForward(features=f, hiddenFeatures=h, type="f16")
    x = normal(g, rows, f)
    X = x.double().requires_grad_()
    p = {k: v.tensor.double().cuda().requires_grad_() for k, v in m.namedParameters()}
    ffn64(X, p, "silu").backward(go.double())
    want = {"x": X.grad, **{k: v.grad for k, v in p.items()}}
    return m.backward(x, go), want


@pytest.mark.parametrize("size", [1 / 2450000, 1.0, 3e5, 1e-30, 1e30])
@pytest.mark.parametrize("rows,f,h", [(1, 32, 64), (500, 47, 100)])
def test_size_of_the_upstream_gradient(rows, f, h, size):
    """A mean over 2.45M nodes (4e-7 lies in f16's subnormals, 6e-8 apart), a
    scaled loss, and far beyond both: f16 holds neither the small nor the large."""
    go = normal(gen(rows + 1), rows, f, std=size)
    got, want = gradients(rows, f, h, go)
    for k, w in want.items():
        # the roundings that the module's own test counts
        assert rel(got[k], w) < 12 * U16, k


def test_sums_over_many_rows():
    """Gradients of one sign add up over 200,000 rows."""
    rows = 200000
    go = torch.ones(rows, 16, device="cuda")
    got, want = gradients(rows, 16, 32, go)
    for k, w in want.items():
        assert torch.isfinite(got[k]).all(), k
        # an element's sum may cancel: rounded terms of sum |g| |h|, so by the
        # largest element rather than by the norm
        assert (got[k].double() - w).abs().max() < 24 * U16 * w.abs().max(), k


def test_zeros_none_and_not_finite():
    m = bg.GatedFeedForward(features=8, hiddenFeatures=16, type="f16")
    x = normal(gen(2), 5, 8)
    for v in m.backward(x, torch.zeros_like(x)).values():
        assert torch.equal(v, torch.zeros_like(v))
    grads = m.backward(x[:0], x[:0])
    assert grads["x"].shape == (0, 8) and torch.equal(grads["up"], torch.zeros_like(grads["up"]))
    bad = torch.ones_like(x)
    bad[2, 3] = torch.inf
    assert not torch.isfinite(m.backward(x, bad)["down"]).all()
