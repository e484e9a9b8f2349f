"""The choice head's gradient beside logits of the type's lowest value, which
masks written into the logits hold."""
import math

import pytest
import torch

import browsergnn_b200 as bg
from tests.test_blocks_gpu import BF, F16, F32, TINY, U, gen, normal, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [F32, BF, F16])
@pytest.mark.parametrize("cols", [7, 700, 3001])
@pytest.mark.parametrize("shift", [0.0, 200.0])
@pytest.mark.parametrize("weight", [1.0, 1024.0])
def test_gradient_with_entropy(t, cols, shift, weight):
    g = gen(cols)
    x = normal(g, 6, cols, t=t, std=2.0) + shift
    low = torch.rand(6, cols, device="cuda", generator=g) < 0.4
    low[:, 0] = False
    x = torch.where(low, torch.finfo(t).min, x).to(t)
    x[5] = torch.finfo(t).min  # a row of nothing else: all equally likely
    target = torch.zeros(6, device="cuda", dtype=torch.int64)
    gl, gh = normal(g, 6, std=weight), normal(g, 6, std=weight)
    logp, ent, lse, _, _ = bg.logProbs(x, target)
    got = bg.logProbsBackward(x, target, lse, ent, gl, gradEntropy=gh)
    X = x.double()
    lp = torch.log_softmax(X, 1)
    p = lp.exp()
    safe = lp.masked_fill(p == 0, 0)
    H = -(p * safe).sum(1, keepdim=True)
    G, E = gl.double()[:, None], gh.double()[:, None]
    want = p * (-G - E * (safe + H))
    want[:, 0] += gl.double()
    # f32: log p to 2^-16 at these sizes (lse up to 210, sums of 3,001 terms)
    mag = p * (G.abs() + E.abs() * (safe.abs() + H + 1)) * (1 + safe.abs())
    mag[:, 0] += gl.double().abs()
    within(got, want, U[t] * want.abs() + 2.0 ** -14 * mag + TINY[t], "logits")
    assert torch.equal(got[:5][low[:5]], torch.zeros_like(got[:5][low[:5]]))


def test_a_difference_beyond_f32():
    """x - max past the lowest f32 value: probability 0, gradient 0."""
    x = torch.tensor([[3e38, -3e38, 2.9e38], [3e38, 3e38, -3.4e38]], device="cuda")
    target = torch.tensor([0, 1], device="cuda")
    logp, ent, lse, _, _ = bg.logProbs(x, target)
    one = torch.ones(2, device="cuda")
    for gh in (None, one):
        d = bg.logProbsBackward(x, target, lse, ent, one, gradEntropy=gh)
        assert torch.equal(d[0], torch.zeros(3, device="cuda"))
        assert abs(d[1, 0].item() + 0.5) < 1e-6 and abs(d[1, 1].item() - 0.5) < 1e-6 and d[1, 2] == 0
    assert logp[0] == 0 and abs(logp[1].item() + math.log(2)) < 1e-6
