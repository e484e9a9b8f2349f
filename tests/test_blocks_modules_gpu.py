"""RMSNorm, GatedFeedForward and LearningPathRecommender.stepLogProb: the block
operators as a model uses them, on a GraphData, against 64-bit forms."""
import math

import numpy as np
import pytest
import torch

import browsergnn_b200 as bg
from tests.helpers import rand_graph

pytestmark = pytest.mark.gpu


def graph(n, f, seed=0):
    ei, e = rand_graph(n, 4 * n, seed)
    x = np.random.default_rng(seed).standard_normal((n, f)).astype(np.float32)
    return bg.GraphData(x=x, numNodes=n, numFeatures=f, edgeIndex=ei, numEdges=e)


def rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


def ffn64(x, p, act):
    n = x * (x.pow(2).mean(1, keepdim=True) + 1e-6).rsqrt() * p["norm"]
    z, u = n @ p["gate"].t(), n @ p["up"].t()
    a = z * torch.sigmoid(z) if act == "silu" else torch.relu(z)
    return x + (a * u) @ p["down"].t()


@pytest.mark.parametrize("type,act", [("bf16", "silu"), ("f16", "relu"), ("e4m3", "silu")])
@pytest.mark.parametrize("n,f,h", [(1, 32, 64), (300, 47, 100), (2000, 64, 256)])
def test_gated_feed_forward(n, f, h, type, act):
    g = graph(n, f)
    m = bg.GatedFeedForward(features=f, hiddenFeatures=h, act=act, type=type)
    out = m.forward(g)
    assert isinstance(out, bg.GraphData) and out.x.dtype == torch.float32
    x = g.x_device().double().requires_grad_()
    p = {k: v.tensor.double().cuda().requires_grad_() for k, v in m.namedParameters()}
    want = ffn64(x, p, act)
    # n, the weights, h: each rounded by at most u; the branch is about as large
    # as the stream.  Norm-wise a sum of roundings is below their sum.
    u = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "e4m3": 2.0 ** -4}[type]
    assert rel(out.x, want.detach()) < 6 * u
    go = torch.randn(n, f, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    if type == "e4m3":
        with pytest.raises(NotImplementedError):
            m.backward(g, go)
        return
    want.backward(go.double())
    grads = m.backward(g, go)
    assert set(grads) == {"x", "norm", "gate", "up", "down"}
    for k, w in [("x", x.grad)] + [(k, v.grad) for k, v in p.items()]:
        assert grads[k].dtype == torch.float32 and grads[k].shape == w.shape
        # the forward's roundings, the gradient's, dg and du, the weights, the
        # result.  ReLU's derivative jumps: z has an error e of at most 2u rms(z)
        # (n and the weights rounded), so a sign flips with a probability of at
        # most 2 pdf(0) E|e| = 2 * 0.4 * 2u, and a flipped element of the half
        # that counts is wrong by all of itself: sqrt(2 * 1.6u) norm-wise.
        jump = math.sqrt(3.2 * u) if act == "relu" else 0.0
        assert rel(grads[k], w) < 12 * u + jump, k


def test_norm_module_and_layers_between():
    g = graph(200, 24)
    norm = bg.RMSNorm(features=24)
    y = norm.forward(g)
    x = g.x_device().double()
    s = (x.pow(2).mean(1, keepdim=True) + 1e-6).rsqrt()
    assert rel(y.x, x * s) < 1e-6
    go = torch.ones(200, 24, device="cuda")
    gr = norm.backward(g, go)
    xh = x * s
    assert rel(gr["x"], s * (1 - xh * xh.mean(1, keepdim=True))) < 1e-5
    assert rel(gr["weight"], xh.sum(0)) < 1e-5
    conv = bg.SAGEConv(inChannels=24, outChannels=24)
    ffn = bg.GatedFeedForward(features=24, hiddenFeatures=48)
    h = conv.forward(ffn.forward(conv.forward(norm.forward(g))))
    assert h.x.shape == (200, 24) and torch.isfinite(h.x).all()
    state = bg.GatedFeedForward(features=24, hiddenFeatures=48)
    state.loadStateDict(ffn.stateDict())
    assert torch.equal(state.forward(g).x, ffn.forward(g).x)


@pytest.mark.parametrize("normalize", [True, False])
def test_step_log_prob(normalize):
    rng = np.random.default_rng(3)
    g = bg.LearningPathRecommender.createSampleCurriculum(40, rng)
    m = bg.LearningPathRecommender(inputFeatures=11, hiddenDim=16, normalizeScores=normalize)
    mastered = [0, 3, 7]
    rec = m.recommend(g, mastered, 5)
    step = m.stepLogProb(g, rec["recommendations"][2]["nodeIndex"], mastered, topK=5)
    assert [a["nodeIndex"] for a in step["alternatives"]] == \
        [r["nodeIndex"] for r in rec["recommendations"]]
    assert step["logProb"] == step["alternatives"][2]["logProb"]
    s = m._scores(g).reshape(-1).double().cpu()
    left = torch.ones(40, dtype=torch.bool)
    left[mastered] = False
    lp = torch.log_softmax(s[left], 0)
    assert abs(step["entropy"] - float(-(lp.exp() * lp).sum())) < 1e-5
    i = int(left.nonzero()[:, 0].tolist().index(rec["recommendations"][2]["nodeIndex"]))
    assert abs(step["logProb"] - float(lp[i])) < 1e-5
    assert m.stepLogProb(g, 3, mastered)["logProb"] == -math.inf
    alone = m.stepLogProb(g, 5, [i for i in range(40) if i != 5], topK=3)
    assert abs(alone["logProb"]) < 1e-6 and len(alone["alternatives"]) == 1
    with pytest.raises(ValueError):
        m.stepLogProb(g, 40)
