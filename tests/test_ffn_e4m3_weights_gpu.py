"""GatedFeedForward's 8-bit weights where a row's largest value is tiny or 0."""
import pytest
import torch

import browsergnn_b200 as bg
from tests.test_blocks_gpu import gen, normal
from tests.test_blocks_modules_gpu import ffn64, rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tiny", [0.0, 1e-45, 1e-43, 1e-40, 1e-37])
def test_rows_of_tiny_weights(tiny):
    g = gen(3)
    m = bg.GatedFeedForward(features=32, hiddenFeatures=48, type="e4m3")
    state = {k: v.tensor.clone() for k, v in m.namedParameters()}
    state["gate"][5] = torch.sign(state["gate"][5]) * tiny
    state["up"][7] = torch.sign(state["up"][7]) * tiny
    m.loadStateDict(state)
    x = normal(g, 60, 32)
    out = m.forward(x)
    p = {k: v.double().cuda() for k, v in state.items()}
    # the roundings that the module's own test counts
    assert rel(out, ffn64(x.double(), p, "silu")) < 6 * 2.0 ** -4
    q, scale = m._eight("gate")
    # e4m3: half a step of the value, and half of its smallest step of the scale
    tol = state["gate"].cuda().double().abs() * 2.0 ** -4 + scale.double()[:, None] * 2.0 ** -10
    assert ((q.double() * scale.double()[:, None] - state["gate"].cuda().double()).abs() <= tol).all()
