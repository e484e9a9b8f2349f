"""LearningPathRecommender.stepLogProb with lists of any length."""
import math

import numpy as np
import pytest

import browsergnn_b200 as bg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nodes", [20, 100])
@pytest.mark.parametrize("topK", [0, 5, 32, 33, 64, 1000])
def test_as_many_alternatives_as_recommend(nodes, topK):
    g = bg.LearningPathRecommender.createSampleCurriculum(nodes, np.random.default_rng(4))
    m = bg.LearningPathRecommender(inputFeatures=11, hiddenDim=16, normalizeScores=False)
    mastered = [0, 2, 7, 11]
    rec = m.recommend(g, mastered, topK)["recommendations"]
    step = m.stepLogProb(g, 5, mastered, topK=topK)
    alt = step["alternatives"]
    assert [a["nodeIndex"] for a in alt] == [r["nodeIndex"] for r in rec]
    assert [a["rank"] for a in alt] == list(range(1, len(alt) + 1))
    short = m.stepLogProb(g, 5, mastered, topK=min(topK, 32))["alternatives"]
    assert alt[:32] == short
    for a in alt:
        if a["nodeIndex"] == 5:
            assert a["logProb"] == step["logProb"]
    if topK >= nodes:  # all that are left: the probabilities of nodes - 4 add up to 1
        assert abs(sum(math.exp(a["logProb"]) for a in alt) - 1) < nodes * 2.0 ** -20
        assert abs(step["entropy"] + sum(math.exp(a["logProb"]) * a["logProb"] for a in alt)) < 1e-4


def test_nothing_left():
    g = bg.LearningPathRecommender.createSampleCurriculum(50, np.random.default_rng(4))
    m = bg.LearningPathRecommender(inputFeatures=11, hiddenDim=16)
    step = m.stepLogProb(g, 5, range(50), topK=40)
    assert step == {"logProb": -math.inf, "entropy": 0.0, "alternatives": []}
    with pytest.raises(ValueError):
        m.stepLogProb(g, 5, topK=-1)
