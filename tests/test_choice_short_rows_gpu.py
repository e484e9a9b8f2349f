"""Long lists of alternatives for short rows."""
import numpy as np
import pytest
import torch

import browsergnn_b200 as bg
from tests.test_blocks_gpu import BF, F16, F32, gen, head64, normal, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [F32, BF, F16])
@pytest.mark.parametrize("cols", [5, 33, 64, 65, 200, 256, 257, 512, 513, 1000, 1024])
@pytest.mark.parametrize("top", [15, 16, 17, 20, 28, 32])
def test_lists(cols, t, top):
    g = gen(cols + top)
    x = normal(g, 8, cols, t=t, std=2.0)
    x[1] = 1.0                        # all equal
    x[2] = torch.arange(cols, device="cuda") / cols          # ascending
    x[3] = -torch.arange(cols, device="cuda") / cols - 1000  # descending, all negative
    x[4, 32:] = -torch.inf            # a lane each, and one element
    x[5] = torch.arange(cols, device="cuda") % 3
    x[6, 3] = torch.nan               # not an alternative
    mask = torch.rand(8, cols, device="cuda", generator=g) < 0.3
    mask[7] = torch.arange(cols, device="cuda") % 32 > 2     # what is left: three lanes'
    target = torch.full((8,), -1, device="cuda", dtype=torch.int32)
    for m in (None, mask):
        _, _, _, ids, tl = bg.logProbs(x, target, mask=m, topK=top)
        _, _, _, _, _, ids_w, tl_w = head64(x.nan_to_num(nan=-torch.inf, neginf=-torch.inf), m, target,
                                            top)
        assert np.array_equal(ids.cpu().numpy(), ids_w)
        rows = [0, 1, 2, 3, 4, 5, 7]
        # f32: log p of size 1,010 at most, sums of 1,024 terms
        within(tl[rows], tl_w[rows], 2.0 ** -17 * (1 + tl_w[rows].abs().nan_to_num(posinf=0)), "top")


def test_a_long_list_costs_what_a_short_one_does():
    """With a border that lets half a row through, a list of 32 took four times
    as long as one of 16."""
    x = normal(gen(1), 8192, 1000)
    target = torch.zeros(8192, device="cuda", dtype=torch.int32)

    def time(top):
        calls = bg.CapturedForward(lambda: [bg.logProbs(x, target, topK=top) for _ in range(10)])
        best = 1e9
        for _ in range(10):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            calls()
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        calls.close()
        return best

    short, long = time(16), time(32)
    assert long < 2.5 * short, (short, long)
