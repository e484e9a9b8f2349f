"""The choice head's gradient for long rows whose log-sum-exp is large: such a
row is summed again, by blocks that share the work."""
import pytest
import torch

import browsergnn_b200 as bg
from tests.test_blocks_gpu import BF, F16, F32, TINY, U, gen, left64, normal, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [F32, BF, F16])
@pytest.mark.parametrize("rows,cols", [(1, 200003), (3, 50001), (40, 9000), (1200, 2500)])
@pytest.mark.parametrize("masked", [False, True])
def test_near_and_far_rows_together(rows, cols, t, masked):
    g = gen(cols)
    x = normal(g, rows, cols)
    at = torch.tensor([500.0, 0.0, -3e4, 127.0], device="cuda")
    x = (x + at[torch.arange(rows, device="cuda") % 4, None]).to(t)
    m = None
    if masked:
        m = torch.rand(rows, cols, device="cuda", generator=g) < 0.4
        m[:, 0] = False
        if rows > 2:
            m[2] = True  # nothing left
    target = torch.zeros(rows, device="cuda", dtype=torch.int64)
    logp, ent, lse, _, _ = bg.logProbs(x, target, mask=m)
    gl, gh = torch.ones(rows, device="cuda"), normal(g, rows)
    got = bg.logProbsBackward(x, target, lse, ent, gl, gradEntropy=gh, mask=m)
    v = left64(x, m)
    whole = torch.logsumexp(v, 1, keepdim=True)
    some = whole > -torch.inf
    lp = v - whole.masked_fill(~some, 0)
    p = lp.exp()
    safe = lp.masked_fill(p == 0, 0)
    H = -(p * safe).sum(1, keepdim=True)
    E = gh.double()[:, None]
    want = p * (-1 - E * (safe + H))
    want[:, 0] += some[:, 0].double()
    # near rows: half the last bit of lse (below 128, 2^-18) is an error of p; far
    # ones: x - lse and its exponentials' sum in f32.  2^-15 of the terms covers either, and the entropy's.
    mag = p * (1 + E.abs() * (safe.abs() + H + 1))
    tol = U[t] * want.abs() + 2.0 ** -15 * mag + 2.0 ** -23 + TINY[t]
    within(got, want, tol, "logits")
    again = bg.logProbsBackward(x, target, lse, ent, gl, gradEntropy=gh, mask=m)
    assert torch.equal(got, again)


def test_a_far_row_costs_what_a_near_one_does():
    """Summed by each of a row's blocks alone it took fifty times as long."""
    x = normal(gen(1), 1, 1000000)
    target = torch.zeros(1, device="cuda", dtype=torch.int32)
    one = torch.ones(1, device="cuda")

    def time(v):
        _, ent, lse, _, _ = bg.logProbs(v, target)
        calls = bg.CapturedForward(  # replayed: the host's part is the same
            lambda: [bg.logProbsBackward(v, target, lse, ent, one) for _ in range(20)])
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

    near, far = time(x), time(x + 500)
    assert far < 8 * near, (near, far)
