"""Two host threads, each on a stream of its own, through the facade at once."""
import threading

import pytest
import torch

import browsergnn_b200 as bg
from tests.test_blocks_gpu import BF, gen, normal

pytestmark = pytest.mark.gpu


def test_products_backward_from_two_threads():
    cases = []
    for seed, m in ((1, 3000), (2, 2500)):
        g = gen(seed)
        cases.append((normal(g, m, 96, t=BF), normal(g, m, 64, t=BF), normal(g, 96, 64, t=BF),
                      normal(g, 96, t=BF)))
    want = [bg.linearFusedBackward(go, x, w, bias=b, act="gelu") for go, x, w, b in cases]
    torch.cuda.synchronize()
    errors = []

    def run(i):
        try:
            go, x, w, b = cases[i]
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(60):
                    got = bg.linearFusedBackward(go, x, w, bias=b, act="gelu")
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(u, v) for u, v in zip(got, want[i])):
                    errors.append(f"thread {i}: other results")
        except Exception as e:  # noqa: BLE001 - reported by the test
            errors.append(repr(e))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
