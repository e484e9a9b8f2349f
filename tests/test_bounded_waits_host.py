"""The bounded waits of the tensor-core kernels, by their sources: a wait that a
whole warp makes is followed by instructions that need all lanes, so its
outcome is the warp's (warp_wait); a single thread's is its own (mbar_wait)."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def epilogue(name):
    text = open(os.path.join(ROOT, "browsergnn_b200", "csrc", name)).read()
    parts = text.split("// ---- epilogue")
    assert len(parts) == 2, "one epilogue"
    return text, re.split(r"\n}\n", parts[1])[0]


@pytest.mark.parametrize("name", ["dense16.cu", "gemm_tc.cu"])
def test_a_warp_gives_up_as_one(name):
    text, body = epilogue(name)
    assert body.count("warp_wait(") >= 1
    assert not re.search(r"\bmbar_wait\(", body)
    helper = re.search(r"bool warp_wait\(.*?\n}\n", text, re.S).group(0)
    assert re.search(r"__all_sync\(0xffffffffu, mbar_(wait|try)\(", helper)
