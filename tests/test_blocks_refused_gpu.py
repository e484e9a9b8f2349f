"""Calls of the block operators' C entry points that are refused before
anything is launched.  Every call here is also harmless where it is not refused:
its pointers are NULL, which is refused too, or its operands are real."""
import pytest

import browsergnn_b200 as bg

pytestmark = pytest.mark.gpu

F32, BF16 = 0, 1


@pytest.mark.parametrize("cols", [2 ** 31, 2 ** 32 - 1])
def test_rows_of_two_to_the_31_elements(cols):
    """A 32-bit column counter would wrap."""
    ctx = bg.get_context()
    none = [None] * 3
    with pytest.raises(bg.BGNNError, match=r"2\^31"):
        ctx.call("bgnn_rms_norm", F32, None, cols, F32, None, 0, F32, None, 1, cols, 1e-6, None, F32,
                 None, None)
    with pytest.raises(bg.BGNNError, match=r"2\^31"):
        ctx.call("bgnn_rms_norm_backward", F32, None, cols, F32, None, cols, None, 0, F32, None, 1,
                 cols, 1e-6, None, None)
    with pytest.raises(bg.BGNNError, match=r"2\^31"):
        ctx.call("bgnn_log_probs", F32, None, cols, 1, cols, None, 0, None, 0, *none, None, None)
    with pytest.raises(bg.BGNNError, match=r"2\^31"):
        ctx.call("bgnn_log_probs_backward", F32, None, cols, 1, cols, None, 0, None, None, None, None,
                 None, None)
