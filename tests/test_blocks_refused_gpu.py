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


def test_out_in_the_residuals_buffer_with_another_type_or_stride():
    """Rows written over others that are still to be read."""
    import torch

    ctx = bg.get_context()
    m, k, n = 40, 24, 16
    x = torch.ones(m, k, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(n, k, dtype=torch.bfloat16, device="cuda")
    r = torch.ones(m, 2 * n, device="cuda")

    def call(rows, res_type, ld_res, out_type, ld_out):
        ctx.call("bgnn_linear_fused", BF16, x.data_ptr(), k, None, w.data_ptr(), k, None, rows, k, n,
                 0, None, 0, 0.0, res_type, r.data_ptr(), ld_res, out_type, r.data_ptr(), ld_out)

    for bad in ((F32, n, BF16, n), (BF16, n, F32, n), (F32, 2 * n, F32, n), (F32, n, F32, 2 * n)):
        with pytest.raises(bg.BGNNError, match="residual's buffer"):
            call(m, *bad)
    assert (r == 1).all()
    call(1, F32, n, F32, 2 * n)  # one row has no stride
    assert (r[0, :n] == 1 + k).all() and (r[1:] == 1).all()
    call(m, F32, 2 * n, F32, 2 * n)
    assert (r[1:, :n] == 1 + k).all() and (r[:, n:] == 1).all()
    r.fill_(1.0)
    wn = torch.ones(n, device="cuda")
    out = torch.empty(m, n, device="cuda")
    f = torch.ones(m, n, device="cuda")
    with pytest.raises(bg.BGNNError, match="residual's buffer"):
        ctx.call("bgnn_rms_norm", F32, f.data_ptr(), n, F32, r.data_ptr(), 2 * n, F32, wn.data_ptr(),
                 m, n, 1e-6, r.data_ptr(), F32, out.data_ptr(), None)
    assert (r == 1).all()
    ctx.call("bgnn_rms_norm", F32, f.data_ptr(), n, F32, r.data_ptr(), n, F32, wn.data_ptr(), m, n,
             1e-6, r.data_ptr(), F32, out.data_ptr(), None)
    assert (r.reshape(-1)[:m * n] == 2).all() and (r.reshape(-1)[m * n:] == 1).all()
