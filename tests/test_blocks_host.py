"""Refusals of the block operators and the choice head that need no GPU: types
and shapes are checked before anything touches a device."""
import ctypes

import pytest
import torch

import browsergnn_b200 as bg

BF, F8 = torch.bfloat16, torch.float8_e4m3fn


def z(*shape, t=BF):
    return torch.zeros(*shape, dtype=t)


REFUSED = [
    (TypeError, "x must be a CUDA", lambda: bg.rmsNorm([1.0], z(1))),
    (TypeError, "x has type", lambda: bg.rmsNorm(z(2, 4, t=torch.float64), z(4))),
    (TypeError, "outType has type", lambda: bg.rmsNorm(z(2, 4), z(4), outType=torch.int8)),
    (ValueError, "weight: expected shape", lambda: bg.rmsNorm(z(2, 4), z(5))),
    (ValueError, "weight: expected shape", lambda: bg.rmsNorm(z(2, 4), z(1, 4))),
    (TypeError, "residual has type",
     lambda: bg.rmsNorm(z(2, 4), z(4), residual=z(2, 4, t=torch.float16))),
    (ValueError, "residual: expected shape", lambda: bg.rmsNorm(z(2, 4), z(4), residual=z(3, 4))),
    (ValueError, "1D or 2D", lambda: bg.rmsNorm(z(2, 2, 4), z(4))),
    (TypeError, "gradOut has type",
     lambda: bg.rmsNormBackward(z(2, 4, t=torch.float32), z(2, 4), z(4))),
    (TypeError, "gradTotal has type",
     lambda: bg.rmsNormBackward(z(2, 4), z(2, 4), z(4), gradTotal=z(2, 4, t=torch.float32))),
    (TypeError, "x has type", lambda: bg.linearFused(z(2, 4, t=torch.float32), z(3, 4))),
    (TypeError, "weight has type",
     lambda: bg.linearFused(z(2, 4), z(3, 4, t=torch.float16))),
    (ValueError, "Expected input size 5, got 4", lambda: bg.linearFused(z(2, 4), z(3, 5))),
    (ValueError, "2D weight", lambda: bg.linearFused(z(2, 4), z(4))),
    (ValueError, "unknown activation", lambda: bg.linearFused(z(2, 4), z(3, 4), act="swish")),
    (ValueError, "need a scale", lambda: bg.linearFused(z(2, 4, t=F8), z(3, 4, t=F8))),
    (ValueError, "only e4m3", lambda: bg.linearFused(z(2, 4), z(3, 4), xScale=z(2))),
    (ValueError, "xScale: expected shape",
     lambda: bg.linearFused(z(2, 4, t=F8), z(3, 4, t=F8), xScale=z(3, t=torch.float32),
                            weightScale=z(3, t=torch.float32))),
    (TypeError, "e4m3 operands have no backward",
     lambda: bg.linearFusedBackward(z(2, 3), z(2, 4, t=F8), z(3, 4, t=F8))),
    (ValueError, "gradOut: expected shape",
     lambda: bg.linearFusedBackward(z(2, 4), z(2, 4), z(3, 4))),
    (TypeError, "gradOut has type",
     lambda: bg.linearFusedBackward(z(2, 3, t=torch.float32), z(2, 4), z(3, 4))),
    (ValueError, "weightUp: expected 3 rows", lambda: bg.gatedLinear(z(2, 4), z(3, 4), z(2, 4))),
    (TypeError, "biasUp has type",
     lambda: bg.gatedLinear(z(2, 4), z(3, 4), z(3, 4), biasGate=z(3),
                            biasUp=z(3, t=torch.float32))),
    (ValueError, "topK", lambda: bg.logProbs(z(2, 4), z(2, t=torch.int32), topK=33)),
    (TypeError, "targets has type", lambda: bg.logProbs(z(2, 4), z(2, t=torch.float32))),
    (ValueError, "targets: expected 2", lambda: bg.logProbs(z(2, 4), z(3, t=torch.int32))),
    (TypeError, "mask has type",
     lambda: bg.logProbs(z(2, 4), z(2, t=torch.int32), mask=z(4, t=torch.int32))),
    (ValueError, "mask: expected shape",
     lambda: bg.logProbs(z(2, 4), z(2, t=torch.int32), mask=z(3, t=torch.uint8))),
    (ValueError, "lse: expected 2",
     lambda: bg.logProbsBackward(z(2, 4), z(2, t=torch.int32), z(3, t=torch.float32),
                                 z(2, t=torch.float32), None)),
    (ValueError, "needs the forward's",
     lambda: bg.logProbsBackward(z(2, 4), z(2, t=torch.int32), None, None, None)),
    (TypeError, "must be a CUDA", lambda: bg.linearFused(z(2, 4), z(3, 4))),
    (TypeError, "must be a CUDA", lambda: bg.logProbs(z(2, 4), z(2, t=torch.int64))),
]


@pytest.mark.parametrize("case", range(len(REFUSED)))
def test_refusals(case):
    kind, text, call = REFUSED[case]
    with pytest.raises(kind, match=text):
        call()


def test_null_context():
    from browsergnn_b200 import _lib

    lib = _lib.load()
    for name in ("bgnn_rms_norm", "bgnn_rms_norm_backward", "bgnn_linear_fused",
                 "bgnn_linear_fused_backward", "bgnn_gated_linear", "bgnn_gated_linear_backward",
                 "bgnn_log_probs", "bgnn_log_probs_backward"):
        args = [None if a is ctypes.c_void_p else a(0) for a in _lib.SIGNATURES[name]]
        assert getattr(lib, name)(*args) == _lib.ERR_INVALID_ARG, name
