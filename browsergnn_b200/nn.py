"""Neural-network modules of src/nn/ on the cuda backend.

Linear (src/nn/linear.ts), the activation modules of src/nn/activation.ts
(ReLU, LeakyReLU, ELU, Sigmoid, Tanh, Softmax, LogSoftmax, GELU, SiLU, PReLU,
Dropout) and the Module / Sequential containers of src/nn/module.ts.  Same
constructor arguments, parameter names and shapes, defaults and errors as the
reference; ``forward`` takes a CUDA tensor (or a GraphData, whose features it
transforms) and returns the same kind.  RMSNorm and GatedFeedForward are this
backend's own, over the mixed-precision operators of blocks.py.

Training-mode Dropout draws from a counter-based generator (libbgnn_cuda's
bgnn_dropout) instead of Math.random(): the keep/scale rule is the
reference's, the random stream is not (the reference's is unseeded).  In eval
mode Dropout is the identity, exactly as in the reference.
"""
from __future__ import annotations

from typing import Optional

import numpy as np

from . import _lib
from .backend import get_context, ptr
from .blocks import (gatedLinear, gatedLinearBackward, linearFused, linearFusedBackward, rmsNorm,
                     rmsNormBackward)
from .graph import GraphData
from .layers import (ELU, LeakyReLU, Module, ReLU, Sequential, _Act, _param, _torch,
                     manual_seed, next_dropout_seed, register_fusable)

__all__ = [
    "Module", "Sequential", "Linear", "ReLU", "LeakyReLU", "ELU", "Sigmoid", "Tanh", "GELU",
    "SiLU", "PReLU", "Softmax", "LogSoftmax", "Dropout", "RMSNorm", "GatedFeedForward",
    "manual_seed",
]


def _tensor_of(input):
    return input.x_device() if isinstance(input, GraphData) else input


def _wrap(input, out):
    return input.withFeatures(out) if isinstance(input, GraphData) else out


class Linear(Module):
    """src/nn/linear.ts:19-115: y = x W^T + b with ``weight`` [out, in] and
    ``bias`` [out] (zeros); the weight is a normal draw scaled by
    sqrt(2 / (in + out)).  Each output is one double sum over the inputs,
    stored to f32, then the bias is added in f32."""

    def __init__(self, config: Optional[dict] = None, **kw):
        super().__init__()
        cfg = dict(config or {})
        cfg.update(kw)
        self.inFeatures = int(cfg["inFeatures"])
        self.outFeatures = int(cfg["outFeatures"])
        self.useBias = bool(cfg.get("bias", True))
        stdv = np.sqrt(2.0 / (self.inFeatures + self.outFeatures))
        self.registerParameter("weight", _param((self.outFeatures, self.inFeatures), stdv))
        if self.useBias:
            self.registerParameter("bias", _param((self.outFeatures,), zeros=True))

    def forward(self, input, _act=None):
        torch = _torch()
        x = _tensor_of(input)
        if not hasattr(x, "is_cuda"):
            x = torch.as_tensor(np.asarray(x, np.float32))
        if x.dim() == 1:
            if x.shape[0] != self.inFeatures:
                raise ValueError(f"Expected input size {self.inFeatures}, got {x.shape[0]}")
            rows = 1
        elif x.dim() == 2:
            if x.shape[1] != self.inFeatures:
                raise ValueError(f"Expected input size {self.inFeatures}, got {x.shape[1]}")
            rows = int(x.shape[0])
        else:
            raise ValueError(f"Linear layer expects 1D or 2D input, got {x.dim()}D")
        if not x.is_cuda:
            x = x.to("cuda")
        x = x.to(torch.float32).contiguous()
        dev = x.device.index
        self.to_device(dev)
        out = torch.empty((rows, self.outFeatures), dtype=torch.float32, device=x.device)
        code, param = (0, 0.0) if _act is None else (_lib.ACT[_act[0]], float(_act[1]))
        get_context(dev).call("bgnn_dense", ptr(x), ptr(self.p("weight")), rows, self.inFeatures,
                              self.outFeatures, ptr(self.p("bias")), code, param, ptr(out))
        if x.dim() == 1:
            out = out.reshape(self.outFeatures)
        return _wrap(input, out)

    def __repr__(self):
        return f"Linear({self.inFeatures} -> {self.outFeatures}, bias={self.useBias})"


class Sigmoid(_Act):
    """Tensor.sigmoid (src/core/tensor.ts:413-419): 1 / (1 + exp(-x)) in double."""
    act = "sigmoid"


class Tanh(_Act):
    """Tensor.tanh (src/core/tensor.ts:424-430)."""
    act = "tanh"


class GELU(_Act):
    """src/nn/activation.ts:129-147 (tanh approximation, evaluated in double)."""
    act = "gelu"


class SiLU(_Act):
    """src/nn/activation.ts:153-168: x / (1 + exp(-x))."""
    act = "silu"


class PReLU(Module):
    """src/nn/activation.ts:175-200: learnable ``weight`` [numParameters]
    filled with ``init``; slope weight[0] or weight[i % numParameters]."""

    def __init__(self, numParameters: int = 1, init: float = 0.25):
        super().__init__()
        torch = _torch()
        self.registerParameter("weight", torch.full((int(numParameters),), float(init),
                                                    dtype=torch.float32))

    def forward(self, input):
        torch = _torch()
        x = _tensor_of(input).contiguous()
        self.to_device(x.device.index)
        w = self.p("weight")
        out = torch.empty_like(x)
        get_context(x.device.index).call("bgnn_prelu", ptr(x), x.numel(), ptr(w), w.numel(),
                                         ptr(out))
        return _wrap(input, out)


class _RowSoftmax(Module):
    log = 0

    def forward(self, input):
        torch = _torch()
        x = _tensor_of(input)
        if x.dim() != 2:
            name = "Log softmax" if self.log else "Softmax"
            raise ValueError(f"{name} currently only supports 2D tensors")
        x = x.contiguous()
        out = torch.empty_like(x)
        rows, cols = x.shape
        get_context(x.device.index).call("bgnn_softmax_rows", ptr(x), rows, cols, None, 0.0,
                                         self.log, ptr(out))
        return _wrap(input, out)


class Softmax(_RowSoftmax):
    """Tensor.softmax along the last axis (src/core/tensor.ts:435-464)."""
    log = 0


class LogSoftmax(_RowSoftmax):
    """Tensor.logSoftmax along the last axis (src/core/tensor.ts:469-499)."""
    log = 1


class Dropout(Module):
    """src/nn/activation.ts:207-245.  Identity in eval mode or for p = 0;
    in training mode element i survives when u_i > p and is scaled by
    1 / (1 - p), u_i from the counter-based generator (one fresh seed per
    call)."""

    def __init__(self, p: float = 0.5):
        super().__init__()
        if p < 0 or p > 1:
            raise ValueError("Dropout probability must be between 0 and 1")
        self.p = float(p)

    def forward(self, input, seed: Optional[int] = None):
        if not self._training or self.p == 0:
            return input
        torch = _torch()
        x = _tensor_of(input).contiguous()
        out = torch.empty_like(x)
        s = next_dropout_seed() if seed is None else int(seed)
        get_context(x.device.index).call("bgnn_dropout", ptr(x), x.numel(), self.p, s, ptr(out))
        return _wrap(input, out)


def _tensor_on_device(module, input):
    """The f32 CUDA rows of a tensor or a GraphData, the module moved to them."""
    torch = _torch()
    x = _tensor_of(input)
    if not hasattr(x, "is_cuda"):
        x = torch.as_tensor(np.asarray(x, np.float32))
    if not x.is_cuda:
        x = x.to("cuda")
    x = x.to(torch.float32)
    module.to_device(x.device.index)
    return x


class RMSNorm(Module):
    """Root-mean-square norm of each row with a learned ``weight`` [features]
    (ones).  No counterpart in the reference; f32 features in and out
    (blocks.rmsNorm has the 16- and 8-bit forms)."""

    def __init__(self, config: Optional[dict] = None, **kw):
        super().__init__()
        cfg = dict(config or {})
        cfg.update(kw)
        self.features = int(cfg["features"])
        self.eps = float(cfg.get("eps", 1e-6))
        self.registerParameter("weight", _torch().ones(self.features))

    def forward(self, input):
        x = _tensor_on_device(self, input)
        return _wrap(input, rmsNorm(x, self.p("weight"), eps=self.eps)[0])

    def backward(self, input, grad_out) -> dict:
        """Gradients of forward(input) for grad_out: {"x", "weight"}."""
        x = _tensor_on_device(self, input)
        gx, gw = rmsNormBackward(grad_out, x, self.p("weight"), eps=self.eps)
        return {"x": gx, "weight": gw}

    def __repr__(self):
        return f"RMSNorm({self.features})"


class GatedFeedForward(Module):
    """A feed-forward half-block on the features' residual stream, between
    message-passing layers: x + (act(n gate^T) * (n up^T)) down^T with
    n = rmsNorm(x, norm).  No counterpart in the reference.

    Features and parameters are f32 (``norm`` [features], ``gate`` and ``up``
    [hiddenFeatures, features], ``down`` [features, hiddenFeatures]); the
    products run on the tensor cores with operands in ``type``: "bf16"
    (default), "f16", or "e4m3" (forward only: the norm's output and the gate
    and up weights in 8 bits with a scale a row, the rest bf16)."""

    def __init__(self, config: Optional[dict] = None, **kw):
        super().__init__()
        torch = _torch()
        cfg = dict(config or {})
        cfg.update(kw)
        self.features = int(cfg["features"])
        self.hiddenFeatures = int(cfg["hiddenFeatures"])
        self.act = cfg.get("act", "silu")
        self.eps = float(cfg.get("eps", 1e-6))
        self.type = cfg.get("type", "bf16")
        if self.type not in ("bf16", "f16", "e4m3"):
            raise ValueError(f"type must be bf16, f16 or e4m3, got {self.type!r}")
        self.registerParameter("norm", torch.ones(self.features))
        stdv = np.sqrt(2.0 / (self.features + self.hiddenFeatures))
        for name in ("gate", "up"):
            self.registerParameter(name, _param((self.hiddenFeatures, self.features), stdv))
        self.registerParameter("down", _param((self.features, self.hiddenFeatures), stdv))

    def _half(self):
        torch = _torch()
        return torch.float16 if self.type == "f16" else torch.bfloat16

    def _eight(self, name):
        """A weight in e4m3 with one scale a row, not below the smallest normal
        number (as rmsNorm's): amax / 448 of a tiny row rounds to 0."""
        torch = _torch()
        w = self.p(name)
        amax = w.abs().amax(dim=1)
        scale = torch.where(amax > 0, (amax / 448.0).clamp_min(torch.finfo(w.dtype).tiny),
                            torch.ones_like(amax))
        return (w / scale[:, None]).to(torch.float8_e4m3fn), scale

    def forward(self, input):
        torch = _torch()
        x = _tensor_on_device(self, input)
        half = self._half()
        if self.type == "e4m3":
            n, _, s = rmsNorm(x, self.p("norm"), eps=self.eps, outType=torch.float8_e4m3fn)
            (g, gs), (u, us) = self._eight("gate"), self._eight("up")
            h = gatedLinear(n, g, u, act=self.act, xScale=s, gateScale=gs, upScale=us)
        else:
            n, _, _ = rmsNorm(x, self.p("norm"), eps=self.eps, outType=half)
            h = gatedLinear(n, self.p("gate").to(half), self.p("up").to(half), act=self.act)
        out = linearFused(h, self.p("down").to(half), residual=x, outType=torch.float32)
        return _wrap(input, out)

    @staticmethod
    def _into_f16(grad_out):
        """(grad_out scaled by a power of two and in f16, the inverse): the
        largest magnitude becomes 0.5 to 1, less where more than 4,096 rows add
        up, so that neither a mean over many rows falls into f16's subnormals
        nor a sum leaves its range."""
        torch = _torch()
        rows = grad_out.numel() // max(1, grad_out.shape[-1])
        if grad_out.numel() == 0:
            return grad_out.to(torch.float16), 1.0
        top = -max(0, (rows - 1).bit_length() - 12)
        by = (top - torch.frexp(grad_out.abs().amax())[1]).clamp(-126, 126)
        one = torch.ones((), device=grad_out.device)
        return (grad_out * torch.ldexp(one, by)).to(torch.float16), torch.ldexp(one, -by)

    def backward(self, input, grad_out) -> dict:
        """Gradients of forward(input) for grad_out [rows, features] (f32):
        {"x", "norm", "gate", "up", "down"}, f32.  The 16-bit activations are
        computed once more from the input; nothing of the forward is kept.
        The gradients between the products, and those of gate, up and down, are
        rounded to ``type`` once on their way; grad_out may be of any size."""
        if self.type == "e4m3":
            raise NotImplementedError("backward with e4m3 operands: train in bf16 or f16")
        x = _tensor_on_device(self, input)
        half = self._half()
        gate, up, down = (self.p(k).to(half) for k in ("gate", "up", "down"))
        n, _, _ = rmsNorm(x, self.p("norm"), eps=self.eps, outType=half)
        h = gatedLinear(n, gate, up, act=self.act)
        g, back = self._into_f16(grad_out) if self.type == "f16" else (grad_out.to(half), None)
        gh, gdown, _ = linearFusedBackward(g, h, down)
        gn, ggate, gup, _, _ = gatedLinearBackward(gh, n, gate, up, act=self.act)
        if back is not None:
            gn, ggate, gup, gdown = (v.float() * back for v in (gn, ggate, gup, gdown))
        gx, gnorm = rmsNormBackward(gn, x, self.p("norm"), eps=self.eps, gradTotal=grad_out)
        return {"x": gx, "norm": gnorm, "gate": ggate.float(), "up": gup.float(),
                "down": gdown.float()}

    def __repr__(self):
        return (f"GatedFeedForward({self.features} -> {self.hiddenFeatures} -> {self.features}, "
                f"{self.act}, {self.type})")


register_fusable(Linear)
