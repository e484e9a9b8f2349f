"""Block operators in mixed precision, and the choice head.

What a node model puts between its message-passing layers and at its end:

  rmsNorm, rmsNormBackward              root-mean-square norm of each row with
                                        the residual's addition; f32, 16-bit
                                        or e4m3 output with a scale a row
  gatedLinear, gatedLinearBackward      act(x Wg^T + bg) * (x Wu^T + bu)
  linearFused, linearFusedBackward      act(x W^T + b) + residual
  logProbs, logProbsBackward            log probability of each row's given
                                        choice, entropy, log-sum-exp and the
                                        top alternatives

The reference has no counterpart: its Linear (src/nn/linear.ts) and softmax
(src/core/tensor.ts:435-499) are f32 and stay `Linear`, `Softmax` and
`LogSoftmax`.  Tensors are CUDA tensors of one device, one- or two-dimensional
([features] is one row), rows any distance apart; results are fresh tensors on
torch's current stream.  Host threads may call at once, each on its own
stream.  Gradients are explicit calls, as the layers' ``backward`` is.  Errors
in arguments raise ValueError or TypeError, what the
library reports raises BGNNError.
"""
from __future__ import annotations

from typing import Optional

from . import _lib
from .backend import get_context, ptr

__all__ = ["rmsNorm", "rmsNormBackward", "rms_norm", "rms_norm_backward", "linearFused",
           "linearFusedBackward", "linear_fused", "linear_fused_backward", "gatedLinear",
           "gatedLinearBackward", "gated_linear", "gated_linear_backward", "logProbs",
           "logProbsBackward", "log_probs", "log_probs_backward"]

TOP_MAX = 32


def _torch():
    import torch

    return torch


_TENSOR = ()  # (torch.Tensor,), filled on first use


def _tensor_class():
    global _TENSOR
    _TENSOR = (_torch().Tensor,)
    return _TENSOR


_CODES = {}  # torch dtype -> bgnn_dtype, filled on first use


def _codes():
    if not _CODES:
        torch = _torch()
        _CODES.update({torch.float32: _lib.F32, torch.bfloat16: _lib.BF16,
                       torch.float16: _lib.F16, torch.float8_e4m3fn: _lib.E4M3})
    return _CODES


def _type(dtype, name, allowed):
    """bgnn_dtype of a torch dtype, one of `allowed`."""
    code = (_CODES or _codes()).get(dtype)
    if code not in allowed:
        names = {v: str(k).replace("torch.", "") for k, v in _codes().items()}
        raise TypeError(f"{name} has type {dtype}; "
                        f"allowed: {', '.join(names[a] for a in allowed)}")
    return code


_FLOATS = (_lib.F32, _lib.BF16, _lib.F16)
_HALVES = (_lib.BF16, _lib.F16)


def _tensor(t, name):
    if not isinstance(t, (_TENSOR or _tensor_class())):
        raise TypeError(f"{name} must be a CUDA tensor")
    return t


def _device(**tensors):
    """The one CUDA device that the given operands are on (after the checks of
    types and shapes, which need no device)."""
    dev = None
    for name, t in tensors.items():
        if t is None:
            continue
        d = t.get_device()  # -1: not on a GPU
        if d < 0:
            raise TypeError(f"{name} must be a CUDA tensor")
        if dev is None:
            dev = d
        elif d != dev:
            raise ValueError(f"{name} is on cuda:{d}, the other operands on cuda:{dev}")
    return dev


def _rows(t, name):
    """[rows, cols] with unit column stride and rows that do not overlap, and
    whether the tensor was one row."""
    _tensor(t, name)
    dim = t.dim()
    if dim == 1:
        t = t.unsqueeze(0)
    elif dim != 2:
        raise ValueError(f"{name}: expects 1D or 2D input, got {dim}D")
    rows, cols = t.shape
    if not t.is_contiguous() and ((cols > 1 and t.stride(1) != 1) or
                                  (rows > 1 and t.stride(0) < cols)):
        t = t.contiguous()
    if cols >= 2 ** 31:
        raise ValueError(f"{name}: a row of {cols} elements")
    return t, dim == 1


def _ld(t):
    """Row stride in elements (a single row's is its length)."""
    rows, cols = t.shape
    return t.stride(0) if rows > 1 else cols


def _vec(t, n, name, allowed):
    """A contiguous [n] vector and its type code; (None, 0) for None."""
    if t is None:
        return None, 0
    _tensor(t, name)
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name}: expected shape [{n}], got {list(t.shape)}")
    return t if t.is_contiguous() else t.contiguous(), _type(t.dtype, name, allowed)


def _same_shape(t, rows, cols, name):
    if tuple(t.shape) != (rows, cols):
        raise ValueError(f"{name}: expected shape [{rows}, {cols}], got {list(t.shape)}")


def _act(act):
    """(bgnn_act, parameter) of None, a name, or (name, parameter)."""
    name, param = act if isinstance(act, tuple) else (act, 1.0 if act == "elu" else 0.01)
    if name not in _lib.ACT:
        raise ValueError(f"unknown activation {name!r}")
    return _lib.ACT[name], float(param)


def _empty(shape, dtype, like):
    return like.new_empty(shape, dtype=dtype)


# ---------------------------------------------------------------------------
def rmsNorm(x, weight, residual=None, eps: float = 1e-6, outType=None):
    """(out, total, scale): the rows of ``total = x + residual`` (rounded to
    the residual's type; x itself without one) scaled to unit root mean
    square and by ``weight``.

    x is f32, bf16 or f16, residual x's type or f32.  outType (x's type when
    None) f32, bf16, f16, or torch.float8_e4m3fn: then ``out * scale[row]`` is
    the result, scale [rows] f32 being the row's largest magnitude / 448;
    scale is None for the other types.  The squares are added in f32: rows
    whose sum of squares passes 3.4e38 give 0."""
    torch = _torch()
    t, one = _rows(x, "x")
    rows, cols = t.shape
    xt = _type(t.dtype, "x", _FLOATS)
    out_dtype = t.dtype if outType is None else outType
    ot = _type(out_dtype, "outType", _FLOATS + (_lib.E4M3,))
    w, wt = _vec(weight, cols, "weight", _FLOATS)
    r, rt, total = None, 0, x
    if residual is not None:
        r, _ = _rows(residual, "residual")
        rt = _type(r.dtype, "residual", (xt, _lib.F32))
        _same_shape(r, rows, cols, "residual")
    dev = _device(x=t, weight=w, residual=r)
    if r is not None:
        total = _empty((rows, cols), r.dtype, t)
    out = _empty((rows, cols), out_dtype, t)
    scale = _empty((rows,), torch.float32, t) if ot == _lib.E4M3 else None
    get_context(dev).call("bgnn_rms_norm", xt, ptr(t), _ld(t), rt, ptr(r),
                          0 if r is None else _ld(r), wt, ptr(w), rows, cols, float(eps),
                          ptr(total) if r is not None else None, ot, ptr(out), ptr(scale))
    if one:
        out = out[0]
        total = total[0] if residual is not None else total
    return out, total, scale


def rmsNormBackward(gradOut, total, weight, eps: float = 1e-6, gradTotal=None):
    """(gradX, gradWeight) of rmsNorm from its ``total`` (x without a
    residual).  gradX, in total's type, is the gradient of x and of the
    residual alike; gradTotal is the gradient that reaches ``total`` along
    the residual stream.  gradOut has total's type, or any when total is f32."""
    t, one = _rows(total, "total")
    rows, cols = t.shape
    tt = _type(t.dtype, "total", _FLOATS)
    g, _ = _rows(gradOut, "gradOut")
    _same_shape(g, rows, cols, "gradOut")
    gt = _type(g.dtype, "gradOut", _FLOATS if tt == _lib.F32 else (tt,))
    w, wt = _vec(weight, cols, "weight", _FLOATS)
    s = None
    if gradTotal is not None:
        s, _ = _rows(gradTotal, "gradTotal")
        _same_shape(s, rows, cols, "gradTotal")
        _type(s.dtype, "gradTotal", (tt,))
    dev = _device(total=t, gradOut=g, weight=w, gradTotal=s)
    gx = _empty((rows, cols), t.dtype, t)
    gw = _empty((cols,), w.dtype, t)
    get_context(dev).call("bgnn_rms_norm_backward", gt, ptr(g), _ld(g), tt, ptr(t), _ld(t),
                          ptr(s), 0 if s is None else _ld(s), wt, ptr(w), rows, cols, float(eps),
                          ptr(gx), ptr(gw))
    return (gx[0] if one else gx), gw


# ---------------------------------------------------------------------------
def _operand(t, name, code=None):
    """An operand of a product: its rows and type."""
    r, one = _rows(t, name)
    c = _type(r.dtype, name, (_lib.BF16, _lib.F16, _lib.E4M3))
    if code is not None and c != code:
        raise TypeError(f"{name} has type {r.dtype}, the other operand another")
    return r, c, one


def _product(x, weights, names, scales, scale_names, xScale):
    """The checks that the products share: x [m, k] and weights [n, k]."""
    xr, code, one = _operand(x, "x")
    m, k = xr.shape
    ws, n = [], None
    for w, name in zip(weights, names):
        if getattr(w, "dim", lambda: 0)() != 2:
            raise ValueError(f"{name}: expects a 2D weight [out, in]")
        r, _, _ = _operand(w, name, code)
        if r.shape[1] != k:
            raise ValueError(f"Expected input size {r.shape[1]}, got {k}")
        if n is not None and r.shape[0] != n:
            raise ValueError(f"{name}: expected {n} rows, got {r.shape[0]}")
        n = int(r.shape[0])
        ws.append(r)
    eight = code == _lib.E4M3
    sc = []
    for s, name, ln in zip([xScale] + list(scales), ["xScale"] + list(scale_names),
                           [m] + [n] * len(ws)):
        if eight and s is None:
            raise ValueError(f"{name}: e4m3 operands need a scale a row")
        if not eight and s is not None:
            raise ValueError(f"{name}: only e4m3 operands have scales")
        sc.append(_vec(s, ln, name, (_lib.F32,))[0])
    return xr, code, one, m, k, n, ws, sc


def _out_type(outType, xr, code):
    torch = _torch()
    if outType is None:
        outType = torch.bfloat16 if code == _lib.E4M3 else xr.dtype
    return outType, _type(outType, "outType", _FLOATS)


def _biases(pair, names, n):
    out, code = [], None
    for b, name in zip(pair, names):
        v, c = _vec(b, n, name, _FLOATS)
        if v is not None:
            if code is not None and c != code:
                raise TypeError(f"{name} has type {v.dtype}, the other bias another")
            code = c
        out.append(v)
    return out, code or 0


def linearFused(x, weight, bias=None, act=None, residual=None, outType=None, xScale=None,
                weightScale=None):
    """act(x weight^T + bias) + residual, [m, out].

    x [m, in] and weight [out, in] are bf16 or f16, or torch.float8_e4m3fn
    with one f32 scale a row each (xScale [m], weightScale [out]); f32
    operands are `Linear`'s.  act: None, a name, or (name, parameter).  bias,
    residual and outType (x's type when None, bf16 under e4m3) are f32, bf16
    or f16."""
    xr, code, one, m, k, n, (w,), (xs, s) = _product(
        x, [weight], ["weight"], [weightScale], ["weightScale"], xScale)
    dtype, ot = _out_type(outType, xr, code)
    (b,), bt = _biases([bias], ["bias"], n)
    a, p = _act(act)
    r, rt = None, 0
    if residual is not None:
        r, _ = _rows(residual, "residual")
        rt = _type(r.dtype, "residual", _FLOATS)
        _same_shape(r, m, n, "residual")
    dev = _device(x=xr, weight=w, bias=b, residual=r, xScale=xs, weightScale=s)
    out = _empty((m, n), dtype, xr)
    get_context(dev).call("bgnn_linear_fused", code, ptr(xr), _ld(xr), ptr(xs), ptr(w), _ld(w),
                          ptr(s), m, k, n, bt, ptr(b), a, p, rt, ptr(r),
                          0 if r is None else _ld(r), ot, ptr(out), n)
    return out[0] if one else out


def _grad_rows(gradOut, xr, m, n):
    g, _ = _rows(gradOut, "gradOut")
    _same_shape(g, m, n, "gradOut")
    if g.dtype != xr.dtype:
        raise TypeError(f"gradOut has type {g.dtype}, the operands {xr.dtype}")
    return g


def _no_eight(x):
    if getattr(x, "dtype", None) == _torch().float8_e4m3fn:
        raise TypeError("e4m3 operands have no backward: train in bf16 or f16")


def linearFusedBackward(gradOut, x, weight, bias=None, act=None):
    """(gradX, gradWeight, gradBias) of linearFused for bf16 or f16 operands;
    gradBias is None without a bias, the residual's gradient is gradOut
    itself.  gradOut [m, out] has the operands' type, and so have gradX and
    gradWeight; gradBias has the bias's."""
    _no_eight(x)
    xr, code, one, m, k, n, (w,), _ = _product(x, [weight], ["weight"], [None],
                                                    ["weightScale"], None)
    g = _grad_rows(gradOut, xr, m, n)
    (b,), bt = _biases([bias], ["bias"], n)
    a, p = _act(act)
    dev = _device(x=xr, weight=w, bias=b, gradOut=g)
    gx, gw = _empty((m, k), xr.dtype, xr), _empty((n, k), xr.dtype, xr)
    gb = None if b is None else _empty((n,), b.dtype, xr)
    get_context(dev).call("bgnn_linear_fused_backward", code, ptr(g), _ld(g), ptr(xr), _ld(xr),
                          ptr(w), _ld(w), m, k, n, bt, ptr(b), a, p, ptr(gx), ptr(gw), ptr(gb))
    return (gx[0] if one else gx), gw, gb


def gatedLinear(x, weightGate, weightUp, biasGate=None, biasUp=None, act="silu", outType=None,
                xScale=None, gateScale=None, upScale=None):
    """act(x weightGate^T + biasGate) * (x weightUp^T + biasUp), [m, hidden].

    x [m, in], both weights [hidden, in]; types and scales as linearFused."""
    xr, code, one, m, k, n, (wg, wu), (xs, gs, us) = _product(
        x, [weightGate, weightUp], ["weightGate", "weightUp"], [gateScale, upScale],
        ["gateScale", "upScale"], xScale)
    dtype, ot = _out_type(outType, xr, code)
    (bg, bu), bt = _biases([biasGate, biasUp], ["biasGate", "biasUp"], n)
    a, p = _act(act)
    dev = _device(x=xr, weightGate=wg, weightUp=wu, biasGate=bg, biasUp=bu, xScale=xs,
                  gateScale=gs, upScale=us)
    out = _empty((m, n), dtype, xr)
    get_context(dev).call("bgnn_gated_linear", code, ptr(xr), _ld(xr), ptr(xs), ptr(wg), _ld(wg),
                          ptr(gs), ptr(wu), _ld(wu), ptr(us), m, k, n, bt, ptr(bg), ptr(bu), a, p,
                          ot, ptr(out), n)
    return out[0] if one else out


def gatedLinearBackward(gradOut, x, weightGate, weightUp, biasGate=None, biasUp=None,
                        act="silu"):
    """(gradX, gradWeightGate, gradWeightUp, gradBiasGate, gradBiasUp) of
    gatedLinear for bf16 or f16 operands, from the forward's inputs alone
    (both products run once more).  The bias gradients are None without the
    bias; types as linearFusedBackward."""
    _no_eight(x)
    xr, code, one, m, k, n, (wg, wu), _ = _product(
        x, [weightGate, weightUp], ["weightGate", "weightUp"], [None, None],
        ["gateScale", "upScale"], None)
    g = _grad_rows(gradOut, xr, m, n)
    (bg, bu), bt = _biases([biasGate, biasUp], ["biasGate", "biasUp"], n)
    a, p = _act(act)
    dev = _device(x=xr, weightGate=wg, weightUp=wu, biasGate=bg, biasUp=bu, gradOut=g)
    gx = _empty((m, k), xr.dtype, xr)
    gwg, gwu = _empty((n, k), xr.dtype, xr), _empty((n, k), xr.dtype, xr)
    gbg = None if bg is None else _empty((n,), bg.dtype, xr)
    gbu = None if bu is None else _empty((n,), bu.dtype, xr)
    get_context(dev).call("bgnn_gated_linear_backward", code, ptr(g), _ld(g), ptr(xr), _ld(xr),
                          ptr(wg), _ld(wg), ptr(wu), _ld(wu), m, k, n, bt, ptr(bg), ptr(bu), a, p,
                          ptr(gx), ptr(gwg), ptr(gwu), ptr(gbg), ptr(gbu))
    return (gx[0] if one else gx), gwg, gwu, gbg, gbu


# ---------------------------------------------------------------------------
def _targets(targets, rows):
    """[rows] u32 ids as an int32 tensor; -1 is "no choice given"."""
    torch = _torch()
    _tensor(targets, "targets")
    if targets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"targets has type {targets.dtype}; allowed: int32, int64")
    t = targets.reshape(-1)
    if t.shape[0] != rows:
        raise ValueError(f"targets: expected {rows} entries, got {t.shape[0]}")
    if t.dtype == torch.int64:  # an id that int32 cannot hold stays out of range
        t = t.clamp(-2, 2 ** 31 - 1).to(torch.int32)
    return t.contiguous()


def _mask(mask, rows, cols):
    """(uint8 mask, row stride): [cols] for all rows, or [rows, cols]."""
    torch = _torch()
    if mask is None:
        return None, 0
    _tensor(mask, "mask")
    if mask.dtype not in (torch.bool, torch.uint8):
        raise TypeError(f"mask has type {mask.dtype}; allowed: bool, uint8")
    if mask.dim() == 1 and mask.shape[0] == cols:
        return mask.contiguous(), 0
    m, _ = _rows(mask, "mask")
    _same_shape(m, rows, cols, "mask")
    return m, _ld(m)


def _floats(t, rows, name):
    torch = _torch()
    if t is None:
        return None
    _tensor(t, name)
    if t.dtype != torch.float32 or t.numel() != rows:
        raise ValueError(f"{name}: expected {rows} float32 values")
    return t.reshape(-1).contiguous()


def logProbs(logits, targets, mask=None, topK: int = 0):
    """(logProb, entropy, lse, topIds, topLogProbs) of each row of logits
    [rows, cols] (f32, bf16 or f16; [cols] is one row), f32 but the ids.

    targets [rows] (int32 or int64) holds each row's given choice, -1 for
    none (log probability 0); mask (bool or uint8, [cols] or [rows, cols])
    takes choices out where it is not 0, as does a logit of -inf.  A target
    that is out has log probability -inf; a row with nothing left has
    log-sum-exp -inf and entropy 0.  topIds / topLogProbs [rows, topK]
    (int32; topK <= 32; None for 0) list the most probable choices, equal
    logits in ascending index, -1 / -inf beyond the last.  A target outside
    the row raises BGNNIndexError at the next synchronising call."""
    torch = _torch()
    x, one = _rows(logits, "logits")
    rows, cols = x.shape
    code = _type(x.dtype, "logits", _FLOATS)
    if not 0 <= int(topK) <= TOP_MAX:
        raise ValueError(f"topK must be in [0, {TOP_MAX}], got {topK}")
    if rows >= 2 ** 31:
        raise ValueError(f"logits: {rows} rows")
    t = _targets(targets, rows)
    m, ldm = _mask(mask, rows, cols)
    dev = _device(logits=x, targets=t, mask=m)
    logp, ent, lse = _empty((3, rows), torch.float32, x).unbind(0)
    ids = top = None
    if topK:
        ids = _empty((rows, int(topK)), torch.int32, x)
        top = _empty((rows, int(topK)), torch.float32, x)
    get_context(dev).call("bgnn_log_probs", code, ptr(x), _ld(x), rows, cols, ptr(m), ldm, ptr(t),
                          int(topK), ptr(logp), ptr(ent), ptr(lse), ptr(ids), ptr(top))
    return logp, ent, lse, ids, top


def logProbsBackward(logits, targets, lse, entropy, gradLogProb, gradEntropy=None, mask=None):
    """The logits' gradient, in their type and shape, for the gradients of
    logProbs' logProb and entropy ([rows] f32, either None), from the lse and
    entropy that logProbs returned for the same logits, targets and mask."""
    x, one = _rows(logits, "logits")
    rows, cols = x.shape
    code = _type(x.dtype, "logits", _FLOATS)
    if rows >= 2 ** 31:
        raise ValueError(f"logits: {rows} rows")
    t = _targets(targets, rows)
    m, ldm = _mask(mask, rows, cols)
    l, h = _floats(lse, rows, "lse"), _floats(entropy, rows, "entropy")
    gl = _floats(gradLogProb, rows, "gradLogProb")
    gh = _floats(gradEntropy, rows, "gradEntropy")
    if l is None or h is None:
        raise ValueError("logProbsBackward needs the forward's lse and entropy")
    dev = _device(logits=x, targets=t, mask=m, lse=l, entropy=h, gradLogProb=gl, gradEntropy=gh)
    out = _empty((rows, cols), x.dtype, x)
    get_context(dev).call("bgnn_log_probs_backward", code, ptr(x), _ld(x), rows, cols, ptr(m), ldm,
                          ptr(t), ptr(l), ptr(h), ptr(gl), ptr(gh), ptr(out))
    return out[0] if one else out


rms_norm, rms_norm_backward = rmsNorm, rmsNormBackward
linear_fused, linear_fused_backward = linearFused, linearFusedBackward
gated_linear, gated_linear_backward = gatedLinear, gatedLinearBackward
log_probs, log_probs_backward = logProbs, logProbsBackward
