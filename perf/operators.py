"""Timed cases of the dense block operators and the choice head.

Four operators, as a node model uses them between and after its message
passing layers:

  norm    rmsNorm / rmsNormBackward: root-mean-square norm of a row with the
          residual's addition, f32 / 16-bit output or e4m3 with a scale a row
  gated   gatedLinear / gatedLinearBackward: act(x Wg^T + bg) * (x Wu^T + bu)
  dense   linearFused / linearFusedBackward: act(x W^T + b) + residual
  choice  logProbs / logProbsBackward: log probability of each row's given
          choice, entropy, log-sum-exp and the top alternatives

``own`` false: plain torch operations in 32 bits; true: the framework's calls.
"""
import math

import torch

own = False

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16,
     "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}
EPS = 1e-6
E4M3_MAX = 448.0


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def norm_case(rows, cols, type, residual, out):
    return {"op": "norm", "rows": rows, "cols": cols, "type": type, "residual": residual,
            "out": out}


def norm_backward_case(rows, cols, type, stream):
    return {"op": "norm_backward", "rows": rows, "cols": cols, "type": type, "stream": stream}


def gated_case(m, k, n, type, act, bias=False):
    return {"op": "gated", "m": m, "k": k, "n": n, "type": type, "act": act, "bias": bias}


def gated_backward_case(m, k, n, type, act, bias=False):
    return {"op": "gated_backward", "m": m, "k": k, "n": n, "type": type, "act": act,
            "bias": bias}


def dense_case(m, k, n, type, act, bias, residual, out):
    return {"op": "dense", "m": m, "k": k, "n": n, "type": type, "act": act, "bias": bias,
            "residual": residual, "out": out}


def dense_backward_case(m, k, n, type, act, bias):
    return {"op": "dense_backward", "m": m, "k": k, "n": n, "type": type, "act": act,
            "bias": bias}


def choice_case(rows, cols, type, mask, top):
    return {"op": "choice", "rows": rows, "cols": cols, "type": type, "mask": mask, "top": top}


def choice_backward_case(rows, cols, type, mask):
    return {"op": "choice_backward", "rows": rows, "cols": cols, "type": type, "mask": mask}


def listed():
    return [
        # one new node (or token) before an 8-bit projection: latency
        dict(norm_case(1, 1024, "bf16", "bf16", "e4m3"), name="norm one row, e4m3 out"),
        # every node of the 2.45M-node graph, f32 residual stream, 16-bit operand out
        dict(norm_case(2450000, 256, "f32", "f32", "bf16"), name="norm all nodes"),
        # training at the citation features' odd width
        dict(norm_backward_case(20000, 1433, "f16", True), name="norm backward, odd width"),
        # one token served
        dict(gated_case(1, 1024, 4096, "bf16", "silu"), name="gated one token"),
        # the half-block over every node of the 2.45M-node graph
        dict(gated_case(2450000, 256, 512, "bf16", "silu"), name="gated all nodes"),
        # a ragged batch served with 8-bit operands
        dict(gated_case(4097, 1024, 2736, "e4m3", "gelu"), name="gated e4m3 ragged"),
        # a training step's backward at ordinary widths
        dict(gated_backward_case(16384, 1024, 4096, "bf16", "silu"), name="gated backward"),
        # the product back onto the f32 residual stream
        dict(dense_case(16384, 4096, 1024, "bf16", None, False, "f32", "f32"),
             name="product onto the stream"),
        # the 47-class transform of the 256-wide layers in training, odd row count
        dict(dense_backward_case(100003, 256, 47, "f16", "gelu", True),
             name="product backward, 47 wide"),
        # one answer over every node of the graph, some already taken
        dict(choice_case(1, 2450000, "f32", "columns", 20), name="choice among all nodes"),
        # a batch's log probabilities with the alternatives
        dict(choice_case(8192, 32000, "bf16", "none", 20), name="choices of a batch"),
        # the loss's gradient, an odd row length, each row with a mask of its own
        dict(choice_backward_case(4096, 50001, "f16", "rows"), name="choices backward"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_backward", "gated", "gated", "gated_backward", "dense",
                     "dense", "dense_backward", "choice", "choice", "choice_backward"])
    if op in ("norm", "norm_backward"):
        cols = _log(rng, 16, 8192)
        rows = _log(rng, 1, min(2450000, max(1, 600000000 // cols)))
        t = rng.choice(["f32", "bf16", "f16"])
        if op == "norm":
            return norm_case(rows, cols, t, rng.choice(["none", t, "f32"]),
                             rng.choice([t, "bf16", "e4m3"]))
        return norm_backward_case(rows, cols, t, rng.random() < 0.5)
    if op in ("choice", "choice_backward"):
        cols = _log(rng, 2, 2450000)
        rows = _log(rng, 1, max(1, min(100000, 200000000 // cols)))
        t = rng.choice(["f32", "bf16", "f16"])
        mask = rng.choice(["none", "columns", "rows"])
        if op == "choice":
            return choice_case(rows, cols, t, mask, rng.choice([0, 1, 5, 20, 32]))
        return choice_backward_case(rows, cols, t, mask)
    k, n = _log(rng, 16, 4096), _log(rng, 16, 4096)
    act = rng.choice(["silu", "gelu", "relu", "sigmoid", "tanh"])
    bias = rng.random() < 0.5
    half = rng.choice(["bf16", "f16"])
    # at most the work of the largest listed case of the direction
    if op.endswith("backward"):
        m = _log(rng, 1, max(1, min(1000000, 60000000000 // (k * n))))
        if op == "gated_backward":
            return gated_backward_case(m, k, n, half, act, bias)
        return dense_backward_case(m, k, n, half, rng.choice([None, act]), bias)
    m = _log(rng, 1, max(1, min(2000000, 60000000000 // (k * n))))
    t = rng.choice([half, half, "e4m3"])
    if op == "gated":
        return gated_case(m, k, n, t, act, bias)
    wide = "bf16" if t == "e4m3" else t
    return dense_case(m, k, n, t, rng.choice([None, act]), bias,
                      rng.choice(["none", wide, "f32"]), rng.choice([wide, "f32"]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _quantised(x):
    """e4m3 values and one f32 scale a row."""
    scale = x.abs().amax(dim=1).clamp_min(1e-12) / E4M3_MAX
    return (x / scale[:, None]).to(T["e4m3"]), scale


def _operand(g, rows, cols, type, std):
    """An operand of a product: (values, scales or None)."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    if std is not None:
        x *= std
    if type == "e4m3":
        return _quantised(x)
    return x.to(T[type]), None


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = dict(case)

    def normal(*shape, type="f32", std=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * std).to(T[type])

    if op.startswith("norm"):
        r, c, t = case["rows"], case["cols"], case["type"]
        s["weight"] = normal(c, std=0.2) + 1.0
        if op == "norm":
            s["x"] = normal(r, c, type=t)
            s["residual_in"] = (None if case["residual"] == "none"
                                else normal(r, c, type=case["residual"], std=3.0))
        else:
            s["total"] = normal(r, c, type=t, std=3.0)
            s["grad"] = normal(r, c, type=t)
            s["grad_total"] = normal(r, c, type=t) if case["stream"] else None
    elif op.startswith("choice"):
        r, c = case["rows"], case["cols"]
        s["logits"] = normal(r, c, type=case["type"], std=2.0)
        s["targets"] = torch.randint(0, c, (r,), device="cuda", generator=g, dtype=torch.int32)
        s["mask_in"] = None
        if case["mask"] == "columns":
            s["mask_in"] = (torch.rand(c, device="cuda", generator=g) < 0.1).to(torch.uint8)
        elif case["mask"] == "rows":
            m = torch.rand(r, c, device="cuda", generator=g) < 0.3
            m |= torch.rand(r, 1, device="cuda", generator=g) < 0.01  # rows left empty
            s["mask_in"] = m.to(torch.uint8)
        if op == "choice_backward":
            x = _left(s["logits"], s["mask_in"])
            lse = torch.logsumexp(x, dim=1)
            p = torch.exp(x - torch.where(lse == -math.inf, 0.0, lse)[:, None])
            s["lse"] = lse
            s["entropy"] = torch.where(lse == -math.inf, 0.0, lse - torch.where(
                p > 0, p * x, 0.0).sum(dim=1))
            # a mean over the rows; f16 trains with a scaled loss, for its narrow exponent
            by = 1024.0 if case["type"] == "f16" else 1.0 / r
            s["grad_logp"] = -by * torch.rand(r, device="cuda", generator=g)
            s["grad_entropy"] = 0.01 * by * torch.randn(r, device="cuda", generator=g)
    else:
        m, k, n, t = case["m"], case["k"], case["n"], case["type"]
        std = math.sqrt(2.0 / (k + n))
        s["x"], s["x_scale"] = _operand(g, m, k, t, None)
        wide = "bf16" if t == "e4m3" else t
        if op.startswith("gated"):
            s["wg"], s["wg_scale"] = _operand(g, n, k, t, std)
            s["wu"], s["wu_scale"] = _operand(g, n, k, t, std)
            s["bg"] = normal(n, type=wide, std=0.1) if case["bias"] else None
            s["bu"] = normal(n, type=wide, std=0.1) if case["bias"] else None
        else:
            s["w"], s["w_scale"] = _operand(g, n, k, t, std)
            s["b"] = normal(n, type=wide, std=0.1) if case["bias"] else None
            if op == "dense":
                s["residual_in"] = (None if case["residual"] == "none"
                                    else normal(m, n, type=case["residual"]))
        if op.endswith("backward"):
            s["grad"] = normal(m, n, type=t)
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _left(logits, mask):
    """The logits in 32 bits, -inf where the mask takes a choice out."""
    x = logits.float()
    return x if mask is None else torch.where(mask != 0, -math.inf, x)


def _value(x, scale):
    return x.float() if scale is None else x.float() * scale[:, None]


def _act(z, act):
    if act is None:
        return z
    if act == "relu":
        return torch.clamp_min(z, 0.0)
    if act == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    if act == "tanh":
        return torch.tanh(z)
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    c = math.sqrt(2.0 / math.pi)  # gelu, tanh form
    return 0.5 * z * (1.0 + torch.tanh(c * (z + 0.044715 * z * z * z)))


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 - s)
    if act == "tanh":
        t = torch.tanh(z)
        return 1.0 - t * t
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)


def _project(x, w, b):
    z = x @ w.t()
    return z if b is None else z + b.float()


def _plain_norm(s):
    x = s["x"]
    out = T[s["out"]]
    total = x
    if s["residual_in"] is not None:
        total = (x.float() + s["residual_in"].float()).to(s["residual_in"].dtype)
    t = total.float()
    y = t * torch.rsqrt((t * t).mean(dim=1, keepdim=True) + EPS) * s["weight"]
    r = {}
    if s["residual_in"] is not None:
        r["total"] = total
    if out == T["e4m3"]:
        amax = y.abs().amax(dim=1, keepdim=True)
        scale = torch.where(amax > 0, amax / E4M3_MAX, 1.0)
        r["out"], r["scale"] = (y / scale).to(out), scale[:, 0]
    else:
        r["out"] = y.to(out)
    return r


def _plain_norm_backward(s):
    t, gy, w = s["total"].float(), s["grad"].float(), s["weight"]
    rs = torch.rsqrt((t * t).mean(dim=1, keepdim=True) + EPS)
    xh = t * rs
    gw = gy * w
    gx = rs * (gw - xh * (gw * xh).mean(dim=1, keepdim=True))
    if s["grad_total"] is not None:
        gx = gx + s["grad_total"].float()
    return {"x": gx.to(s["total"].dtype), "weight": (gy * xh).sum(dim=0)}


def _plain_gated(s):
    x = _value(s["x"], s["x_scale"])
    g = _project(x, _value(s["wg"], s["wg_scale"]), s["bg"])
    u = _project(x, _value(s["wu"], s["wu_scale"]), s["bu"])
    return {"out": (_act(g, s["act"]) * u).to(T["bf16" if s["type"] == "e4m3" else s["type"]])}


def _plain_gated_backward(s):
    x, wg, wu, dh = s["x"].float(), s["wg"].float(), s["wu"].float(), s["grad"].float()
    t = s["x"].dtype
    g, u = _project(x, wg, s["bg"]), _project(x, wu, s["bu"])
    dg, du = dh * u * _act_grad(g, s["act"]), dh * _act(g, s["act"])
    r = {"x": (dg @ wg + du @ wu).to(t), "wg": (dg.t() @ x).to(t), "wu": (du.t() @ x).to(t)}
    if s["bg"] is not None:
        r["bg"], r["bu"] = dg.sum(dim=0).to(t), du.sum(dim=0).to(t)
    return r


def _plain_dense(s):
    z = _project(_value(s["x"], s["x_scale"]), _value(s["w"], s["w_scale"]), s["b"])
    z = _act(z, s["act"])
    if s["residual_in"] is not None:
        z = z + s["residual_in"].float()
    return {"out": z.to(T[s["out"]])}


def _plain_dense_backward(s):
    x, w, dz = s["x"].float(), s["w"].float(), s["grad"].float()
    t = s["x"].dtype
    if s["act"] is not None:
        dz = dz * _act_grad(_project(x, w, s["b"]), s["act"])
    r = {"x": (dz @ w).to(t), "w": (dz.t() @ x).to(t)}
    if s["b"] is not None:
        r["b"] = dz.sum(dim=0).to(t)
    return r


def _plain_choice(s):
    x = _left(s["logits"], s["mask_in"])
    rows, cols = x.shape
    top = s["top"]
    mx = x.amax(dim=1, keepdim=True)
    mx = torch.where(mx == -math.inf, 0.0, mx)
    e = torch.exp(x - mx)
    z = e.sum(dim=1)
    empty = z == 0
    lse = mx[:, 0] + torch.log(z)
    xt = torch.gather(x, 1, s["targets"].long()[:, None])[:, 0]
    r = {"logp": torch.where(empty, -math.inf, xt - lse), "lse": lse}
    ent = torch.where(e > 0, e * (x - mx), 0.0).sum(dim=1)
    r["entropy"] = torch.where(empty, 0.0, torch.log(z) - ent / z)
    if top:
        bits = (x + 0.0).view(torch.int32)  # a whole number that orders as the logit does
        key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * 4294967296
        key += 4294967295 - torch.arange(cols, device=x.device)  # ties: lowest index first
        key = torch.topk(key, min(top, cols), dim=1).values
        ids = 4294967295 - (key & 4294967295)
        v = torch.gather(x, 1, ids)
        none = v == -math.inf
        ids = torch.where(none, -1, ids).int()
        lp = torch.where(none, -math.inf, v - lse[:, None])
        r["top_ids"] = torch.nn.functional.pad(ids, (0, top - ids.shape[1]), value=-1)
        r["top_logp"] = torch.nn.functional.pad(lp, (0, top - lp.shape[1]), value=-math.inf)
    return r


def _plain_choice_backward(s):
    x = _left(s["logits"], s["mask_in"])
    lse = s["lse"][:, None]
    logp = x - torch.where(lse == -math.inf, 0.0, lse)
    p = torch.exp(logp)
    gl, ge = s["grad_logp"][:, None], s["grad_entropy"][:, None]
    d = torch.where(p > 0, p * (-gl - ge * (logp + s["entropy"][:, None])), 0.0)
    at = s["targets"].long()[:, None]
    d.scatter_add_(1, at, torch.where(torch.gather(x, 1, at) > -math.inf, gl, 0.0))
    return {"logits": d.to(s["logits"].dtype)}


PLAIN = {"norm": _plain_norm, "norm_backward": _plain_norm_backward, "gated": _plain_gated,
         "gated_backward": _plain_gated_backward, "dense": _plain_dense,
         "dense_backward": _plain_dense_backward, "choice": _plain_choice,
         "choice_backward": _plain_choice_backward}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own_run(s):
    import browsergnn_b200 as bg

    op = s["op"]
    if op == "norm":
        out, total, scale = bg.rmsNorm(s["x"], s["weight"], residual=s["residual_in"], eps=EPS,
                                       outType=T[s["out"]])
        r = {"out": out}
        if s["residual_in"] is not None:
            r["total"] = total
        if scale is not None:
            r["scale"] = scale
        return r
    if op == "norm_backward":
        gx, gw = bg.rmsNormBackward(s["grad"], s["total"], s["weight"], eps=EPS,
                                    gradTotal=s["grad_total"])
        return {"x": gx, "weight": gw}
    if op == "gated":
        return {"out": bg.gatedLinear(s["x"], s["wg"], s["wu"], biasGate=s["bg"],
                                      biasUp=s["bu"], act=s["act"], xScale=s["x_scale"],
                                      gateScale=s["wg_scale"], upScale=s["wu_scale"])}
    if op == "gated_backward":
        gx, gwg, gwu, gbg, gbu = bg.gatedLinearBackward(
            s["grad"], s["x"], s["wg"], s["wu"], biasGate=s["bg"], biasUp=s["bu"], act=s["act"])
        r = {"x": gx, "wg": gwg, "wu": gwu}
        if s["bg"] is not None:
            r["bg"], r["bu"] = gbg, gbu
        return r
    if op == "dense":
        return {"out": bg.linearFused(s["x"], s["w"], bias=s["b"], act=s["act"],
                                      residual=s["residual_in"], outType=T[s["out"]],
                                      xScale=s["x_scale"], weightScale=s["w_scale"])}
    if op == "dense_backward":
        gx, gw, gb = bg.linearFusedBackward(s["grad"], s["x"], s["w"], bias=s["b"], act=s["act"])
        r = {"x": gx, "w": gw}
        if s["b"] is not None:
            r["b"] = gb
        return r
    if op == "choice":
        logp, entropy, lse, ids, top = bg.logProbs(s["logits"], s["targets"], mask=s["mask_in"],
                                                   topK=s["top"])
        r = {"logp": logp, "entropy": entropy, "lse": lse}
        if s["top"]:
            r["top_ids"], r["top_logp"] = ids, top
        return r
    return {"logits": bg.logProbsBackward(s["logits"], s["targets"], s["lse"], s["entropy"],
                                          s["grad_logp"], gradEntropy=s["grad_entropy"],
                                          mask=s["mask_in"])}


def run(state):
    if own:
        return _own_run(state)
    return PLAIN[state["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "norm":
        e = case["rows"] * case["cols"]
        b = e * (SIZE[case["type"]] + SIZE[case["out"]]) + 4 * case["cols"]
        if case["residual"] != "none":
            b += 2 * e * SIZE[case["residual"]]
        if case["out"] == "e4m3":
            b += 4 * case["rows"]
        return {"bytes": b, "flops": 6 * e}
    if op == "norm_backward":
        e, z = case["rows"] * case["cols"], SIZE[case["type"]]
        return {"bytes": e * z * (4 if case["stream"] else 3) + 8 * case["cols"], "flops": 12 * e}
    if op.startswith("choice"):
        r, c, z = case["rows"], case["cols"], SIZE[case["type"]]
        b = r * c * z + {"none": 0, "columns": c, "rows": r * c}[case["mask"]]
        if op == "choice":
            return {"bytes": b + r * (16 + 8 * case["top"]), "flops": 5 * r * c}
        return {"bytes": b + r * c * z + 20 * r, "flops": 6 * r * c}
    m, k, n, z = case["m"], case["k"], case["n"], SIZE[case["type"]]
    two = 2 if op.startswith("gated") else 1
    wide = 2 if case["type"] == "e4m3" else z
    b = (m * k + two * n * k) * z
    if case["type"] == "e4m3":
        b += 4 * (m + two * n)
    if case["bias"]:
        b += two * n * wide
    f = 2 * two * m * k * n
    if op == "gated":
        return {"bytes": b + m * n * wide, "flops": f}
    if op == "dense":
        b += m * n * SIZE[case["out"]]
        if case["residual"] != "none":
            b += m * n * SIZE[case["residual"]]
        return {"bytes": b, "flops": f}
    b += b + m * n * z  # the gradients have their inputs' sizes
    return {"bytes": b, "flops": f * (3 if op == "gated_backward" or case["act"] else 2)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _d(x, scale=None):
    if x is None:
        return None
    x = x.double()
    return x if scale is None else x * scale.double().unsqueeze(1)


def _sigma(z):
    """The logistic function without overflow."""
    return torch.where(z >= 0, 1 / (1 + torch.exp(-z.abs())),
                       torch.exp(-z.abs()) / (1 + torch.exp(-z.abs())))


def _f(z, act):
    """(act(z), act'(z)) in 64 bits. tanh t = 2 sigma(2t) - 1."""
    if act is None:
        return z, torch.ones_like(z)
    if act == "relu":
        on = z > 0
        return torch.where(on, z, torch.zeros_like(z)), on.double()
    if act == "tanh":
        t = 2 * _sigma(2 * z) - 1
        return t, (1 - t) * (1 + t)
    if act == "sigmoid":
        p = _sigma(z)
        return p, p * _sigma(-z)
    if act == "silu":
        p = _sigma(z)
        return z * p, p + z * p * _sigma(-z)
    a = 2 * math.sqrt(2 / math.pi)  # 0.5 (1 + tanh(v)) = sigma(2 v)
    p = _sigma(a * (z + 0.044715 * z ** 3))
    return z * p, p + z * p * (1 - p) * a * (1 + 0.134145 * z ** 2)


def _mm(a, b):
    return torch.einsum("ik,jk->ij", a, b)


def _plus(z, b):
    return z if b is None else z + b.double()


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        x, r = s["x"], s["residual_in"]
        t = x.double() if r is None else (x.double() + r.double()).to(r.dtype).double()
        y = s["weight"].double() * t / (t.pow(2).sum(1, keepdim=True) / t.shape[1] + EPS).sqrt()
        res = {"out": y}
        if r is not None:
            res["total"] = x.double() + r.double()
        if case["out"] == "e4m3":
            res["scale"] = y.abs().max(dim=1).values / E4M3_MAX
            res["out"] = y / res["scale"].unsqueeze(1)
        return res
    if op == "norm_backward":
        t, gy, w = _d(s["total"]), _d(s["grad"]), _d(s["weight"])
        n = t.shape[1]
        ms = t.pow(2).sum(1, keepdim=True) / n + EPS
        # d/dt_i sum_j gy_j w_j t_j ms^-1/2
        dot = (gy * w * t).sum(1, keepdim=True)
        gx = gy * w / ms.sqrt() - t * dot / (n * ms * ms.sqrt())
        if s["grad_total"] is not None:
            gx = gx + s["grad_total"].double()
        return {"x": gx, "weight": (gy * t / ms.sqrt()).sum(0)}
    if op.startswith("choice"):
        x = s["logits"].double()
        if s["mask_in"] is not None:
            x = x.masked_fill(s["mask_in"].bool().expand_as(x), -math.inf)
        at = s["targets"].long().unsqueeze(1)
        lse = torch.logsumexp(x, 1)
        some = lse > -math.inf
        logp = x - lse.masked_fill(~some, 0).unsqueeze(1)
        p = logp.exp()
        ent = -(p * logp.masked_fill(p == 0, 0)).sum(1)
        if op == "choice":
            res = {"logp": logp.gather(1, at).squeeze(1).masked_fill(~some, -math.inf),
                   "lse": lse, "entropy": ent}
            if case["top"]:
                v = torch.topk(logp, min(case["top"], x.shape[1]), dim=1).values
                res["top_logp"] = torch.cat([v, v.new_full(
                    (v.shape[0], case["top"] - v.shape[1]), -math.inf)], 1)
            return res
        gl, ge = s["grad_logp"].double(), s["grad_entropy"].double()
        d = -p * (gl.unsqueeze(1) + ge.unsqueeze(1) *
                  (logp.masked_fill(p == 0, 0) + ent.unsqueeze(1)))
        hit = (x.gather(1, at).squeeze(1) > -math.inf).double()
        d[torch.arange(d.shape[0], device=d.device), at.squeeze(1)] += gl * hit
        return {"logits": d}
    x = _d(s["x"], s["x_scale"])
    if op.startswith("gated"):
        wg, wu = _d(s["wg"], s["wg_scale"]), _d(s["wu"], s["wu_scale"])
        u = _plus(_mm(x, wu), s["bu"])
        a, da = _f(_plus(_mm(x, wg), s["bg"]), case["act"])
        if op == "gated":
            return {"out": a * u}
        dh = s["grad"].double()
        du, dg = dh * a, dh * u * da
        res = {"x": _mm(dg, wg.t()) + _mm(du, wu.t()), "wg": _mm(dg.t(), x.t()),
               "wu": _mm(du.t(), x.t())}
        if s["bg"] is not None:
            res["bg"], res["bu"] = dg.sum(0), du.sum(0)
        return res
    w = _d(s["w"], s["w_scale"])
    if op == "dense":
        z = _f(_plus(_mm(x, w), s["b"]), case["act"])[0]
        return {"out": _plus(z, s["residual_in"])}
    dz = s["grad"].double()
    if case["act"] is not None:
        dz = dz * _f(_plus(_mm(x, w), s["b"]), case["act"])[1]
    res = {"x": _mm(dz, w.t()), "w": _mm(dz.t(), x.t())}
    if s["b"] is not None:
        res["b"] = dz.sum(0)
    return res
