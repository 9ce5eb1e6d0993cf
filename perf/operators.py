"""Measured cases of the feed-forward operators: the matrix product with bias, activation and
residual in its epilogue (`linear`), the gated projection (`gated`), and the backward pass of each.

x [M, K] holds one token per row; weights are [N, K]; biases and their gradients are float32;
everything else has the case's type. `pad` adds that many unused elements to the rows of every
matrix (0: contiguous), so odd widths also come as odd row strides.

linear           p = x w^T + b, out = act(p) + residual           (p returned where `save` is set)
linear backward  dp = dout act'(p), dx = dp w, dw = dp^T x, db = sum over rows of dp
gated            a = x wa^T + ba, g = x wg^T + bg, out = act(a) g   (a, g returned where `save` is set)
gated backward   da = dout g act'(a), dg = dout act(a), dx = da wa + dg wg, dwa = da^T x,
                 dwg = dg^T x, dba and dbg the sums over rows of da and dg
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def _case(name, op, M, N, K, dtype="bf16", act="none", bias=True, residual=False, save=False, pad=0):
    return {"name": name, "op": op, "M": M, "N": N, "K": K, "dtype": dtype, "act": act, "bias": bias,
            "residual": residual, "save": save, "pad": pad}


def listed():
    return [
        # one option marker through the decision head's first layer: latency
        _case("linear token", "linear", 1, 768, 768, act="gelu"),
        # sixteen single tokens against a weight larger than the L2 cache: the weight's bytes count
        _case("linear weight stream", "linear", 16, 8192, 8192, residual=True),
        # odd sizes, contiguous (so odd row strides), stored for the backward pass
        _case("linear odd fp16", "linear", 1003, 771, 1155, dtype="fp16", act="silu", residual=True, save=True),
        # the encoder's down projection with its residual, one micro-batch of 16 rows of 512 tokens
        _case("linear down 16x512", "linear", 8192, 768, 1152, residual=True),
        # a whole router-scale batch of 256 rows of 512 tokens, kept for training
        _case("linear up 256x512", "linear", 131072, 1152, 768, act="gelu", save=True),
        # gradients of a few rows
        _case("linear grad 4x512", "linear_backward", 2048, 768, 1152, act="gelu_tanh"),
        # gradients of 64 rows of 512 tokens, no activation (the down projection)
        _case("linear grad 64x512", "linear_backward", 32768, 768, 1152),
        # one token through the encoder's gated projection: latency
        _case("gated token", "gated", 1, 1152, 768, act="gelu", bias=False),
        # the encoder's gated projection over a micro-batch, as its forward runs it
        _case("gated 16x512", "gated", 8192, 1152, 768, act="gelu", bias=False),
        # a wide gated projection kept for training
        _case("gated wide fp16", "gated", 4096, 8192, 4096, dtype="fp16", act="silu", save=True),
        # odd sizes backwards, padded rows
        _case("gated grad odd", "gated_backward", 1111, 903, 515, act="gelu", pad=2),
        # gradients of the encoder's gated projection over 128 rows of 512 tokens
        _case("gated grad 128x512", "gated_backward", 65536, 1152, 768, act="gelu", bias=False),
    ]


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = max(_cost(c) for c in listed())

    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        op = rng.choice(("linear", "linear_backward", "gated", "gated_backward"))
        N, K = size(16, 8192), size(16, 8192)
        if rng.random() < 0.6:  # widths of models: multiples of 64
            N, K = max(64, N // 64 * 64), max(64, K // 64 * 64)
        forward = op in ("linear", "gated")
        c = {"op": op, "M": size(1, 131072), "N": N, "K": K, "dtype": rng.choice(("bf16", "bf16", "fp16")),
             "act": rng.choice(ACTS), "bias": rng.random() < 0.6, "residual": op == "linear" and rng.random() < 0.5,
             "save": forward and rng.random() < 0.4, "pad": rng.choice((0, 0, 0, 1, 8))}
        if _cost(c) <= most:
            return c


def _mat(rows, cols, c, g=None, std=1.0):
    """A [rows, cols] matrix of the case's type with `pad` unused elements behind each row."""
    t = torch.empty((rows, cols + c["pad"]), device="cuda", dtype=DTYPES[c["dtype"]])[:, :cols]
    if g is not None:
        t.copy_(torch.randn((rows, cols), device="cuda", generator=g).mul_(std))
    return t


def prepare(case, seed):
    c = case
    M, N, K = c["M"], c["N"], c["K"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    gated = c["op"].startswith("gated")
    s = {"c": c, "x": _mat(M, K, c, g)}
    for i in ("a", "g") if gated else ("",):
        s["w" + i] = _mat(N, K, c, g, K ** -0.5)
        s["b" + i] = torch.randn(N, device="cuda", generator=g).mul_(0.3) if c["bias"] else None
    if c["op"] in ("linear", "gated"):
        s["out"] = _mat(M, N, c)
        s["residual"] = _mat(M, N, c, g) if c["residual"] else None
        for i in ("a", "g") if gated else ("",):
            s["p" + i] = _mat(M, N, c) if c["save"] else None
    else:
        s["dout"] = _mat(M, N, c, g, 0.5)
        for i in ("a", "g") if gated else ("",):
            s["p" + i] = None
            if gated or c["act"] != "none":  # what the forward pass stored
                s["p" + i] = _mat(M, N, c)
                p = s["x"].float() @ s["w" + i].float().t()
                s["p" + i].copy_(p if s["b" + i] is None else p.add_(s["b" + i]))
            s["dw" + i] = _mat(N, K, c)
            s["db" + i] = torch.empty(N, device="cuda") if c["bias"] else None
        s["dx"] = _mat(M, K, c)
    return s


def _act(p, act):
    if act == "relu":
        return torch.where(p > 0, p, torch.zeros_like(p))
    if act == "gelu":
        return p * (0.5 * (1.0 + torch.erf(p * math.sqrt(0.5))))
    if act == "gelu_tanh":
        return p * (0.5 * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (p + 0.044715 * p * p * p))))
    if act == "silu":
        return p / (1.0 + torch.exp(-p))
    return p


def _slope(p, act):
    """act'(p)."""
    if act == "relu":
        return (p > 0).to(p.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(p * math.sqrt(0.5))) + p * torch.exp(-0.5 * p * p) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        k = math.sqrt(2.0 / math.pi)
        t = torch.tanh(k * (p + 0.044715 * p * p * p))
        return 0.5 * (1.0 + t) + 0.5 * p * (1.0 - t * t) * k * (1.0 + 3 * 0.044715 * p * p)
    if act == "silu":
        e = 1.0 / (1.0 + torch.exp(-p))
        return e * (1.0 + p * (1.0 - e))
    return torch.ones_like(p)


def _affine(x, w, b):
    p = x.float() @ w.float().t()
    return p if b is None else p + b


def _row_sum(d):
    return d.sum(0, dtype=torch.float64).float()


def _plain(s):
    c = s["c"]
    t = DTYPES[c["dtype"]]
    if c["op"] == "linear":
        p = _affine(s["x"], s["w"], s["b"])
        out = _act(p, c["act"])
        if s["residual"] is not None:
            out = out + s["residual"].float()
        return {"out": out.to(t), "p": p.to(t)} if c["save"] else {"out": out.to(t)}
    if c["op"] == "gated":
        a, g = _affine(s["x"], s["wa"], s["ba"]), _affine(s["x"], s["wg"], s["bg"])
        out = {"out": (_act(a, c["act"]) * g).to(t)}
        if c["save"]:
            out |= {"a": a.to(t), "g": g.to(t)}
        return out
    dout, x = s["dout"].float(), s["x"].float()
    if c["op"] == "linear_backward":
        dp = dout if c["act"] == "none" else dout * _slope(s["p"].float(), c["act"])
        got = {"dx": (dp @ s["w"].float()).to(t), "dw": (dp.t() @ x).to(t)}
        if c["bias"]:
            got["db"] = _row_sum(dp)
        return got
    a, g = s["pa"].float(), s["pg"].float()
    da, dg = dout * g * _slope(a, c["act"]), dout * _act(a, c["act"])
    got = {"dx": (da @ s["wa"].float() + dg @ s["wg"].float()).to(t), "dwa": (da.t() @ x).to(t), "dwg": (dg.t() @ x).to(t)}
    if c["bias"]:
        got |= {"dba": _row_sum(da), "dbg": _row_sum(dg)}
    return got


def _framework():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "julia1-rs_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import julia1
    return julia1


def _own(s):
    j1 = s.get("j1")
    if j1 is None:
        j1 = s["j1"] = _framework()
        s["act"] = {"none": j1.ACT_NONE, "relu": j1.ACT_RELU, "gelu": j1.ACT_GELU, "gelu_tanh": j1.ACT_GELU_TANH,
                    "silu": j1.ACT_SILU}[s["c"]["act"]]
    c, st = s["c"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "linear":
        j1.op_linear(s["x"], s["w"], s["out"], bias=s["b"], act=s["act"], residual=s["residual"], pre=s["p"], stream=st,
                     sync=False)
        return {"out": s["out"], "p": s["p"]} if c["save"] else {"out": s["out"]}
    if c["op"] == "gated":
        j1.op_gated(s["x"], s["wa"], s["wg"], s["out"], ba=s["ba"], bg=s["bg"], act=s["act"], pre_a=s["pa"], pre_g=s["pg"],
                    stream=st, sync=False)
        return {"out": s["out"], "a": s["pa"], "g": s["pg"]} if c["save"] else {"out": s["out"]}
    if "ws" not in s:  # the scratch that a program keeps for its sizes
        size = j1.op_linear_backward_workspace if c["op"] == "linear_backward" else j1.op_gated_backward_workspace
        s["ws"] = torch.empty(size(c["M"], c["N"], c["K"]), device="cuda", dtype=torch.uint8)
    if c["op"] == "linear_backward":
        j1.op_linear_backward(s["dout"], s["x"], s["w"], pre=s["p"], act=s["act"], dx=s["dx"], dw=s["dw"], dbias=s["db"],
                              workspace=s["ws"], stream=st, sync=False)
        return {"dx": s["dx"], "dw": s["dw"], "db": s["db"]} if c["bias"] else {"dx": s["dx"], "dw": s["dw"]}
    j1.op_gated_backward(s["dout"], s["x"], s["wa"], s["wg"], s["pa"], s["pg"], act=s["act"], dx=s["dx"], dwa=s["dwa"],
                         dwg=s["dwg"], dba=s["dba"], dbg=s["dbg"], workspace=s["ws"], stream=st, sync=False)
    got = {"dx": s["dx"], "dwa": s["dwa"], "dwg": s["dwg"]}
    return got | {"dba": s["dba"], "dbg": s["dbg"]} if c["bias"] else got


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    c = case
    M, N, K = c["M"], c["N"], c["K"]
    n = 2 if c["op"].startswith("gated") else 1  # projections
    bias = 4 * n * N if c["bias"] else 0
    if c["op"] in ("linear", "gated"):
        elements = M * K + n * N * K + M * N * (1 + int(c["residual"]) + n * int(c["save"]))
        return {"bytes": 2 * elements + bias, "flops": 2 * n * M * N * K}
    saved = n if n == 2 or c["act"] != "none" else 0
    return {"bytes": 2 * (M * N * (1 + saved) + 2 * M * K + 2 * n * N * K) + bias, "flops": 4 * n * M * N * K}


def exact(case, seed):
    """The definitions in float64, the gradients by differentiating them."""
    c, s = case, prepare(case, seed)
    f = {"none": lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu,
         "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh"),
         "silu": torch.nn.functional.silu}[c["act"]]
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and k not in ("out", "dx", "dw", "dwa", "dwg")}
    names = ("a", "g") if c["op"].startswith("gated") else ("",)
    if c["op"] in ("linear", "gated"):
        p = []
        for i in names:
            p.append(torch.einsum("mk,nk->mn", d["x"], d["w" + i]))
            if c["bias"]:
                p[-1] += d["b" + i]
        out = f(p[0]) * p[1] if c["op"] == "gated" else f(p[0])
        if c["residual"]:
            out = out + d["residual"]
        got = {"out": out}
        if c["save"]:
            got |= dict(zip(("a", "g") if c["op"] == "gated" else ("p",), p))
        return got
    p = [d["p" + i].requires_grad_() if "p" + i in d else torch.zeros_like(d["dout"]).requires_grad_() for i in names]
    out = f(p[0]) * p[1] if c["op"] == "gated_backward" else f(p[0])
    grads = torch.autograd.grad(out, p, d["dout"])
    got = {"dx": sum(torch.einsum("mn,nk->mk", q, d["w" + i]) for q, i in zip(grads, names))}
    for q, i in zip(grads, names):
        got["dw" + i] = torch.einsum("mn,mk->nk", q, d["x"])
        if c["bias"]:
            got["db" + i] = q.sum(0)
    return got
