"""The feed-forward operators against their definitions in float64.

Tolerances are derived, per element, from what the kernels round:
* a result of type T is rounded once: eps(T) / 2 of its value (and half of fp16's smallest
  step, 2^-25, where a value is subnormal);
* a contraction in FP32 of n terms is off by at most (n + 2) 2^-23 of the sum of the terms'
  magnitudes (2^-23, not 2^-24: tensor cores may cut instead of rounding);
* an activation is off by at most ACT_ERR |p| and has slope at most 1.13, so it passes 1.13 of
  its argument's error on; a slope is off by at most SLOPE_ERR (both follow from the errors of
  one exponential, one reciprocal and, for the erf form, 1.5e-7 of its approximation);
* backward, the gradients at the pre-activations are rounded to T before the two products.
"""
import math

import pytest
import torch

import julia1 as j1

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
ACTS = {"none": j1.ACT_NONE, "relu": j1.ACT_RELU, "gelu": j1.ACT_GELU, "gelu_tanh": j1.ACT_GELU_TANH, "silu": j1.ACT_SILU}
ACT_ERR, SLOPE_ERR, LIP = 2e-6, 5e-6, 1.13


def act64(p, act):
    f = torch.nn.functional
    return {"none": lambda v: v, "relu": torch.relu, "gelu": f.gelu, "gelu_tanh": lambda v: f.gelu(v, approximate="tanh"),
            "silu": f.silu}[act](p)


def slope64(p, act):
    q = p.detach().clone().requires_grad_()
    return torch.autograd.grad(act64(q, act).sum(), q)[0] if act != "none" else torch.ones_like(p)


def unit(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return 2.0 ** -25 if t == HF else 0.0


def acc_err(n):
    return (n + 2) * 2.0 ** -23


def mat(rows, cols, dtype, gen=None, std=1.0, pad=0, fill=float("nan")):
    """A [rows, cols] view of rows that are `pad` longer; what is behind a row holds `fill`."""
    t = torch.full((rows, cols + pad), fill, device="cuda", dtype=dtype)
    v = t[:, :cols]
    if gen is not None:
        v.copy_(torch.randn((rows, cols), generator=gen, device="cuda") * std)
    return v


def pad_untouched(v, fill=float("nan")):
    """Nothing was written behind the rows of v (a view of mat())."""
    base = v._base
    if base is not None and base.dim() == 1:  # a matrix somewhere in a buffer: what lies before it
        return bool(base[:v.storage_offset()].isnan().all())
    if base is None or base.shape[1] == v.shape[1]:
        return True
    rest = base[:, v.shape[1]:].float()
    return bool((rest.isnan() if math.isnan(fill) else rest == fill).all())


def close(name, got, ref, tol):
    assert got.shape == ref.shape
    off = (got.double() - ref).abs()
    ok = off <= tol
    assert bool(ok.all()), "%s: %d of %d outside, worst %.3g of its tolerance, |off| %.3g" % (
        name, int((~ok).sum()), ok.numel(), float((off / tol.clamp_min(1e-300)).max()), float(off.max()))


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def affine64(x, w, b):
    x, w = x.double(), w.double()
    p, mag = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        p, mag = p + b.double(), mag + b.double().abs()
    return p, acc_err(x.shape[1]) * mag


def check_linear(M, N, K, dtype, act, bias, residual, save, pad=0, seed=0, inplace=False):
    g = gen(seed)
    x, w = mat(M, K, dtype, g, 1.0, pad), mat(N, K, dtype, g, K ** -0.5, pad)
    b = torch.randn(N, generator=g, device="cuda") * 0.5 if bias else None
    r = mat(M, N, dtype, g, 1.0, pad) if residual else None
    r64 = r.double() if residual else 0.0
    out = r if inplace else mat(M, N, dtype, pad=pad)
    pre = mat(M, N, dtype, pad=pad) if save else None
    j1.op_linear(x, w, out, bias=b, act=ACTS[act], residual=r, pre=pre)
    p, ep = affine64(x, w, b)
    ref = act64(p, act) + r64
    e = LIP * ep + (ACT_ERR * p.abs() if act not in ("none", "relu") else 0.0)
    close("out", out, ref, unit(dtype) * (ref.abs() + e) + e + 2.0 ** -23 * ref.abs() + tiny(dtype) + 1e-30)
    if save:
        close("pre", pre, p, unit(dtype) * (p.abs() + ep) + ep + tiny(dtype) + 1e-30)
    assert pad_untouched(out) and (pre is None or pad_untouched(pre))


def check_gated(M, N, K, dtype, act, bias, save, pad=0, seed=0):
    g = gen(seed)
    x = mat(M, K, dtype, g, 1.0, pad)
    wa, wg = mat(N, K, dtype, g, K ** -0.5, pad), mat(N, K, dtype, g, K ** -0.5, pad)
    ba, bg = (torch.randn(N, generator=g, device="cuda") * 0.5 for _ in range(2)) if bias else (None, None)
    out = mat(M, N, dtype, pad=pad)
    pa, pg = (mat(M, N, dtype, pad=pad) for _ in range(2)) if save else (None, None)
    j1.op_gated(x, wa, wg, out, ba=ba, bg=bg, act=ACTS[act], pre_a=pa, pre_g=pg)
    a, ea = affine64(x, wa, ba)
    q, eq = affine64(x, wg, bg)
    f = act64(a, act)
    ref = f * q
    e = q.abs() * (LIP * ea + ACT_ERR * a.abs()) + f.abs() * eq + 2.0 ** -23 * ref.abs() + eq * LIP * ea
    close("out", out, ref, unit(dtype) * (ref.abs() + e) + e + tiny(dtype) + 1e-30)
    if save:
        close("pre_a", pa, a, unit(dtype) * (a.abs() + ea) + ea + tiny(dtype) + 1e-30)
        close("pre_g", pg, q, unit(dtype) * (q.abs() + eq) + eq + tiny(dtype) + 1e-30)
    assert pad_untouched(out)
    assert not save or (pad_untouched(pa) and pad_untouched(pg))


def scratch(n):
    return torch.full((max(n, 1),), 255, device="cuda", dtype=torch.uint8)  # NaN in every type


def check_grads(dtype, x, ds, es, ws, dx, dws, dbs):
    """dx = sum ds ws, dws = ds^T x, dbs = sum of rows of ds, where the computed ds (before their
    rounding to dtype) are off by at most es."""
    u, t = unit(dtype), tiny(dtype)
    x = x.double()
    rounded = [u * (d.abs() + e) + e + t for d, e in zip(ds, es)]
    if dx is not None:
        ref = sum(d @ w.double() for d, w in zip(ds, ws))
        mag = sum((d.abs() + r) @ w.double().abs() for d, r, w in zip(ds, rounded, ws))
        e = sum(r @ w.double().abs() for r, w in zip(rounded, ws)) + acc_err(len(ds) * ds[0].shape[1]) * mag
        close("dx", dx, ref, u * (ref.abs() + e) + e + t + 1e-30)
        assert pad_untouched(dx)
    for i, dw in enumerate(dws):
        if dw is None:
            continue
        ref = ds[i].t() @ x
        e = rounded[i].t() @ x.abs() + acc_err(x.shape[0]) * ((ds[i].abs() + rounded[i]).t() @ x.abs())
        close("dw%d" % i, dw, ref, u * (ref.abs() + e) + e + t + 1e-30)
        assert pad_untouched(dw)
    for i, db in enumerate(dbs):
        if db is None:
            continue
        e = es[i].sum(0) + acc_err(x.shape[0]) * (ds[i].abs() + es[i]).sum(0)
        close("db%d" % i, db, ds[i].sum(0), e + 1e-30)


def check_linear_backward(M, N, K, dtype, act, pad=0, seed=0, want="dx dw db"):
    g = gen(seed)
    x, w, dout = mat(M, K, dtype, g, 1.0, pad), mat(N, K, dtype, g, K ** -0.5, pad), mat(M, N, dtype, g, 0.5, pad)
    pre = mat(M, N, dtype, g, 1.5, pad) if act != "none" else None
    dx = mat(M, K, dtype, pad=pad) if "dx" in want else None
    dw = mat(N, K, dtype, pad=pad) if "dw" in want else None
    db = torch.full((N,), float("nan"), device="cuda") if "db" in want else None
    j1.op_linear_backward(dout, x, w, pre=pre, act=ACTS[act], dx=dx, dw=dw, dbias=db,
                          workspace=scratch(j1.op_linear_backward_workspace(M, N, K)))
    d = dout.double()
    if act == "none":
        dp, e = d, torch.zeros_like(d)
    else:
        dp = d * slope64(pre.double(), act)
        e = d.abs() * SLOPE_ERR + 2.0 ** -23 * dp.abs()
    check_grads(dtype, x, [dp], [e], [w], dx, [dw], [db])


def check_gated_backward(M, N, K, dtype, act, pad=0, seed=0, want="dx dw db"):
    g = gen(seed)
    x, dout = mat(M, K, dtype, g, 1.0, pad), mat(M, N, dtype, g, 0.5, pad)
    wa, wg = mat(N, K, dtype, g, K ** -0.5, pad), mat(N, K, dtype, g, K ** -0.5, pad)
    pa, pg = mat(M, N, dtype, g, 1.5, pad), mat(M, N, dtype, g, 1.0, pad)
    dx = mat(M, K, dtype, pad=pad) if "dx" in want else None
    dwa, dwg = (mat(N, K, dtype, pad=pad) for _ in range(2)) if "dw" in want else (None, None)
    dba, dbg = (torch.full((N,), float("nan"), device="cuda") for _ in range(2)) if "db" in want else (None, None)
    j1.op_gated_backward(dout, x, wa, wg, pa, pg, act=ACTS[act], dx=dx, dwa=dwa, dwg=dwg, dba=dba, dbg=dbg,
                         workspace=scratch(j1.op_gated_backward_workspace(M, N, K)))
    d, a, q = dout.double(), pa.double(), pg.double()
    da, dg = d * q * slope64(a, act), d * act64(a, act)
    ea = (d * q).abs() * SLOPE_ERR + 2.0 ** -22 * da.abs()
    eg = d.abs() * ACT_ERR * a.abs() + 2.0 ** -22 * dg.abs()
    check_grads(dtype, x, [da, dg], [ea, eg], [wa, wg], dx, [dwa, dwg], [dba, dbg])


# one row to several tiles; widths around the tile sizes (64, 128, 256) and 16-byte rows; odd widths
SIZES = [(1, 1, 1), (1, 8, 16), (2, 3, 5), (5, 64, 64), (16, 1152, 768), (17, 200, 136), (33, 65, 96), (64, 127, 72),
         (100, 129, 257), (128, 128, 128), (129, 256, 64), (200, 264, 328), (255, 768, 768), (256, 31, 33),
         (300, 1155, 771), (513, 130, 1000), (1000, 1152, 768), (2048, 96, 40)]
TYPES = [(BF, "gelu"), (HF, "silu"), (BF, "none"), (HF, "gelu_tanh"), (BF, "relu")]


def _id(v):
    return str(v).replace("torch.", "")


@pytest.mark.parametrize("i,size", list(enumerate(SIZES)), ids=[_id(s) for s in SIZES])
def test_linear(torch_cuda, i, size):
    for j, (dtype, act) in enumerate(TYPES):
        check_linear(*size, dtype, act, bias=(i + j) % 3 > 0, residual=(i + j) % 2 > 0, save=j % 2 == 0, seed=i)


@pytest.mark.parametrize("i,size", list(enumerate(SIZES)), ids=[_id(s) for s in SIZES])
def test_gated(torch_cuda, i, size):
    for j, (dtype, act) in enumerate(TYPES):
        check_gated(*size, dtype, act, bias=(i + j) % 3 > 0, save=j % 2 == 0, seed=i)


@pytest.mark.parametrize("i,size", list(enumerate(SIZES)), ids=[_id(s) for s in SIZES])
def test_linear_backward(torch_cuda, i, size):
    for j, (dtype, act) in enumerate(TYPES):
        check_linear_backward(*size, dtype, act, seed=i)


@pytest.mark.parametrize("i,size", list(enumerate(SIZES)), ids=[_id(s) for s in SIZES])
def test_gated_backward(torch_cuda, i, size):
    for j, (dtype, act) in enumerate(TYPES):
        check_gated_backward(*size, dtype, act, seed=i)


@pytest.mark.parametrize("pad", [1, 2, 4, 8, 56])
def test_padded_rows(torch_cuda, pad):
    """Rows longer than the matrix, with NaN behind them: not read, not written."""
    for size in ((40, 72, 136), (300, 100, 70), (3, 264, 200)):
        check_linear(*size, BF, "gelu", True, True, True, pad=pad)
        check_gated(*size, HF, "silu", True, True, pad=pad)
        check_linear_backward(*size, BF, "gelu", pad=pad)
        check_gated_backward(*size, BF, "silu", pad=pad)


def test_residual_in_place(torch_cuda):
    for size in ((1, 768, 64), (300, 771, 64), (1000, 768, 128)):
        check_linear(*size, BF, "gelu", True, True, False, inplace=True)
        check_linear(*size, HF, "none", False, True, True, pad=8, inplace=True)


@pytest.mark.parametrize("want", ["dx", "dw", "db", "dx dw", "dw db"])
def test_some_gradients_only(torch_cuda, want):
    for act in ("none", "silu"):
        check_linear_backward(150, 136, 72, BF, act, want=want)
        check_gated_backward(150, 136, 72, BF, act, want=want)


def test_long_contractions(torch_cuda):
    """Few results over many terms: a long K forward, many rows in the weight gradients."""
    check_linear(8, 40, 20000, BF, "none", True, False, False)
    check_linear(130, 70, 9999, HF, "gelu", True, False, False)
    check_linear_backward(40000, 64, 48, BF, "gelu")
    check_gated_backward(30011, 72, 56, BF, "gelu")
    check_gated_backward(9000, 33, 45, HF, "silu")


def test_halves_of_one_buffer(torch_cuda):
    """Weights as the two halves of one Wi, the stored pre-activations side by side in one buffer."""
    M, N, K = 200, 96, 64
    g = gen(3)
    x, wi = mat(M, K, BF, g), mat(2 * N, K, BF, g, K ** -0.5)
    pre, out = torch.empty((M, 2 * N), device="cuda", dtype=BF), torch.empty((M, N), device="cuda", dtype=BF)
    j1.op_gated(x, wi[:N], wi[N:], out, act=j1.ACT_GELU, pre_a=pre[:, :N], pre_g=pre[:, N:])
    ref, e = affine64(x, wi, None)
    close("pre", pre, ref, unit(BF) * (ref.abs() + e) + e)
    dwi, dx = torch.empty_like(wi), torch.empty_like(x)
    j1.op_gated_backward(out, x, wi[:N], wi[N:], pre[:, :N], pre[:, N:], act=j1.ACT_GELU, dx=dx, dwa=dwi[:N],
                         dwg=dwi[N:], workspace=scratch(j1.op_gated_backward_workspace(M, N, K)))
    two = [torch.empty((N, K), device="cuda", dtype=BF) for _ in range(2)]
    j1.op_gated_backward(out, x, wi[:N].clone(), wi[N:].clone(), pre[:, :N].clone(), pre[:, N:].clone(),
                         act=j1.ACT_GELU, dwa=two[0], dwg=two[1],
                         workspace=scratch(j1.op_gated_backward_workspace(M, N, K)))
    assert torch.equal(dwi, torch.cat(two))


def test_no_rows(torch_cuda):
    x, w = torch.empty((0, 24), device="cuda", dtype=BF), torch.ones((40, 24), device="cuda", dtype=BF)
    out = torch.empty((0, 40), device="cuda", dtype=BF)
    j1.op_linear(x, w, out)
    j1.op_gated(x, w, w, out)
    dw = [mat(40, 24, BF, pad=3) for _ in range(2)]
    db = [torch.full((40,), float("nan"), device="cuda") for _ in range(2)]
    j1.op_linear_backward(out, x, w, act=j1.ACT_NONE, dw=dw[0], dbias=db[0], workspace=scratch(
        j1.op_linear_backward_workspace(0, 40, 24)))
    assert bool((dw[0] == 0).all()) and bool((db[0] == 0).all()) and pad_untouched(dw[0])
    dw[0].fill_(1.0)
    j1.op_gated_backward(out, x, w, w, out, out, dwa=dw[0], dwg=dw[1], dba=db[0], dbg=db[1], workspace=scratch(
        j1.op_gated_backward_workspace(0, 40, 24)))
    assert all(bool((t == 0).all()) for t in dw + db)


@pytest.mark.parametrize("act", ACTS)
def test_extreme_values(torch_cuda, act):
    """Large finite pre-activations give finite results and gradients (0 or the value itself on the
    far sides), a NaN stays in its own row forward, an infinity keeps its sign."""
    K, N = 16, 24
    vals = torch.tensor([-3e38, -1e30, -1e4, -60.0, -40.0, -6.0, 0.0, 6.0, 40.0, 60.0, 1e4, 1e30, 3e38, -0.0, 1e-30, -1e-30],
                        device="cuda")
    M = vals.numel()
    x, w = torch.zeros((M, K), device="cuda", dtype=BF), torch.zeros((N, K), device="cuda", dtype=BF)
    x[:, 0], w[:, 0] = vals, 1.0
    p = x[:, :1].double().expand(M, N)
    out, pre = torch.empty((M, N), device="cuda", dtype=BF), torch.empty((M, N), device="cuda", dtype=BF)
    j1.op_linear(x, w, out, act=ACTS[act], pre=pre)
    ref = act64(p, act)
    assert torch.equal(pre, x[:, :1].expand(M, N))
    # far negative values: within 2e-6 * 40 of 0, see ACT_ERR
    close("out", out, ref, unit(BF) * ref.abs() * 1.01 + ACT_ERR * p.abs().clamp_max(40.0))
    dout = torch.ones((M, N), device="cuda", dtype=BF)
    db = torch.empty(N, device="cuda")
    dx = torch.empty_like(x)
    j1.op_linear_backward(dout, x, w, pre=pre, act=ACTS[act], dx=dx, dbias=db,
                          workspace=scratch(j1.op_linear_backward_workspace(M, N, K)))
    s = slope64(p.clamp(-100, 100), act)
    close("dx", dx[:, :1], N * s[:, :1], N * (SLOPE_ERR + 2 * unit(BF) * s[:, :1].abs()))
    close("db", db, s.sum(0), torch.full_like(db, M * 2 * SLOPE_ERR).double())
    x[3, 0] = float("nan")
    x[5, 0] = float("inf")
    j1.op_linear(x, w, out, act=ACTS[act])
    assert bool(out[3].isnan().all()) and bool((out[5] == float("inf")).all())
    assert not bool(out[torch.arange(M, device="cuda") != 3].isnan().any())


def test_offsets_past_32_bits(torch_cuda):
    """Rows far apart: element offsets above 2^32 in every matrix of M rows."""
    M, N, K, far = 70000, 24, 40, 65536  # 70000 x 65536 = 4.6e9 elements, 9.2 GB
    g = gen(5)
    big = torch.zeros((M, far), device="cuda", dtype=BF)
    x, out, r, pre = big[:, 0:K], big[:, 64:64 + N], big[:, 128:128 + N], big[:, 256:256 + N]
    x.copy_(torch.randn((M, K), generator=g, device="cuda"))
    r.copy_(torch.randn((M, N), generator=g, device="cuda"))
    w = mat(N, K, BF, g, K ** -0.5)
    j1.op_linear(x, w, out, act=j1.ACT_GELU, residual=r, pre=pre)
    small = [torch.empty((M, N), device="cuda", dtype=BF) for _ in range(2)]
    j1.op_linear(x.contiguous(), w, small[0], act=j1.ACT_GELU, residual=r.contiguous(), pre=small[1])
    assert torch.equal(out, small[0]) and torch.equal(pre, small[1])
    p, e = affine64(x[-1000:], w, None)
    close("pre", pre[-1000:], p, unit(BF) * (p.abs() + e) + e)
    dx = big[:, 512:512 + K]
    dw = [torch.empty_like(w) for _ in range(2)]
    ws = scratch(j1.op_linear_backward_workspace(M, N, K))
    j1.op_linear_backward(out, x, w, pre=pre, act=j1.ACT_GELU, dx=dx, dw=dw[0], workspace=ws)
    dxs = torch.empty((M, K), device="cuda", dtype=BF)
    j1.op_linear_backward(small[0], x.contiguous(), w, pre=small[1], act=j1.ACT_GELU, dx=dxs, dw=dw[1], workspace=ws)
    assert torch.equal(dx, dxs) and torch.equal(dw[0], dw[1])


def _block(M, N, K, dtype, seed):
    """Buffers of a feed-forward block: y = x + (gelu(x wa^T) (x wg^T)) wo^T + bo."""
    g = gen(seed)
    e = lambda *s: torch.empty(s, device="cuda", dtype=dtype)  # noqa: E731
    return dict(M=M, N=N, K=K, x=mat(M, K, dtype, g), wa=mat(N, K, dtype, g, K ** -0.5), wg=mat(N, K, dtype, g, K ** -0.5),
                wo=mat(K, N, dtype, g, N ** -0.5), bo=torch.randn(K, generator=g, device="cuda") * 0.3,
                h=e(M, N), pa=e(M, N), pg=e(M, N), y=e(M, K), dy=mat(M, K, dtype, g), dh=e(M, N), dx=e(M, K),
                dwa=e(N, K), dwg=e(N, K), dwo=e(K, N), dbo=torch.empty(K, device="cuda"),
                ws=scratch(max(j1.op_gated_backward_workspace(M, N, K), j1.op_linear_backward_workspace(M, K, N))))


def _step(b, stream=None, sync=False):
    o = dict(stream=stream, sync=sync)
    j1.op_gated(b["x"], b["wa"], b["wg"], b["h"], act=j1.ACT_GELU, pre_a=b["pa"], pre_g=b["pg"], **o)
    j1.op_linear(b["h"], b["wo"], b["y"], bias=b["bo"], residual=b["x"], **o)
    j1.op_linear_backward(b["dy"], b["h"], b["wo"], dx=b["dh"], dw=b["dwo"], dbias=b["dbo"], workspace=b["ws"], **o)
    j1.op_gated_backward(b["dh"], b["x"], b["wa"], b["wg"], b["pa"], b["pg"], act=j1.ACT_GELU, dx=b["dx"], dwa=b["dwa"],
                         dwg=b["dwg"], workspace=b["ws"], **o)


RESULTS = ("h", "pa", "pg", "y", "dh", "dx", "dwa", "dwg", "dwo", "dbo")


@pytest.mark.parametrize("M,N,K,dtype", [(1, 1152, 768, BF), (513, 1152, 768, BF), (300, 200, 136, HF), (77, 65, 51, BF)])
def test_feed_forward_block(torch_cuda, M, N, K, dtype):
    """The operators in a row against float64 autograd of the whole block. Each step's inputs are
    rounded to the type: a handful of roundings of eps / 2 stack up, relative to the result's norm."""
    b = _block(M, N, K, dtype, 7)
    _step(b, sync=True)
    d = {k: b[k].double().requires_grad_() for k in ("x", "wa", "wg", "wo", "bo")}
    h = act64(d["x"] @ d["wa"].t(), "gelu") * (d["x"] @ d["wg"].t())
    y = d["x"] + h @ d["wo"].t() + d["bo"]
    grads = dict(zip(d, torch.autograd.grad(y, list(d.values()), b["dy"].double())))
    refs = {"h": h, "y": y, "dx": grads["x"] - b["dy"].double(), "dwa": grads["wa"], "dwg": grads["wg"],
            "dwo": grads["wo"], "dbo": grads["bo"]}
    for k, ref in refs.items():
        # at most six roundings precede any result (pre, h or dh, da / dg, the result, and FP32 sums)
        off = (b[k].double() - ref).norm() / ref.norm()
        assert off <= 6 * unit(dtype), (k, float(off))


def test_gradients_against_differences(torch_cuda):
    """The gradients against central differences of the float64 definition along random directions:
    independent of any formula for the slopes."""
    M, N, K = 9, 12, 10
    for act in ("gelu", "gelu_tanh", "silu"):
        b = _block(M, N, K, HF, 11)
        j1.op_gated(b["x"], b["wa"], b["wg"], b["h"], act=ACTS[act], pre_a=b["pa"], pre_g=b["pg"])
        b["dh"].copy_(torch.randn((M, N), generator=gen(1), device="cuda"))
        j1.op_gated_backward(b["dh"], b["x"], b["wa"], b["wg"], b["pa"], b["pg"], act=ACTS[act], dx=b["dx"], dwa=b["dwa"],
                             dwg=b["dwg"], workspace=b["ws"])

        def value(x, wa, wg):
            return float((act64(x @ wa.t(), act) * (x @ wg.t()) * b["dh"].double()).sum())

        at = [b[k].double() for k in ("x", "wa", "wg")]
        for i, k in enumerate(("dx", "dwa", "dwg")):
            v = torch.randn(at[i].shape, generator=gen(20 + i), device="cuda", dtype=torch.float64)
            step = 1e-5
            up, dn = list(at), list(at)
            up[i], dn[i] = at[i] + step * v, at[i] - step * v
            num = (value(*up) - value(*dn)) / (2 * step)
            got = float((b[k].double() * v).sum())
            # the roundings of pre, da / dg and the result, each eps / 2 of terms that sum up in magnitude
            scale = float((b[k].double().abs() * v.abs()).sum())
            assert abs(got - num) <= 8 * unit(HF) * scale + 1e-6, (act, k, got, num)


def test_same_bits_again(torch_cuda):
    for size in ((1, 768, 768), (2048, 1152, 768), (777, 333, 129)):
        b = _block(*size, BF, 13)
        _step(b, sync=True)
        first = {k: b[k].clone() for k in RESULTS}
        for _ in range(3):
            b["ws"].random_(0, 255)
            for k in RESULTS:
                b[k].fill_(float("nan"))
            _step(b, sync=True)
            for k in RESULTS:
                assert torch.equal(b[k], first[k]), k


def test_two_streams_at_once(torch_cuda):
    """Blocks with a workspace each on two streams, interleaved, give what they give alone."""
    blocks = [_block(1500, 768, 384, BF, 17), _block(700, 520, 264, HF, 19), _block(600, 333, 129, BF, 20)]
    refs = []
    for b in blocks:
        _step(b, sync=True)
        refs.append({k: b[k].clone() for k in RESULTS})
        for k in RESULTS:
            b[k].fill_(float("nan"))
    streams = [torch.cuda.Stream() for _ in blocks]
    torch.cuda.synchronize()
    for _ in range(5):
        for b, s in zip(blocks, streams):
            _step(b, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for b, ref in zip(blocks, refs):
        for k in RESULTS:
            assert torch.equal(b[k], ref[k]), k


@pytest.mark.parametrize("M,N,K", [(600, 384, 256), (333, 259, 131), (5, 200, 96)])
def test_captured_and_replayed(torch_cuda, M, N, K):
    """A whole step in a CUDA graph, replayed on new inputs in the same buffers; also where operands
    are copied to aligned rows first (odd widths)."""
    b = _block(M, N, K, BF, 23)
    _step(b, sync=True)
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        _step(b, stream=torch.cuda.current_stream().cuda_stream)
    for seed in (1, 2):
        g = gen(seed)
        for k in ("x", "dy"):
            b[k].copy_(torch.randn(b[k].shape, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = {k: b[k].clone() for k in RESULTS}
        _step(b, sync=True)
        for k in RESULTS:
            assert torch.equal(b[k], got[k]), k


def test_two_graphs_and_an_eager_call(torch_cuda):
    """Two captured steps with a workspace each, replayed at once on two streams while a third step runs
    eagerly, all with copied operands."""
    blocks = [_block(257, 131, 67, BF, 31), _block(300, 203, 77, HF, 32), _block(129, 99, 101, BF, 33)]
    refs = []
    for b in blocks:
        _step(b, sync=True)
        refs.append({k: b[k].clone() for k in RESULTS})
    graphs = []
    for b in blocks[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            _step(b, stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for b in blocks:
        for k in RESULTS:
            b[k].fill_(float("nan"))
    streams = [torch.cuda.Stream() for _ in blocks]
    torch.cuda.synchronize()
    for _ in range(4):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        _step(blocks[2], stream=streams[2].cuda_stream)
    torch.cuda.synchronize()
    for b, ref in zip(blocks, refs):
        for k in RESULTS:
            assert torch.equal(b[k], ref[k]), k


def test_unaligned_bases(torch_cuda):
    """Operands and results that start anywhere in a buffer, at its first and last elements too: the
    copies to aligned rows read nothing outside them."""
    for off, (M, N, K) in enumerate(((70, 40, 64), (33, 130, 72), (129, 65, 257), (1, 9, 300), (17, 8, 8), (64, 3, 5)), 1):
        g = gen(off)

        def at(rows, cols, std=1.0):
            buf = torch.full((rows * cols + off,), float("nan"), device="cuda", dtype=BF)
            v = buf[off:].view(rows, cols)
            v.copy_(torch.randn((rows, cols), generator=g, device="cuda") * std)
            return v

        x, w, r, out, dout = at(M, K), at(N, K, K ** -0.5), at(M, N), at(M, N), at(M, N)
        j1.op_linear(x, w, out, residual=r)
        p, e = affine64(x, w, None)
        ref = p + r.double()
        close("out", out, ref, unit(BF) * (ref.abs() + e) + e + 2.0 ** -23 * ref.abs())
        dx, dw = at(M, K), at(N, K)
        j1.op_linear_backward(dout, x, w, dx=dx, dw=dw, workspace=scratch(j1.op_linear_backward_workspace(M, N, K)))
        d = dout.double()
        check_grads(BF, x, [d], [torch.zeros_like(d)], [w], dx, [dw], [])


def test_copies_allocation_failure(torch_cuda):
    x, w, out = (torch.ones(s, device="cuda", dtype=BF) for s in ((4, 17), (8, 17), (4, 8)))
    j1.inject_fault(j1.FAULT_ALLOC, 1)
    try:
        with pytest.raises(j1.J1Error) as e:
            j1.op_linear(x, w, out)
    finally:
        j1.inject_fault(j1.FAULT_ALLOC, 0)
    assert e.value.status == j1.OOM
    j1.op_linear(x, w, out)
    assert bool((out == 17).all())
    j1.inject_fault(j1.FAULT_ALLOC, 1)  # nothing is allocated for aligned rows
    try:
        j1.op_linear(x[:, :16].contiguous(), w[:, :16].contiguous(), out)
    finally:
        j1.inject_fault(j1.FAULT_ALLOC, 0)
    assert bool((out == 16).all())


def test_refused_pointers(torch_cuda):
    x = torch.zeros((4, 16), dtype=BF)
    w, out = torch.zeros((8, 16), device="cuda", dtype=BF), torch.zeros((4, 8), device="cuda", dtype=BF)
    with pytest.raises(j1.J1Error) as e:
        j1.op_linear(x, w, out)
    assert e.value.status == j1.INVALID_ARG and "x is not device memory" in str(e.value)
    with pytest.raises(j1.J1Error) as e:
        j1.op_linear(x.pin_memory(), w, out)
    assert e.value.status == j1.INVALID_ARG and "x is not device memory" in str(e.value)
    j1.inject_fault(j1.FAULT_LAUNCH, 1)
    try:
        with pytest.raises(j1.J1Error) as e:
            j1.op_linear(x.cuda(), w, out)
    finally:
        j1.inject_fault(j1.FAULT_LAUNCH, 0)
    assert e.value.status == j1.CUDA
    j1.op_linear(x.cuda(), w, out)
    assert bool((out == 0).all())


def test_managed_memory_is_refused(torch_cuda):
    import ctypes as C
    torch.zeros(1, device="cuda")
    rt, p = C.CDLL("libcudart.so.12"), C.c_void_p()
    assert rt.cudaMallocManaged(C.byref(p), C.c_size_t(4096), C.c_uint(1)) == 0
    try:
        w, out = torch.zeros((8, 16), device="cuda", dtype=BF), torch.zeros((4, 8), device="cuda", dtype=BF)
        a = j1.J1LinearArgs(0, 0, 4, 8, 16, p, 16, w.data_ptr(), 16, None, None, 0, out.data_ptr(), 8, None, 0)
        assert j1.lib().j1_op_linear(a, None, 1) == j1.INVALID_ARG and "x is not device memory" in j1.last_error()
    finally:
        rt.cudaFree(p)


def test_many_shapes_at_once(torch_cuda):
    """Products of CTA pairs, of clusters that share a tile and of single CTAs, started together on a stream each,
    give what they give alone: none holds accumulators another waits for."""
    blocks = [_block(9500, 704, 512, BF, 41), _block(1, 768, 768, BF, 42), _block(40, 1152, 768, HF, 43),
              _block(300, 128, 640, BF, 44), _block(2048, 768, 192, HF, 45), _block(129, 64, 2048, BF, 46)]
    refs = []
    for b in blocks:
        _step(b, sync=True)
        refs.append({k: b[k].clone() for k in RESULTS})
    streams = [torch.cuda.Stream() for _ in blocks]
    torch.cuda.synchronize()
    for i in range(20):
        for j in range(len(blocks)):
            k = (i + j) % len(blocks)
            _step(blocks[k], stream=streams[k].cuda_stream)
    torch.cuda.synchronize()
    for b, ref in zip(blocks, refs):
        for k in RESULTS:
            assert torch.equal(b[k], ref[k]), k


@pytest.mark.parametrize("shared", [True, False])
def test_two_threads(torch_cuda, shared):
    """Steps from two host threads, on one stream (their kernels interleave) or one each: kernels of a backward pass
    that start before the one ahead has ended still follow what they read, whatever is queued between them."""
    import threading
    blocks = [_block(300, 768, 384, BF, 51), _block(200, 333, 129, HF, 52)]
    refs = []
    for b in blocks:
        _step(b, sync=True)
        refs.append({k: b[k].clone() for k in RESULTS})
        for k in RESULTS:
            b[k].fill_(float("nan"))
    one = torch.cuda.Stream()
    streams = [one, one if shared else torch.cuda.Stream()]
    errors = []
    torch.cuda.synchronize()

    def work(b, s):
        try:
            for _ in range(30):
                _step(b, stream=s.cuda_stream)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(blocks, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for b, ref in zip(blocks, refs):
        for k in RESULTS:
            assert torch.equal(b[k], ref[k]), k


# Sizes whose products take every tile shape, cluster size and stream-K plan on a GPU of 148 SMs.
PLANS = [("linear", (1, 32, 816)), ("linear", (100, 32, 816)), ("linear", (1, 880, 7464)), ("linear", (90, 880, 7464)),
         ("linear", (1, 2080, 2546)), ("linear", (33, 2080, 2546)), ("linear", (50, 32, 200)), ("linear", (300, 40, 72)),
         ("linear", (296, 3192, 336)), ("linear", (664, 3392, 392)), ("linear", (1479, 2472, 824)), ("linear", (5051, 69, 7661)),
         ("gated", (1, 32, 200)), ("gated", (70, 32, 200)), ("gated", (1, 32, 488)), ("gated", (120, 65, 488)),
         ("gated", (283, 3344, 728)), ("gated", (500, 700, 130)),
         ("linear_backward", (1, 65, 36)), ("linear_backward", (1, 198, 33)), ("linear_backward", (1, 824, 32)),
         ("linear_backward", (1, 2489, 2153)), ("linear_backward", (40, 1397, 4828)), ("linear_backward", (206, 33, 32)),
         ("linear_backward", (478, 34, 32)), ("linear_backward", (71, 32, 32)), ("linear_backward", (155, 326, 4840)),
         ("linear_backward", (1073, 402, 5106)), ("linear_backward", (1541, 986, 1431)), ("linear_backward", (2949, 32, 4868)),
         ("linear_backward", (6012, 32, 2272)), ("linear_backward", (7356, 160, 2552)),
         ("gated_backward", (1, 33, 38)), ("gated_backward", (1, 391, 32)), ("gated_backward", (1, 1128, 2120)),
         ("gated_backward", (2, 3807, 835)), ("gated_backward", (1, 1168, 7560)), ("gated_backward", (226, 32, 32)),
         ("gated_backward", (1035, 529, 2089)), ("gated_backward", (1309, 32, 2320)), ("gated_backward", (3338, 1070, 65)),
         ("gated_backward", (4729, 32, 5184)), ("gated_backward", (7109, 96, 2560))]


@pytest.mark.parametrize("i,op,size", [(i, op, s) for i, (op, s) in enumerate(PLANS)],
                         ids=["%s-%s" % (op, _id(s)) for op, s in PLANS])
def test_every_plan(torch_cuda, i, op, size):
    dtype, act = TYPES[i % len(TYPES)]
    if op == "linear":
        check_linear(*size, dtype, act, bias=True, residual=True, save=True, seed=i)
        check_linear(*size, dtype, act, bias=False, residual=False, save=False, seed=i)
    elif op == "gated":
        check_gated(*size, dtype, act, bias=True, save=True, seed=i)
        check_gated(*size, dtype, act, bias=False, save=False, seed=i)
    elif op == "linear_backward":
        check_linear_backward(*size, dtype, act, seed=i)
    else:
        check_gated_backward(*size, dtype, act, seed=i)


@pytest.mark.parametrize("pad", [0, 1, 8])
def test_pairs_store_nothing_behind_rows(torch_cuda, pad):
    """Tiles of CTA pairs over ragged rows and columns, stored as boxes where rows are whole 16-byte units (no padding, 8)
    and element-wise otherwise; the residual in place, the rows behind the last one left as they were."""
    for i, (dtype, act) in enumerate(TYPES[:3]):
        for M, N, K in ((1479, 2472, 824), (700, 3392, 392)):
            check_linear(M, N, K, dtype, act, bias=True, residual=True, save=True, pad=pad, seed=i, inplace=True)
        check_gated(283, 3344, 728, dtype, act, bias=True, save=True, pad=pad, seed=i)
    M, N, K = 1479, 2472, 824
    g = gen(9)
    x, w = mat(M, K, BF, g), mat(N, K, BF, g, K ** -0.5)
    out, pre = (torch.full((M + 33, N), float("nan"), device="cuda", dtype=BF) for _ in range(2))
    j1.op_linear(x, w, out[:M], act=j1.ACT_GELU, pre=pre[:M])
    assert bool(out[M:].isnan().all()) and bool(pre[M:].isnan().all())
    assert not bool(out[:M].isnan().any()) and not bool(pre[:M].isnan().any())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,N,K", [(1, 5, 2000), (1, 300, 257), (16, 250, 129), (64, 64, 64), (170, 23, 40), (1, 4096, 72)])
def test_few_gradients_in_two_parts(torch_cuda, dtype, M, N, K):
    """Up to 2^12 gradients at the pre-activations reach the products in two parts: what the second part is rounded by
    is a unit of a unit of the value (and a subnormal's half step), far below the result's own rounding."""
    g = gen(M + N)
    u, t = unit(dtype), tiny(dtype)
    x, dout = mat(M, K, dtype, g), mat(M, N, dtype, g, 0.5)
    ws = [mat(N, K, dtype, g, K ** -0.5) for _ in range(2)]
    pre = [mat(M, N, dtype, g, 1.5) for _ in range(2)]
    scr = scratch(j1.op_gated_backward_workspace(M, N, K))
    d, p, q = dout.double(), pre[0].double(), pre[1].double()

    def check(ds, es, weights, dx, dws):
        off = [u * u * (v.abs() + e) + e + t for v, e in zip(ds, es)]
        ref = sum(v @ w.double() for v, w in zip(ds, weights))
        mag = sum((v.abs() + o) @ w.double().abs() for v, o, w in zip(ds, off, weights))
        e = sum(o @ w.double().abs() for o, w in zip(off, weights)) + acc_err(2 * len(ds) * N) * mag
        close("dx", dx, ref, u * (ref.abs() + e) + e + t + 1e-30)
        for v, o, dw in zip(ds, off, dws):
            ref = v.t() @ x.double()
            e = o.t() @ x.double().abs() + acc_err(2 * M) * ((v.abs() + o).t() @ x.double().abs())
            close("dw", dw, ref, u * (ref.abs() + e) + e + t + 1e-30)

    dx, dw = mat(M, K, dtype), [mat(N, K, dtype) for _ in range(2)]
    j1.op_linear_backward(dout, x, ws[0], pre=pre[0], act=j1.ACT_GELU, dx=dx, dw=dw[0], workspace=scr)
    dp = d * slope64(p, "gelu")
    check([dp], [d.abs() * SLOPE_ERR + 2.0 ** -23 * dp.abs()], ws[:1], dx, dw[:1])
    j1.op_gated_backward(dout, x, ws[0], ws[1], pre[0], pre[1], act=j1.ACT_SILU, dx=dx, dwa=dw[0], dwg=dw[1], workspace=scr)
    da, dg = d * q * slope64(p, "silu"), d * act64(p, "silu")
    check([da, dg], [(d * q).abs() * SLOPE_ERR + 2.0 ** -22 * da.abs(), d.abs() * p.abs() * ACT_ERR + 2.0 ** -23 * dg.abs()],
          ws, dx, dw)


def check_in_parts(dtype, x, ds, es, weights, dx, dws, floor=0.0):
    """dx and dw where the gradients at the pre-activations (ds, computed within es) reach the products in two parts:
    the first cut to the type's bits, the second rounded to them, so within a unit of a unit of the value, and `floor`
    for what lies below the second part's range."""
    u, t, x = unit(dtype), tiny(dtype), x.double()
    off = [u * u * (v.abs() + e) + e + floor for v, e in zip(ds, es)]
    if dx is not None:
        ref = sum(v @ w.double() for v, w in zip(ds, weights))
        mag = sum((v.abs() + o) @ w.double().abs() for v, o, w in zip(ds, off, weights))
        e = sum(o @ w.double().abs() for o, w in zip(off, weights)) + acc_err(2 * len(ds) * ds[0].shape[1]) * mag
        close("dx", dx, ref, u * (ref.abs() + e) + e + t + 1e-30)
    for v, o, dw in zip(ds, off, dws):
        ref = v.t() @ x
        e = o.t() @ x.abs() + acc_err(2 * x.shape[0]) * ((v.abs() + o).t() @ x.abs())
        close("dw", dw, ref, u * (ref.abs() + e) + e + t + 1e-30)


def rounded_once(name, got, ref):
    """The errors of one rounding are uniform over a spacing s: squares of mean s^2 / 12 and variance s^4 / 180. All of
    them together stay within five standard deviations of their mean and 10% for what else is in 32 bits (a dozen
    roundings of 2^-24 per slope and sum: 1/200 of an FP16 unit); a second rounding of the terms doubles the mean."""
    s2 = (torch.finfo(got.dtype).eps * torch.exp2(ref.abs().clamp_min(float(torch.finfo(got.dtype).tiny)).log2().floor())) ** 2
    most = float(s2.sum() / 12 + 5 * (s2 * s2).sum().sqrt() / math.sqrt(180))
    off = float((got.double() - ref).norm())
    assert off <= 1.1 * math.sqrt(most), (name, off, math.sqrt(float(s2.sum()) / 12))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,N,K", [(1, 4104, 72), (64, 65, 300), (2, 8192, 64), (513, 130, 200), (2048, 768, 200), (4096, 64, 64),
                                   (777, 333, 129), (30000, 136, 72)])
def test_gradients_are_rounded_once_at_every_size(torch_cuda, dtype, M, N, K):
    """However many gradients at the pre-activations there are, their rounding stays far below the results' own."""
    g = gen(M + N)
    x, dout = mat(M, K, dtype, g), mat(M, N, dtype, g, 0.5)
    ws = [mat(N, K, dtype, g, K ** -0.5) for _ in range(2)]
    pre = [mat(M, N, dtype, g, 1.5) for _ in range(2)]
    scr = scratch(j1.op_gated_backward_workspace(M, N, K))
    d, p, q = dout.double(), pre[0].double(), pre[1].double()
    dx, dw = mat(M, K, dtype), [mat(N, K, dtype) for _ in range(2)]
    for act in ("gelu", "relu"):
        j1.op_linear_backward(dout, x, ws[0], pre=pre[0], act=ACTS[act], dx=dx, dw=dw[0], workspace=scr)
        dp = d * slope64(p, act)
        e = d.abs() * SLOPE_ERR + 2.0 ** -23 * dp.abs() if act == "gelu" else torch.zeros_like(d)
        check_in_parts(dtype, x, [dp], [e], ws[:1], dx, dw[:1], tiny(dtype) * 4)
        rounded_once("dx", dx, dp @ ws[0].double())
        rounded_once("dw", dw[0], dp.t() @ x.double())
    j1.op_gated_backward(dout, x, *ws, *pre, act=j1.ACT_SILU, dx=dx, dwa=dw[0], dwg=dw[1], workspace=scr)
    da, dg = d * q * slope64(p, "silu"), d * act64(p, "silu")
    check_in_parts(dtype, x, [da, dg], [(d * q).abs() * SLOPE_ERR + 2.0 ** -22 * da.abs(),
                                        d.abs() * p.abs() * ACT_ERR + 2.0 ** -23 * dg.abs()], ws, dx, dw, tiny(dtype) * 4)
    rounded_once("gated dx", dx, da @ ws[0].double() + dg @ ws[1].double())
    rounded_once("dwa", dw[0], da.t() @ x.double())
    rounded_once("dwg", dw[1], dg.t() @ x.double())


@pytest.mark.parametrize("M,N,K", [(4096, 40, 24), (3, 100, 65), (300, 264, 72)])
@pytest.mark.parametrize("size", [2.0 ** -14, 2.0 ** -22, 2.0 ** 13])
def test_fp16_gradients_keep_their_range(torch_cuda, M, N, K, size):
    """FP16 gradients at the pre-activations far below and above the type's range, whose results are in it: both parts
    are scaled by a power of two of the call, so only what is 2^-38 of the largest is lost."""
    g = gen(M + K)
    big = size > 1
    x = mat(M, K, HF, g, M ** -0.5 * 2.0 ** -12 if big else 8.0)
    ws = [mat(N, K, HF, g, N ** -0.5 * 2.0 ** -12 if big else 8.0) for _ in range(2)]
    dout = mat(M, N, HF, g, size)
    a = mat(M, N, HF, g, 1.5)
    if not big:
        a.sub_(4.0)  # slopes and values of the far side
    q = mat(M, N, HF, g, 16.0 if big else 0.01)
    scr = scratch(j1.op_gated_backward_workspace(M, N, K))
    dx, dw = mat(M, K, HF), [mat(N, K, HF) for _ in range(2)]
    db = [torch.empty(N, device="cuda") for _ in range(2)]
    d, p, r = dout.double(), a.double(), q.double()
    rel = 2.0 ** -18  # of a slope or value on the far side: its exponential's argument is rounded twice, |p| < 12

    def check(ds, es, weights, dws):
        floor = 2.0 ** -38 * max(float(v.abs().max()) for v in ds)
        check_in_parts(HF, x, ds, es, weights, dx, dws, floor)
        for v, e, b in zip(ds, es, db):
            close("db", b, v.sum(0), e.sum(0) + acc_err(M) * (v.abs() + e).sum(0))

    s = slope64(p, "silu")
    dp = d * s
    j1.op_linear_backward(dout, x, ws[0], pre=a, act=j1.ACT_SILU, dx=dx, dw=dw[0], dbias=db[0], workspace=scr)
    slope_err = rel * (s.abs() + torch.sigmoid(p))
    check([dp], [d.abs() * slope_err], ws[:1], dw[:1])
    assert bool((dw[0] != 0).any()) and not bool(dx.isinf().any())
    da, dg = d * r * s, d * act64(p, "silu")
    j1.op_gated_backward(dout, x, *ws, a, q, act=j1.ACT_SILU, dx=dx, dwa=dw[0], dwg=dw[1], dba=db[0], dbg=db[1], workspace=scr)
    check([da, dg], [(d * r).abs() * slope_err, rel * dg.abs()], ws, dw)


def test_fp16_gradients_of_zeros_and_infinities(torch_cuda):
    """The scale of a call whose gradients are all 0, or that holds infinities and NaN beside small ones."""
    M, N, K = 40, 24, 16
    g = gen(2)
    x, w, pre = mat(M, K, HF, g), mat(N, K, HF, g), mat(M, N, HF, g)
    dout, dx, dw = torch.zeros((M, N), device="cuda", dtype=HF), mat(M, K, HF), mat(N, K, HF)
    scr = scratch(j1.op_linear_backward_workspace(M, N, K))
    call = lambda: j1.op_linear_backward(dout, x, w, pre=pre, act=j1.ACT_GELU, dx=dx, dw=dw, workspace=scr)  # noqa: E731
    call()
    assert bool((dx == 0).all()) and bool((dw == 0).all())
    dout.copy_(torch.randn((M, N), generator=g, device="cuda") * 2.0 ** -12)
    call()
    ref = dx.clone()
    dout[7, 3], dout[9, 5], dout[11, 7] = float("inf"), float("nan"), -float("inf")
    call()
    assert bool(dx[9].isnan().all()) and bool(dx[[7, 11]].isinf().all())
    rest = [i for i in range(M) if i not in (7, 9, 11)]
    assert torch.equal(dx[rest], ref[rest])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("act,M,N,K", [("gelu", 4, 64, 40), ("silu", 30, 20, 33), ("relu", 1, 40, 264),
                                       ("gelu_tanh", 130, 100, 72)])
def test_infinite_operands_of_gradients(torch_cuda, dtype, act, M, N, K):
    """An infinite weight, input or output gradient gives the infinities of the definition, in its own column or row,
    and no NaN where that has none: both parts of a gradient at a pre-activation have its sign, and neither is 0."""
    g = gen(M + N)
    x, dout = mat(M, K, dtype, g), mat(M, N, dtype, g, 0.5)
    ws = [mat(N, K, dtype, g, K ** -0.5) for _ in range(2)]
    pre = [mat(M, N, dtype, g, 1.5) for _ in range(2)]
    inf = float("inf")
    ws[0][N // 2, 3], ws[1][N // 3, 5] = inf, -inf
    x[M // 2, 7], x[M // 3, 9] = -inf, inf
    d, p, q = dout.double(), pre[0].double(), pre[1].double()
    dx, dw = mat(M, K, dtype), [mat(N, K, dtype) for _ in range(2)]
    scr = scratch(j1.op_gated_backward_workspace(M, N, K))

    def same(name, got, ref):
        got = got.double()
        for what in (torch.isnan, torch.isposinf, torch.isneginf):
            assert torch.equal(what(got), what(ref)), (name, what.__name__, int((what(got) != what(ref)).sum()))

    for late in (False, True):
        if late:  # a gradient that is infinite itself, in finite weights and inputs
            for t in ws + [x]:
                t[t.isinf()] = 1.0
            dout[M - 1, 2], dout[M // 2, N - 1] = inf, -inf
            d = dout.double()
        dp = d * slope64(p, act)
        j1.op_linear_backward(dout, x, ws[0], pre=pre[0], act=ACTS[act], dx=dx, dw=dw[0], workspace=scr)
        same("linear dx", dx, (dp[:, :, None] * ws[0].double()).sum(1))
        same("linear dw", dw[0], (dp[:, :, None] * x.double()[:, None]).sum(0))
        da, dg = d * q * slope64(p, act), d * act64(p, act)
        j1.op_gated_backward(dout, x, *ws, *pre, act=ACTS[act], dx=dx, dwa=dw[0], dwg=dw[1], workspace=scr)
        same("gated dx", dx, (da[:, :, None] * ws[0].double() + dg[:, :, None] * ws[1].double()).sum(1))
        same("gated dwa", dw[0], (da[:, :, None] * x.double()[:, None]).sum(0))
        same("gated dwg", dw[1], (dg[:, :, None] * x.double()[:, None]).sum(0))


def test_tiny_bf16_gradients(torch_cuda):
    """Gradients at the pre-activations near the end of BF16's range keep both parts, down to its smallest step, 2^-133."""
    M, N, K = 40, 64, 48
    g = gen(6)
    x, w, pre = mat(M, K, BF, g, 2.0 ** 100), mat(N, K, BF, g, 2.0 ** 100), mat(M, N, BF, g, 1.5)
    dout, dx, dw = mat(M, N, BF, g, 2.0 ** -116), mat(M, K, BF), mat(N, K, BF)
    j1.op_linear_backward(dout, x, w, pre=pre, act=j1.ACT_SILU, dx=dx, dw=dw,
                          workspace=scratch(j1.op_linear_backward_workspace(M, N, K)))
    d, s = dout.double(), slope64(pre.double(), "silu")
    check_in_parts(BF, x, [d * s], [d.abs() * 2.0 ** -20], [w], dx, [dw], 2.0 ** -133)


def _phi(p):
    return torch.exp(torch.special.log_ndtr(p))


# act(p) and act'(p) without the cancellation that 1 + erf or 1 + tanh has on the far side
def _tail(p, act):
    if act == "gelu":
        s = _phi(p)
        return p * s, s + p * torch.exp(-0.5 * p * p) / math.sqrt(2.0 * math.pi)
    z = p if act == "silu" else 2.0 * math.sqrt(2.0 / math.pi) * (p + 0.044715 * p ** 3)
    dz = torch.ones_like(p) if act == "silu" else 2.0 * math.sqrt(2.0 / math.pi) * (1.0 + 3 * 0.044715 * p * p)
    s = torch.sigmoid(z)
    return p * s, s + p * s * torch.sigmoid(-z) * dz


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_far_side_of_activations(torch_cuda, dtype, act):
    """Negative pre-activations, where activation and slope are small: relative to the value itself, as long as it
    is a normal number of the type. The exponential's argument (up to 126 binary orders) passes a few roundings of
    2^-24 of itself, which the result has as a relative error; value and slope of one unit roundings besides. Factors
    below 2^-126 may be 0 in 32 bits, and the slope has one of them times p and the argument's slope."""
    p = torch.arange(-16.0, 0.0, 2.0 ** -6, device="cuda").to(dtype)
    M, N, K = p.numel(), 8, 16
    x, w = torch.zeros((M, K), device="cuda", dtype=dtype), torch.zeros((N, K), device="cuda", dtype=dtype)
    x[:, 0], w[:, 0] = p, 1.0
    out, dx = torch.empty((M, N), device="cuda", dtype=dtype), torch.empty((M, K), device="cuda", dtype=dtype)
    j1.op_linear(x, w, out, act=ACTS[act])
    value, slope = _tail(p.double(), act)
    orders = (value / p.double()).log2().abs()  # of the logistic function or Phi
    rel = 8 * 2.0 ** -24 * (orders + 8)
    least = float(torch.finfo(dtype).tiny)
    normal = value.abs() > 2 * least
    assert int(normal.sum()) > (240 if dtype == HF else 600)
    close("out", out[normal], value[normal, None].expand(-1, N), ((unit(dtype) + rel) * value.abs() + 2.0 ** -126 * p.double().abs())[normal, None])
    # dx = N equal columns of act'(p), each with what its two terms of opposite sign were off by
    w.zero_()
    w[0, :] = 1.0
    dout = torch.zeros((M, N), device="cuda", dtype=dtype)
    dout[:, 0] = 1.0
    pre = p[:, None].expand(M, N).contiguous()
    j1.op_linear_backward(dout, x, w, pre=pre, act=ACTS[act], dx=dx, workspace=scratch(j1.op_linear_backward_workspace(M, N, K)))
    terms = (value / p.double()).abs() + (slope - value / p.double()).abs()
    steep = {"gelu": p.double().abs(), "silu": torch.ones_like(value), "gelu_tanh": 1.6 * (1 + 0.135 * p.double() ** 2)}[act]
    normal = slope.abs() > 2 * least
    close("dx", dx[normal], slope[normal, None].expand(-1, K), ((unit(dtype) + unit(dtype) ** 2) * slope.abs() + 2 * rel * terms + 2.0 ** -126 * (1 + p.double().abs() * steep))[normal, None])


# ... and those that the list above does not reach: clusters of eight on wide tiles, and stream-K products whose groups are
# single tiles, pairs or more of them, along the rows of tiles or along their columns.
MORE_PLANS = [("gated_backward", (70, 8, 8), BF, "silu"), ("gated_backward", (10135, 8, 905), HF, "gelu"),
              ("gated_backward", (14182, 206, 203), BF, "gelu"), ("gated_backward", (3511, 466, 1153), BF, "gelu"),
              ("gated_backward", (9357, 1923, 157), HF, "silu"), ("gated_backward", (3796, 66, 4978), BF, "silu"),
              ("gated_backward", (3375, 1234, 450), HF, "gelu"), ("gated_backward", (7425, 1223, 717), BF, "gelu"),
              ("gated_backward", (3313, 196, 2555), BF, "gelu_tanh"), ("gated_backward", (13273, 615, 759), HF, "gelu"),
              ("linear_backward", (9732, 9, 892), BF, "gelu"), ("linear_backward", (16058, 412, 202), HF, "silu"),
              ("linear_backward", (7039, 401, 1953), BF, "gelu"), ("linear_backward", (3432, 230, 5080), BF, "gelu"),
              ("linear_backward", (3986, 5250, 200), HF, "gelu"), ("linear_backward", (3740, 191, 5228), BF, "silu"),
              ("linear_backward", (1, 631, 4838), BF, "gelu"), ("linear_backward", (1, 3723, 845), HF, "gelu"),
              ("linear_backward", (28426, 469, 1793), BF, "none"), ("linear_backward", (47429, 1171, 764), BF, "none")]


@pytest.mark.parametrize("i,op,size,dtype,act", [(i,) + p for i, p in enumerate(MORE_PLANS)],
                         ids=["%s-%s" % (p[0], _id(p[1])) for p in MORE_PLANS])
def test_more_plans(torch_cuda, i, op, size, dtype, act):
    check = check_linear_backward if op == "linear_backward" else check_gated_backward
    check(*size, dtype, act, seed=i)


FIRST_CALLS = """
import sys, threading
sys.path.insert(0, %r)
import torch
import julia1 as j1
x, w = (torch.ones(n, 64, device="cuda", dtype=torch.bfloat16) for n in (40, 24))
outs = [torch.zeros(40, 24, device="cuda", dtype=torch.bfloat16) for _ in range(12)]
torch.cuda.synchronize()
gate, errors = threading.Barrier(len(outs)), []

def call(out):
    try:
        gate.wait()
        j1.op_linear(x, w, out)
    except Exception as e:
        errors.append(e)

threads = [threading.Thread(target=call, args=(o,)) for o in outs]
[t.start() for t in threads]
[t.join() for t in threads]
assert not errors, errors
assert all(bool((o == 64).all()) for o in outs)
"""


def test_first_calls_of_many_threads(torch_cuda):
    """The first calls of a process on a device, from several threads at once (its error word and size are looked up by one)."""
    import os
    import subprocess
    import sys
    path = os.path.dirname(os.path.dirname(os.path.abspath(j1.__file__)))
    for _ in range(2):
        r = subprocess.run([sys.executable, "-c", FIRST_CALLS % path], capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stdout + r.stderr


CAPTURED_FIRST = """
import sys
sys.path.insert(0, %r)
import torch
import julia1 as j1
none, wide = torch.empty(0, 8, device="cuda", dtype=torch.bfloat16), torch.empty(8, 8, device="cuda", dtype=torch.bfloat16)
j1.op_linear(none, wide, none)  # the first call, without rows
torch.manual_seed(1)
steps = []
for dtype in (torch.bfloat16, torch.float16):
    for M, N, K in ((1, 64, 40), (300, 72, 136), (77, 65, 51), (2000, 1100, 712), (700, 3392, 392), (7356, 160, 512)):
        e = lambda *s: torch.randn(s, device="cuda").to(dtype)
        t = dict(x=e(M, K), wa=e(N, K), wg=e(N, K), pa=e(M, N), pg=e(M, N), out=e(M, N), y=e(M, N), dout=e(M, N), dx=e(M, K),
                 dwa=e(N, K), dwg=e(N, K), dl=e(M, K), dwl=e(N, K), db=torch.empty(N, device="cuda"), dba=torch.empty(N, device="cuda"),
                 ws=torch.empty(j1.op_gated_backward_workspace(M, N, K), device="cuda", dtype=torch.uint8))
        for act in range(5):
            steps.append((t, act, {k: torch.empty_like(t[k]) for k in ("out", "y", "dx", "dwa", "dwg", "dl", "dwl", "db", "dba")}))

def step(t, act, stream):
    o = dict(act=act, stream=stream, sync=False)
    j1.op_gated(t["x"], t["wa"], t["wg"], t["out"], **o)
    j1.op_linear(t["x"], t["wa"], t["y"], bias=t["db"].fill_(0.5), residual=t["dout"], **o)
    j1.op_gated_backward(t["dout"], t["x"], t["wa"], t["wg"], t["pa"], t["pg"], dx=t["dx"], dwa=t["dwa"], dwg=t["dwg"], dba=t["dba"],
                         workspace=t["ws"], **o)
    j1.op_linear_backward(t["dout"], t["x"], t["wa"], pre=t["pa"], dx=t["dl"], dw=t["dwl"], dbias=t["db"], workspace=t["ws"], **o)

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    for t, act, got in steps:
        step(t, act, torch.cuda.current_stream().cuda_stream)
        for k in got:
            got[k].copy_(t[k])
graph.replay()
torch.cuda.synchronize()
for t, act, got in steps:
    step(t, act, None)
    torch.cuda.synchronize()
    for k in got:
        assert torch.equal(got[k], t[k]), (k, act, t["x"].shape)
"""


def test_captured_after_one_call(torch_cuda):
    """One call of any kind on a device, without rows even, and every kernel of the operators may be captured."""
    import os
    import subprocess
    import sys
    path = os.path.dirname(os.path.dirname(os.path.abspath(j1.__file__)))
    r = subprocess.run([sys.executable, "-c", CAPTURED_FIRST % path], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def test_first_call_in_a_capture(torch_cuda):
    """The first call on a device may be in a capture itself: what it prepares is not part of the graph and does not end it."""
    import os
    import subprocess
    import sys
    path = os.path.dirname(os.path.dirname(os.path.abspath(j1.__file__)))
    first = "j1.op_linear(none, wide, none)"
    assert CAPTURED_FIRST.count(first) == 1
    r = subprocess.run([sys.executable, "-c", CAPTURED_FIRST.replace(first, "pass") % path], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
