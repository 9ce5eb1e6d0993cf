"""Host-side checks of the feed-forward operators (no GPU needed): every refusal happens before
any device call, the argument structs match the header, the workspace sizes are host arithmetic."""
import ctypes as C
import os
import re

import pytest
import torch

import julia1 as j1
from conftest import ROOT, has_gpu

BF, HF = torch.bfloat16, torch.float16


def _linear(M=4, N=8, K=16, dtype=BF):
    return dict(x=torch.zeros(M, K, dtype=dtype), w=torch.zeros(N, K, dtype=dtype), out=torch.zeros(M, N, dtype=dtype))


def _gated(M=4, N=8, K=16, dtype=BF):
    t = _linear(M, N, K, dtype)
    return dict(x=t["x"], wa=t["w"], wg=t["w"].clone(), out=t["out"])


def _linear_grad(M=4, N=8, K=16, dtype=BF):
    t = _linear(M, N, K, dtype)
    return dict(dout=t["out"], x=t["x"], w=t["w"], pre=t["out"].clone(), act=j1.ACT_GELU, dx=t["x"].clone(),
                dw=t["w"].clone(), dbias=torch.zeros(N), workspace=_scratch(j1.op_linear_backward_workspace(M, N, K)))


def _gated_grad(M=4, N=8, K=16, dtype=BF):
    t = _gated(M, N, K, dtype)
    return dict(dout=t["out"], x=t["x"], wa=t["wa"], wg=t["wg"], pre_a=t["out"].clone(), pre_g=t["out"].clone(),
                dx=t["x"].clone(), dwa=t["wa"].clone(), dwg=t["wa"].clone(), dba=torch.zeros(N), dbg=torch.zeros(N),
                workspace=_scratch(j1.op_gated_backward_workspace(M, N, K)))


def _scratch(n):
    t = torch.zeros(n + 256, dtype=torch.uint8)
    return t[-t.data_ptr() % 256:][:n]


OPS = {"linear": (j1.op_linear, _linear), "gated": (j1.op_gated, _gated),
       "linear_backward": (j1.op_linear_backward, _linear_grad), "gated_backward": (j1.op_gated_backward, _gated_grad)}


def _refused(op, message, status=j1.INVALID_ARG, **change):
    call, make = OPS[op]
    args = make()
    args.update(change)
    with pytest.raises(j1.J1Error) as e:
        call(**args)
    assert e.value.status == status and message in str(e.value), str(e.value)


def test_structs_match_the_header():
    text = open(os.path.join(ROOT, "include", "j1.h"), encoding="utf-8").read()
    for name, struct in (("j1_linear_args", j1.J1LinearArgs), ("j1_linear_grad_args", j1.J1LinearGradArgs),
                         ("j1_gated_args", j1.J1GatedArgs), ("j1_gated_grad_args", j1.J1GatedGradArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = []
        for line in body.split(";"):
            m = re.match(r"\s*(const void\*|void\*|const float\*|float\*|int32_t|int64_t|size_t)\s+(.*)", line, re.S)
            if m:
                kind = {"int32_t": C.c_int32, "int64_t": C.c_int64, "size_t": C.c_size_t}.get(m.group(1), C.c_void_p)
                fields += [(n.strip(), kind) for n in m.group(2).split(",")]
        assert fields == list(struct._fields_), name


def test_enums_match_the_header():
    text = open(os.path.join(ROOT, "include", "j1.h"), encoding="utf-8").read()
    values = re.findall(r"\bJ1_((?:ACT|DTYPE)_[A-Z0-9_]+)\s*=\s*(\d+)", text)
    assert len(values) == 7
    for name, v in values:
        assert getattr(j1, name) == int(v)


@pytest.mark.parametrize("op", OPS)
def test_types_and_shapes_are_refused(op):
    _refused(op, "bfloat16 or float16", status=j1.UNSUPPORTED, x=torch.zeros(4, 16))
    _refused(op, "expected", x=torch.zeros(4, 17, dtype=BF))
    _refused(op, "two dimensions", x=torch.zeros(4, 2, 8, dtype=BF))
    _refused(op, "expected", **{"w" if "linear" in op else "wg": torch.zeros(8, 16, dtype=HF)})
    _refused(op, "contiguous", x=torch.zeros(16, 4, dtype=BF).t())
    _refused(op, "row stride below", x=torch.zeros(1, 16, dtype=BF).expand(4, 16))
    _refused(op, "unknown activation", act=5)
    _refused(op, "unknown activation", act=-1)


def test_bias_is_float32_and_contiguous():
    _refused("linear", "float32", bias=torch.zeros(8, dtype=BF))
    _refused("linear", "float32", bias=torch.zeros(7))
    _refused("linear", "float32", bias=torch.zeros(16)[::2])
    _refused("gated", "float32", bg=torch.zeros(8, dtype=torch.float64))
    _refused("linear_backward", "float32", dbias=torch.zeros(8, dtype=HF))


def test_overlaps_are_refused():
    t = _linear(8, 16, 16)
    _refused("linear", "out overlaps x", x=t["x"], w=t["w"], out=t["x"])
    _refused("linear", "out overlaps w", x=torch.zeros(16, 16, dtype=BF), w=t["w"], out=t["w"])
    buf = torch.zeros(8, 16, dtype=BF)
    _refused("linear", "out overlaps pre", x=t["x"], w=t["w"], out=buf, pre=buf)
    # the residual may be the output itself, not a shifted or restrided view of it
    wide = torch.zeros(8, 40, dtype=BF)
    _refused("linear", "out overlaps residual", x=t["x"], w=t["w"], out=wide[:, :16], residual=wide[:, 8:24])
    g = _gated_grad()
    _refused("gated_backward", "dwa overlaps dwg", dwa=g["dwa"], dwg=g["dwa"])
    _refused("linear_backward", "dx overlaps x", **{k: g[k] for k in ("x",)}, dx=g["x"])
    ws = _scratch(j1.op_linear_backward_workspace(4, 8, 16))
    _refused("linear_backward", "overlaps workspace", workspace=ws, dx=ws[:4 * 16 * 2].view(BF).view(4, 16))


@pytest.mark.skipif(has_gpu(), reason="checks the no-device error path")
@pytest.mark.parametrize("op", OPS)
def test_accepted_calls_reach_the_device(op):
    """Without a GPU a call whose arguments are fine ends at the device, not at a check; also for
    halves of one buffer side by side, in-place residuals and stacked weights."""
    call, make = OPS[op]
    variants = [make(), make(1, 1, 1), make(3, 5, 7, HF), make(0, 4, 4)]
    if op == "linear":
        v = make()
        v["residual"] = v["out"]
        variants.append(v)
    if op == "gated":
        both = torch.zeros(4, 16, dtype=BF)
        wi = torch.zeros(16, 16, dtype=BF)
        variants.append(dict(x=torch.zeros(4, 16, dtype=BF), wa=wi[:8], wg=wi[8:], out=torch.zeros(4, 8, dtype=BF),
                             pre_a=both[:, :8], pre_g=both[:, 8:]))
    if op == "gated_backward":
        v = make()
        dwi = torch.zeros(16, 16, dtype=BF)
        v.update(dwa=dwi[:8], dwg=dwi[8:])
        variants.append(v)
    for v in variants:
        with pytest.raises(j1.J1Error) as e:
            call(**v)
        assert e.value.status == j1.CUDA, str(e.value)


def test_what_belongs_together_is_asked_for():
    t = torch.zeros(4, 8, dtype=BF)
    _refused("gated", "go together", pre_a=t)
    _refused("gated_backward", "go together", dwg=None)
    _refused("linear_backward", "no gradient wanted", dx=None, dw=None, dbias=None)
    _refused("gated_backward", "no gradient wanted", dx=None, dwa=None, dwg=None, dba=None, dbg=None)
    _refused("linear_backward", "pre is NULL", pre=None)
    L = j1.lib()
    for op in OPS:
        assert getattr(L, "j1_op_" + op)(None, None, 1) == j1.INVALID_ARG
    a = j1.J1LinearGradArgs(j1.DTYPE_BF16, 0, 4, 8, 16, t.data_ptr(), 8)
    a.dw, a.lddw = torch.zeros(8, 16, dtype=BF).data_ptr(), 16
    assert L.j1_op_linear_backward(a, None, 1) == j1.INVALID_ARG and "dw needs x" in j1.last_error()


def test_raw_sizes_are_refused():
    L = j1.lib()
    t = torch.zeros(64, dtype=BF)
    for sizes, status in (((-1, 8, 8), j1.INVALID_ARG), ((8, 0, 8), j1.INVALID_ARG), ((8, 8, 0), j1.INVALID_ARG),
                          ((2 ** 30 + 1, 8, 8), j1.UNSUPPORTED)):
        a = j1.J1LinearArgs(0, 0, *sizes, t.data_ptr(), 8, t.data_ptr(), 8, None, None, 0, t.data_ptr(), 8, None, 0)
        assert L.j1_op_linear(a, None, 1) == status
    a = j1.J1LinearArgs(2, 0, 1, 8, 8, t.data_ptr(), 8, t.data_ptr(), 8, None, None, 0, t.data_ptr(), 8, None, 0)
    assert L.j1_op_linear(a, None, 1) == j1.INVALID_ARG and "dtype" in j1.last_error()
    a = j1.J1LinearArgs(0, 0, 1, 8, 8, t.data_ptr() + 1, 8, t.data_ptr(), 8, None, None, 0, t.data_ptr(), 8, None, 0)
    assert L.j1_op_linear(a, None, 1) == j1.INVALID_ARG and "aligned" in j1.last_error()


def test_workspace_sizes():
    for size in (j1.op_linear_backward_workspace, j1.op_gated_backward_workspace):
        assert size(0, 1, 1) >= 0 and size(1, 1, 1) > 0
        for bad in ((-1, 1, 1), (1, 0, 1), (1, 1, 0)):
            with pytest.raises(j1.J1Error) as e:
                size(*bad)
            assert e.value.status == j1.INVALID_ARG
        with pytest.raises(j1.J1Error) as e:
            size(2 ** 30 + 1, 1, 1)
        assert e.value.status == j1.UNSUPPORTED
        # the gradients at the pre-activations are kept in 16 bits
        assert size(1000, 512, 64) >= 2 * 1000 * 512
    need = j1.op_gated_backward_workspace(4, 8, 16)
    _refused("gated_backward", "needed", workspace=None)
    _refused("gated_backward", "needed", workspace=_scratch(need - 1))
    _refused("gated_backward", "256-byte aligned", workspace=_scratch(need + 16)[16:])


def test_host_failure_becomes_a_status():
    call, make = OPS["linear"]
    j1.inject_fault(j1.FAULT_HOST, 1)
    try:
        with pytest.raises(j1.J1Error) as e:
            call(**make())
    finally:
        j1.inject_fault(j1.FAULT_HOST, 0)
    assert e.value.status == j1.OOM and "j1_op_linear" in str(e.value)


def test_limits_of_sizes_and_strides():
    """A gated block's two projections are the rows of one product, so its N has half the range; a matrix whose
    last element's offset would not fit an address is refused."""
    L = j1.lib()
    p = torch.zeros(64, dtype=BF).data_ptr()
    with pytest.raises(j1.J1Error) as e:
        j1.op_gated_backward_workspace(1, 2 ** 29 + 1, 1)
    assert e.value.status == j1.UNSUPPORTED
    assert j1.op_gated_backward_workspace(1, 2 ** 29, 1) > 2 ** 31 and j1.op_linear_backward_workspace(1, 2 ** 30, 1) > 2 ** 31
    n = 2 ** 29 + 1
    a = j1.J1GatedArgs(0, 0, 1, n, 1, p, 1, p, 1, p, 1, None, None, p, n, None, 0, None, 0)
    assert L.j1_op_gated(a, None, 1) == j1.UNSUPPORTED and "2^29" in j1.last_error()
    a = j1.J1GatedGradArgs(0, 0, 1, n, 1, p, n, p, 1, p, 1, p, 1, p, n, p, n, p, 1, None, 0, None, 0, None, None, p, 1 << 40)
    assert L.j1_op_gated_backward(a, None, 1) == j1.UNSUPPORTED and "2^29" in j1.last_error()
    for ld, status in ((1 << 38, j1.UNSUPPORTED), ((1 << 38) + 1, j1.UNSUPPORTED)):
        a = j1.J1LinearArgs(0, 0, 1 << 20, 8, 8, p, ld, p, 8, None, None, 0, p, 8, None, 0)
        assert L.j1_op_linear(a, None, 1) == status and "x: " in j1.last_error()


def test_workspace_is_contiguous():
    """An expanded tensor counts far more elements than it has memory."""
    for op in ("linear_backward", "gated_backward"):
        _refused(op, "contiguous", workspace=torch.zeros(1, dtype=torch.uint8).expand(1 << 30))


def _plan_kind(product, M, N, K, act):
    ctas, columns, split, workers, group, across = j1.selftest_ffn_plan(product, M, N, K, act)
    return product, ctas, columns, split, min(group, 3) if workers else 0, across


def test_gpu_tests_take_every_kind_of_plan():
    """Tile shape, cluster size, stream-K groups of one, two or more tiles and their direction: what products of sizes up
    to 131072 x 8192 x 8192 run as on 148 SMs is also run by the GPU tests, so a change of the plans' model shows here."""
    import random
    import test_ffn_gpu as gpu
    products = {"linear": ("linear",), "gated": ("gated",), "linear_backward": ("linear dx", "linear dw"),
                "gated_backward": ("gated dx", "gated dw")}
    run = [(op, size, act) for size in gpu.SIZES for op in products for _, act in gpu.TYPES]
    run += [(op, size, gpu.TYPES[i % len(gpu.TYPES)][1]) for i, (op, size) in enumerate(gpu.PLANS)]
    run += [(op, size, act) for op, size, _, act in gpu.MORE_PLANS]
    tested = {_plan_kind(p, *size, gpu.ACTS[act]) for op, size, act in run for p in products[op]}
    rng, found = random.Random(1), {}
    for _ in range(60000):
        size = tuple(int(2 ** rng.uniform(lo, hi)) for lo, hi in ((0, 17), (3, 13), (3, 13)))
        p, act = rng.choice(j1.FFN_PRODUCTS), rng.choice((j1.ACT_NONE, j1.ACT_GELU))
        found.setdefault(_plan_kind(p, *size, act), (size, act))
    assert len(found) > 50
    missing = {k: v for k, v in found.items() if k not in tested}
    assert not missing, missing


def test_plan_query_refusals():
    L, plan = j1.lib(), (C.c_int32 * 6)()
    for args in ((6, 0, 8, 8, 8, 148), (-1, 0, 8, 8, 8, 148), (0, 5, 8, 8, 8, 148), (0, 0, 0, 8, 8, 148), (0, 0, 8, 0, 8, 148),
                 (0, 0, 8, 8, 8, 1)):
        assert L.j1_selftest_ffn_plan(*args, plan) == j1.INVALID_ARG
    assert L.j1_selftest_ffn_plan(0, 0, 8, 8, 8, 148, None) == j1.INVALID_ARG
    assert L.j1_selftest_ffn_plan(1, 0, 1, 2 ** 29 + 1, 1, 148, plan) == j1.UNSUPPORTED


@pytest.mark.parametrize("size", [j1.op_linear_backward_workspace, j1.op_gated_backward_workspace])
def test_workspace_sizes_beyond_32_bits(size):
    """Sizes that a C int does not hold are refused, not cut to its bits."""
    for at in range(3):
        for n, status in ((2 ** 32 + 64, j1.UNSUPPORTED), (2 ** 31, j1.UNSUPPORTED), (-2 ** 32 + 64, j1.INVALID_ARG)):
            args = [64, 64, 64]
            args[at] = n
            with pytest.raises(j1.J1Error) as e:
                size(*args)
            assert e.value.status == status, args
