"""The C forms that the Python calls never make: each gradient alone or with any
other, the bias's in fp32, padded outputs; a norm's weight or bias gradient
alone and padded rows.  Products and sums against 64 bits with the tolerances of
test_gpu_layer_backward.py and test_gpu_layer_norm.py; padded outputs against the
dense call's bits, with the gaps as they were."""
import ctypes
import itertools

import pytest
import torch

from test_gpu_layer_backward import _act, _check, _check_product, _rand, _slope

pytestmark = pytest.mark.gpu
ACT = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
PARTS = [p for r in (1, 2, 3) for p in itertools.combinations(("dx", "dw", "db"), r)]


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _padded(rows, cols, pad, gpu, dtype=torch.bfloat16):
    return torch.full((rows, cols + pad), 7.0, dtype=dtype, device=gpu)


def _call(qgemm, gpu, parts, dy, pre, x, w, act, features, fp32_bias, pad):
    """The requested gradients, as padded matrices; operands of the others are not given."""
    (m, k), n = x.shape, w.shape[0]
    dx, dw = _padded(m, k, pad, gpu), _padded(n, k, pad, gpu)
    db = torch.full((n + 8,), 7.0, dtype=torch.float32 if fp32_bias else torch.bfloat16, device=gpu)
    g = qgemm.LayerGrad(dy=dy.data_ptr(), m=m, n=n, k=k, features=features, stride_dy=dy.stride(0), activation=ACT[act],
                        dbias_dtype=0 if fp32_bias else 1)
    if pre is not None:
        g.pre, g.stride_pre = pre.data_ptr(), pre.stride(0)
    if "dx" in parts:
        g.dx, g.stride_dx, g.w, g.stride_w = dx.data_ptr(), k + pad, w.data_ptr(), w.stride(0)
    if "dw" in parts:
        g.dw, g.stride_dw, g.x, g.stride_x = dw.data_ptr(), k + pad, x.data_ptr(), x.stride(0)
    if "db" in parts:
        g.dbias = db.data_ptr()
    lib = qgemm.lib()
    need = lib.qgemm_layer_backward_workspace_bytes(ctypes.byref(g))
    ws = torch.full((need + 256,), 0xA5, dtype=torch.uint8, device=gpu)
    ws[:2048] = 0
    assert lib.qgemm_layer_backward(ctypes.byref(g), ws.data_ptr(), need, _stream()) == 0
    launch = qgemm.last_launch()
    torch.cuda.synchronize()
    assert bool((ws[need:] == 0xA5).all())
    # what was not asked for is not written, and nothing beside the rows
    for name, t, width in (("dx", dx, k), ("dw", dw, k)):
        assert bool((t[:, width if name in parts else 0:] == 7).all()), name
    assert bool((db[n if "db" in parts else 0:] == 7).all())
    return {"dx": dx[:, :k], "dw": dw[:, :k], "db": db[:n]}, launch


def _problem(qgemm, gpu, kind, act, m, n, k):
    """n: rows of w, or the features of a gated block."""
    x, pre_scale = _rand(gpu, 2, m, k), 1.5
    dy = _rand(gpu, 1, m, n)
    if kind == "linear":
        w = _rand(gpu, 3, n, k, scale=0.05)
        pre = None if act == "none" else _rand(gpu, 4, m, n, scale=pre_scale)
        dp = dy.double() * (1.0 if act == "none" else _slope(pre.double(), act))
        return dy, pre, x, w, dp, 0
    w = qgemm.interleave_gate_up(_rand(gpu, 3, n, k, scale=0.05), _rand(gpu, 4, n, k, scale=0.05))
    pre = _rand(gpu, 5, m, w.shape[0])
    g, u = (t.t() for t in qgemm.split_gate_up(pre.double().t().contiguous(), n))
    dg, du = dy.double() * u * _slope(g, act), dy.double() * _act(g, act)
    return dy, pre, x, w, qgemm.interleave_gate_up(dg.t().contiguous(), du.t().contiguous()).t(), n


# one tile, ragged tiles, either sum split
SHAPES = [(1, 16, 8), (65, 127, 264), (1000, 96, 2048), (77, 4096, 512), (2049, 513, 520)]


@pytest.mark.parametrize("parts", PARTS, ids="-".join)
@pytest.mark.parametrize("kind,act", [("linear", "none"), ("linear", "silu"), ("gated", "gelu")])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_any_gradients(qgemm, gpu, parts, kind, act, m, n, k):
    dy, pre, x, w, dp, features = _problem(qgemm, gpu, kind, act, m, n, k)
    for fp32_bias in (False, True):
        if fp32_bias and "db" not in parts:
            continue
        got, launch = _call(qgemm, gpu, parts, dy, pre, x, w, act, features, fp32_bias, 0)
        if "dx" in parts:
            _check_product(got["dx"], dp, w.double())
        if "dw" in parts:
            _check_product(got["dw"], dp.t(), x.double())
        if "db" in parts:
            ref = dp.sum(0)
            _check(got["db"], ref, 2.0 ** (-24 if fp32_bias else -8) * ref.abs() + 2.0 ** -17 * dp.abs().sum(0) + 1e-30)
        padded, again = _call(qgemm, gpu, parts, dy, pre, x, w, act, features, fp32_bias, 24)
        assert again == launch
        for name in parts:
            assert torch.equal(padded[name], got[name])


def test_splits_are_among_them(qgemm, gpu):
    """Either product alone runs with a split sum, and without one."""
    seen = set()
    for m, n, k in SHAPES:
        dy, pre, x, w, _, features = _problem(qgemm, gpu, "linear", "silu", m, n, k)
        for part in ("dx", "dw"):
            launch = _call(qgemm, gpu, (part,), dy, pre, x, w, "silu", features, False, 0)[1]
            seen.add((part, "splitk1>" not in launch))
    assert seen == {("dx", True), ("dx", False), ("dw", True), ("dw", False)}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n", [(1, 7), (37, 100), (50, 513), (33, 2048), (9, 4100), (20, 8192), (5, 16384), (3, 17000)])
def test_norm_gradients_alone(qgemm, gpu, dtype, m, n):
    """dweight or dbias NULL, padded dx: the bits of the call with both."""
    code = 0 if dtype == torch.float32 else 1
    x, dy = (torch.randn((m, n), generator=torch.Generator(gpu).manual_seed(s), device=gpu).to(dtype) for s in (1, 2))
    w = torch.randn(n, device=gpu)
    _, mean, rstd = qgemm.layer_norm(x, w, stats=True)
    want = qgemm.layer_norm_backward(dy, x, mean, rstd, w)
    lib = qgemm.lib()
    need = lib.qgemm_layer_norm_backward_workspace_bytes(m, n)
    vec = 16 // x.element_size()                         # rows whose starts keep the dense call's load width
    for parts, pad in itertools.product((("dw", "db"), ("dw",), ("db",), ()), (0, vec)):
        dx = _padded(m, n, pad, gpu, dtype)
        dw, db = (torch.full((n + 4,), 7.0, device=gpu) for _ in range(2))
        ws = torch.full((need + 256,), 0xA5, dtype=torch.uint8, device=gpu)
        ws[:2048] = 0
        st = lib.qgemm_layer_norm_backward(dy.data_ptr(), n, x.data_ptr(), n, code, m, n, mean.data_ptr(), rstd.data_ptr(),
                                           w.data_ptr(), 0, dx.data_ptr(), n + pad, dw.data_ptr() if "dw" in parts else None,
                                           db.data_ptr() if "db" in parts else None, ws.data_ptr() if parts else None,
                                           need if parts else 0, _stream())
        assert st == 0
        torch.cuda.synchronize()
        assert torch.equal(dx[:, :n], want[0]) and bool((dx[:, n:] == 7).all()) and bool((ws[need:] == 0xA5).all())
        for name, t, ref in (("dw", dw, want[1]), ("db", db, want[2])):
            assert bool((t[n if name in parts else 0:] == 7).all())
            assert name not in parts or torch.equal(t[:n], ref)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [7, 96, 1000, 7168, 17000])
def test_norm_padded_output(qgemm, gpu, dtype, n):
    m, code, pad = 21, 0 if dtype == torch.float32 else 1, 16
    x = torch.randn((m, n), device=gpu).to(dtype)
    w = torch.randn(n, device=gpu).bfloat16()
    want, mean, rstd = qgemm.layer_norm(x, w, w, stats=True)
    y, stats = _padded(m, n, pad, gpu, dtype), torch.full((2, m + 4), 7.0, device=gpu)
    st = qgemm.lib().qgemm_layer_norm(x.data_ptr(), code, m, n, n, w.data_ptr(), w.data_ptr(), 1, 1e-5, y.data_ptr(), n + pad,
                                      stats[0].data_ptr(), stats[1].data_ptr(), _stream())
    assert st == 0
    torch.cuda.synchronize()
    assert torch.equal(y[:, :n], want) and bool((y[:, n:] == 7).all())
    assert torch.equal(stats[0, :m], mean) and torch.equal(stats[1, :m], rstd) and bool((stats[:, m:] == 7).all())
