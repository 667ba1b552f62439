"""silu, gelu and gelu_tanh relative to their own values on the negative side,
where they are small, in fp32: A = 0, so that p is the bias, and the slopes as
the fp32 bias gradient of a one-row call.

Tolerances: an exponential of argument a is off by |a| 2.5 x 2^-24 (the
rounding of a, of a log2 e, and log2 e's own) and 2^-23; a reciprocal by 2^-23;
Phi's rational part by 2^-20; the argument of gelu_tanh's sigmoid has four
roundings more.  Ten roundings of 2^-24 cover the products.  A slope is a
difference of terms of which each has that error."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
ARG = {"silu": lambda v: v.abs(), "gelu": lambda v: v * v / 2, "gelu_tanh": lambda v: 1.6 * v.abs() * (1 + 0.045 * v * v)}
CODE = {"silu": 2, "gelu": 3, "gelu_tanh": 4}
LOW = {"silu": -80.0, "gelu": -12.8, "gelu_tanh": -9.5}         # the values stay normal numbers


def _rel(act, v):
    return ARG[act](v) * 6.5 * 2.0 ** -24 + 2.0 ** -20 + 16 * 2.0 ** -24


def _phi(v):
    return torch.special.erfc(-v * 0.5 ** 0.5) / 2


def _value(act, v):
    s = {"silu": torch.sigmoid(v), "gelu": _phi(v),
         "gelu_tanh": torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3))}[act]
    return v * s


def _points(act, n):
    return torch.cat((torch.linspace(LOW[act], 0, n // 2), torch.linspace(-3, 3, n // 4), torch.linspace(0, 20, n - n // 2 - n // 4)))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m", [1, 130])
def test_values(qgemm, gpu, act, m):
    n, k = 4096, 128
    bias = _points(act, n).to(gpu)
    a, asc = qgemm.quant_mxfp8(torch.zeros((m, k), device=gpu))
    b, bsc = qgemm.quant_mxfp8(torch.ones((n, k), device=gpu))
    y = qgemm.linear_a8w8_mxfp8(a, b, asc, bsc, bias=bias, activation=act, dtype=torch.float32)
    v = bias.double().cpu()
    ref = _value(act, v)
    off = (y.double().cpu() - ref).abs() / (_rel(act, v) * ref.abs() + 1e-300)
    assert torch.isfinite(y).all() and float(off.max()) <= 1, (float(off.max()), float(v[off.max(0).indices.max() % n]))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_slopes(qgemm, gpu, act):
    n = 4096
    pre = _points(act, n).bfloat16().to(gpu).reshape(1, n)
    dy = torch.ones_like(pre)
    db = torch.empty(n, device=gpu)
    g = qgemm.LayerGrad(dy=dy.data_ptr(), pre=pre.data_ptr(), dbias=db.data_ptr(), m=1, n=n, k=8, stride_dy=n, stride_pre=n,
                        dbias_dtype=0, activation=CODE[act])
    need = qgemm.lib().qgemm_layer_backward_workspace_bytes(ctypes.byref(g))
    ws = torch.zeros(need, dtype=torch.uint8, device=gpu)
    st = qgemm.lib().qgemm_layer_backward(ctypes.byref(g), ws.data_ptr(), need,
                                          ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert st == 0
    torch.cuda.synchronize()
    v = pre[0].double().cpu()
    leaf = v.clone().requires_grad_()
    ref, = torch.autograd.grad(_value(act, leaf).sum(), leaf)
    s = _value(act, torch.where(v == 0, 1e-30, v)) / torch.where(v == 0, 1e-30, v)     # sigmoid or Phi
    terms = {"silu": s + v.abs() * s * (1 - s), "gelu": s + v.abs() * torch.exp(-v * v / 2) * 0.4,
             "gelu_tanh": s + v.abs() * s * (1 - s) * 1.6 * (1 + 0.135 * v * v)}[act]
    # 1 - s of a sigmoid is off by the sigmoid's own rounding
    slack = 2.0 ** -22 * v.abs() * (1 + 0.135 * v * v) * s if act != "gelu" else 0.0
    off = (db.double().cpu() - ref).abs() / (_rel(act, v) * terms + slack)
    assert torch.isfinite(db).all() and float(off.max()) <= 1, float(off.max())
