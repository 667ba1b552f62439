"""Rows whose offsets pass 32 bits: views with a very long pitch give the bits
of their contiguous copies, and matrices of more than 2^31 elements the sums in
64 bits (tolerances of test_gpu_layer_backward.py)."""
import pytest
import torch

from test_gpu_layer_backward import _check_product, _check_sums, _rand

pytestmark = pytest.mark.gpu


def _far(rows, cols, pitch, seed, gpu, dtype=torch.bfloat16):
    """An [rows, cols] view with rows `pitch` elements apart, and its contiguous copy."""
    flat = torch.empty((rows - 1) * pitch + cols, dtype=dtype, device=gpu)
    v = flat.as_strided((rows, cols), (pitch, 1))
    g = torch.Generator(gpu).manual_seed(seed)
    v.copy_(torch.randn((rows, cols), generator=g, device=gpu))
    return v, v.clone(memory_format=torch.contiguous_format)


def _same(got, want):
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("n", [96, 7168, 17000])
def test_norm(qgemm, gpu, n):
    pitch = 2 ** 31 - 8
    x, xc = _far(3, n, pitch, 1, gpu)
    dy, dyc = _far(3, n, pitch, 2, gpu)
    w = torch.randn(n, device=gpu)
    want = qgemm.layer_norm(xc, w, w, stats=True)
    _same(qgemm.layer_norm(x, w, w, stats=True), want)
    _same(qgemm.layer_norm_backward(dy, x, *want[1:], w), qgemm.layer_norm_backward(dyc, xc, *want[1:], w))
    del x, dy
    torch.cuda.empty_cache()


@pytest.mark.parametrize("act", ["none", "silu"])
def test_backward_of_far_rows(qgemm, gpu, act):
    m, n, k = 5, 192, 256
    dy, dyc = _far(m, n, 2 ** 30 + 3, 1, gpu)
    pre, prec = _far(m, n, 2 ** 30 + 5, 2, gpu)
    x, w = _rand(gpu, 3, m, k), _rand(gpu, 4, n, k)
    _same(qgemm.linear_backward(dy, x, w, pre, activation=act), qgemm.linear_backward(dyc, x, w, prec, activation=act))
    del dy, pre
    torch.cuda.empty_cache()


@pytest.mark.parametrize("m", [2, 70, 600])
def test_residual_of_far_rows(qgemm, gpu, m):
    n, k, pitch = 256, 512, 2 ** 31 // m + 8 * m
    res, resc = _far(m, n, pitch, 1, gpu)
    a, sa = qgemm.quant_mxfp8(_rand(gpu, 2, m, k).float())
    b, sb = qgemm.quant_mxfp8(_rand(gpu, 3, n, k).float())
    for dtype in (torch.bfloat16, torch.float32):
        _same((qgemm.linear_a8w8_mxfp8(a, b, sa, sb, residual=res, dtype=dtype),),
              (qgemm.linear_a8w8_mxfp8(a, b, sa, sb, residual=resc, dtype=dtype),))
    del res
    torch.cuda.empty_cache()


def test_backward_of_large_matrices(qgemm, gpu):
    """x and dx of 2.6e9 elements: rows at their ends and around 2^31 elements, and dw's columns."""
    m, n, k = 40000, 64, 65536
    g = torch.Generator(gpu).manual_seed(1)
    x = torch.empty((m, k), dtype=torch.bfloat16, device=gpu)
    for i in range(0, m, 4000):
        x[i:i + 4000] = torch.randn((4000, k), generator=g, device=gpu)
    dy, w, pre = _rand(gpu, 2, m, n), _rand(gpu, 3, n, k, scale=0.05), _rand(gpu, 4, m, n)
    dx, dw, db = qgemm.linear_backward(dy, x, w, pre, activation="relu")
    dp = dy.double() * (pre > 0)
    _check_sums(db, dp)
    at = 2 ** 31 // k
    for rows in (slice(0, 64), slice(at - 64, at + 64), slice(m - 64, m)):
        _check_product(dx[rows], dp[rows], w.double())
    for cols in (slice(0, 512), slice(k // 2, k // 2 + 512), slice(k - 512, k)):
        _check_product(dw[:, cols], dp.t(), x[:, cols].double())
    del x, dx
    torch.cuda.empty_cache()


def test_norm_of_large_matrices(qgemm, gpu):
    m, n = 300001, 7168                            # 2.15e9 elements
    x = torch.empty((m, n), dtype=torch.bfloat16, device=gpu)
    g = torch.Generator(gpu).manual_seed(1)
    for i in range(0, m, 30000):
        rows = min(30000, m - i)
        x[i:i + rows] = torch.randn((rows, n), generator=g, device=gpu)
    w = torch.randn(n, device=gpu)
    y, mean, rstd = qgemm.layer_norm(x, w, w, stats=True)
    dx, _, _ = qgemm.layer_norm_backward(x, x, mean, rstd, w)
    for rows in (slice(0, 8), slice(2 ** 31 // n - 4, 2 ** 31 // n + 4), slice(m - 8, m)):
        part = x[rows].clone()
        want = qgemm.layer_norm(part, w, w, stats=True)
        _same((y[rows], mean[rows], rstd[rows]), want)
        _same(qgemm.layer_norm_backward(part, part, *want[1:], w)[:1], (dx[rows],))
    del x, y, dx
    torch.cuda.empty_cache()
