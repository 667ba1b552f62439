"""The activations' slopes where they are easily wrong, read off the bias's
gradient of one-row calls (dbias is dp itself)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def _dp(qgemm, gpu, act, pre, dy):
    """dp [n] of one row."""
    n = len(pre)
    pre, dy = (torch.tensor([v], device=gpu).bfloat16() for v in (pre, dy))
    x, w = torch.ones((1, 8), device=gpu).bfloat16(), torch.ones((n, 8), device=gpu).bfloat16()
    _, dw, db = qgemm.linear_backward(dy, x, w, pre, activation=act)
    assert torch.equal(dw[:, 0].float().nan_to_num(7.0), db.float().nan_to_num(7.0))
    return db.float().tolist()


def _same(got, want):
    assert len(got) == len(want)
    for i, (a, b) in enumerate(zip(got, want)):
        assert a == b or (a != a and b != b), (i, a, b)


def test_relu_passes_or_stops(qgemm, gpu):
    pre = [-1.0, -1.0, -INF, 0.0, -0.0, 0.0, 1.0, 1.0, 1.0, INF, INF, NAN, NAN, 2.0 ** -126, -(2.0 ** -126), 5.0]
    dy = [INF, NAN, INF, NAN, INF, 3.0, 2.0, INF, NAN, 4.0, -INF, 5.0, INF, 6.0, 7.0, 0.0]
    want = [0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 2.0, INF, NAN, 4.0, -INF, 5.0, INF, 6.0, 0.0, 0.0]
    _same(_dp(qgemm, gpu, "relu", pre, dy), want)


def test_gated_relu_passes_or_stops(qgemm, gpu):
    """dg is dh u or 0; du = dh relu(g) is a product."""
    g = [-1.0, -1.0, 2.0, 2.0, NAN, 0.0]
    u = [INF, 1.0, 3.0, INF, 2.0, NAN]
    dh = [1.0, INF, 5.0, 1.0, 4.0, 1.0]
    f = len(g)
    gate, up, d = (torch.tensor([v], device=gpu).bfloat16() for v in (g, u, dh))
    pre = qgemm.interleave_gate_up(gate.t(), up.t()).t().contiguous()
    x, w = torch.ones((1, 8), device=gpu).bfloat16(), torch.ones((32, 8), device=gpu).bfloat16()
    _, _, db = qgemm.gated_backward(d, x, w, pre, activation="relu", bias_grad=True)
    dg, du = (t.float().tolist() for t in qgemm.split_gate_up(db, f))
    _same(dg, [0.0, 0.0, 15.0, INF, 8.0, 0.0])
    _same(du, [0.0, NAN, 10.0, 2.0, NAN, 0.0])


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_largest_pre_activations(qgemm, gpu, act):
    """Far from zero the slope is 1 or 0, up to the largest finite values."""
    big = [1e4, 1e13, 1e19, 2e19, 1e30, 3e38]
    _same(_dp(qgemm, gpu, act, big + [-v for v in big] + [0.0, 0.0], [2.0] * 14), [2.0] * 6 + [0.0] * 6 + [1.0] * 2)
    n = len(big)
    bias = torch.tensor(big + [-v for v in big] + [0.0, 0.0], device=gpu)       # A = 0: p is the bias
    a, asc = qgemm.quant_mxfp8(torch.zeros((1, 128), device=gpu))
    b, bsc = qgemm.quant_mxfp8(torch.ones((14, 128), device=gpu))
    y = qgemm.linear_a8w8_mxfp8(a, b, asc, bsc, bias=bias, activation=act, dtype=torch.float32)[0]
    assert torch.equal(y[:n], bias[:n]) and not y[n:].any()
