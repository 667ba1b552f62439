"""Layer norm of single rows whose column numbers, or twice them, pass 31 bits.

Tolerances as in test_gpu_layer_norm.py: 32 x 2^-24 of the sizes that go into
a value for its fp32 roundings (a thread adds 64 elements in fp32 and those
sums in 64 bits; the 1024 threads' are added in fp32 by wave, then 16 of them:
about ten levels), 2^-8 of the value for a bf16 output."""
import pytest
import torch

pytestmark = pytest.mark.gpu
EPS = 1e-5
CHUNK = 1 << 27


def _chunks(n):
    return [slice(i, min(i + CHUNK, n)) for i in range(0, n, CHUNK)]


def _row(n, gpu, seed, mean):
    g = torch.Generator(gpu).manual_seed(seed)
    x = torch.empty((1, n), dtype=torch.bfloat16, device=gpu)
    for s in _chunks(n):
        x[0, s] = 2 * torch.randn(s.stop - s.start, generator=g, device=gpu) + mean
    return x


def _stats(x):
    n = x.shape[1]
    mean = sum(x[0, s].double().sum() for s in _chunks(n)) / n
    var = sum((x[0, s].double() - mean).square().sum() for s in _chunks(n)) / n
    return mean, 1 / torch.sqrt(var + EPS)


def test_forward(qgemm, gpu):
    n = 2 ** 31 - 1
    x = _row(n, gpu, 1, 3.0)
    y, mean, rstd = qgemm.layer_norm(x, eps=EPS, stats=True)
    m64, r64 = _stats(x)
    assert abs(float(mean) - float(m64)) <= 32 * 2.0 ** -24 * 16 and abs(float(rstd / r64) - 1) <= 32 * 2.0 ** -24 * 4
    for s in _chunks(n):
        ref = (x[0, s].double() - m64) * r64
        assert bool(((y[0, s].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 32 * 2.0 ** -24 * 16).all())
        del ref
    torch.cuda.empty_cache()


def test_backward(qgemm, gpu):
    n = 2 ** 30 + 8            # 2 n passes 31 bits
    x, dy = _row(n, gpu, 1, 3.0), _row(n, gpu, 2, 0.5)
    m64, r64 = _stats(x)
    mean, rstd = m64.float().reshape(1), r64.float().reshape(1)
    need = qgemm.lib().qgemm_layer_norm_backward_workspace_bytes(1, n)
    ws = torch.empty(need, dtype=torch.uint8, device=gpu)
    dx, dw, db = qgemm.layer_norm_backward(dy, x, mean, rstd, workspace=ws)
    m64, r64 = mean.double(), rstd.double()
    sums = [0.0, 0.0]
    for s in _chunks(n):
        xh = (x[0, s].double() - m64) * r64
        sums[0] += dy[0, s].double().sum() / n
        sums[1] += (dy[0, s].double() * xh).sum() / n
    for s in _chunks(n):
        xh, g = (x[0, s].double() - m64) * r64, dy[0, s].double()
        ref = r64 * (g - sums[0] - xh * sums[1])
        assert bool(((dx[0, s].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 32 * 2.0 ** -24 * 64).all())
        # one row: dweight and dbias are its terms
        assert bool(((dw[s].double() - g * xh).abs() <= 32 * 2.0 ** -24 * (g * (1 + xh.abs())).abs() + 32 * 2.0 ** -24).all())
        assert torch.equal(db[s], dy[0, s].float())
        del xh, g, ref
    del ws, dx, dw, db
    torch.cuda.empty_cache()
