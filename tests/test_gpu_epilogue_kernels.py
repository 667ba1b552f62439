"""Every kernel that a linear layer or gated block can run, by name: each tile of
the ring kernel with and without scale panels, the 128 x 128 kernel in its
stages, the four-wave kernel in its panel widths, and the slice sum after a
split of each, at ragged rows and columns, in both output types.  The test
asserts which kernel ran.  Tolerances as in test_gpu_linear_gated.py."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
FMT = ("fp8", "fp4")


def _ring():
    for fp4 in (0, 1):
        for k in (256, 1024 if fp4 else 512):                   # rows of scales by dwords, then in panels
            for mb, m in ((1, 13), (2, 30), (4, 57)):
                for nb, n, f in ((1, 33, 7), (2, 4101, 2060), (4, 12281, 6140)):
                    if mb == 4 and nb == 4:
                        continue
                    yield f"ring_gemm<{FMT[fp4]},MX,RAW,mb{mb},nb{nb},linear>", fp4, 0, m, n, k
                    yield f"ring_gemm<{FMT[fp4]},MX,RAW,mb{mb},nb{nb},gated>", fp4, 1, m, f, k


def _ring_split():
    shapes = {(0, 1, 1): (1, 33, 7, 5120), (0, 1, 2): (1, 1001, 500, 7168), (0, 1, 4): (1, 2113, 1050, 7168),
              (0, 2, 1): (17, 33, 7, 3328), (0, 2, 2): (17, 1001, 500, 5120), (0, 2, 4): (17, 1537, 1050, 8192),
              (0, 4, 1): (33, 33, 7, 2304), (0, 4, 2): (33, 1537, 500, 5120),
              (1, 1, 1): (1, 33, 7, 16384), (1, 1, 2): (1, 1001, 500, 16384), (1, 1, 4): (1, 1537, 2060, 16384),
              (1, 2, 1): (17, 33, 7, 7168), (1, 2, 2): (17, 1001, 500, 16384), (1, 2, 4): (17, 1537, 1050, 16384),
              (1, 4, 1): (33, 33, 7, 5120), (1, 4, 2): (33, 1537, 500, 16384)}
    for (fp4, mb, nb), (m, n, f, k) in shapes.items():
        yield f"ring_gemm<{FMT[fp4]},MX,RAW,mb{mb},nb{nb},fp32,splitk", fp4, 0, m, n, k
        yield f"ring_gemm<{FMT[fp4]},MX,RAW,mb{mb},nb{nb},fp32,splitk", fp4, 1, m, f, k


def _mid():
    for fp4 in (0, 1):
        for k in (256, 1024 if fp4 else 512):
            for tail, m, n, f in (("st2", 129, 24571, 12280), ("st4,ntb", 65, 33, 7), ("st4", 129, 33, 7), ("st4", 300, 1030, 520)):
                yield f"mid_gemm<{FMT[fp4]},MX,RAW,linear,{tail}>", fp4, 0, m, n, k
                yield f"mid_gemm<{FMT[fp4]},MX,RAW,gated,{tail}>", fp4, 1, m, f, k
    for fp4, tail, m, n, f, k in ((0, "st2,ntb", 17, 24571, 12280, 4096), (0, "st2", 129, 12281, 6140, 4096),
                                  (0, "st4,ntb", 65, 33, 7, 2048), (0, "st4,ntb", 65, 33, 7, 2304), (0, "st4", 129, 33, 7, 3328),
                                  (1, "st2,ntb", 17, 24571, 12280, 8192), (1, "st2", 129, 12281, 6140, 8192),
                                  (1, "st4,ntb", 65, 33, 7, 4096), (1, "st4", 129, 33, 7, 7168)):
        yield f"mid_gemm<{FMT[fp4]},MX,RAW,fp32,{tail},splitk", fp4, 0, m, n, k
        yield f"mid_gemm<{FMT[fp4]},MX,RAW,fp32,{tail},splitk", fp4, 1, m, f, k


def _wide():
    for fp4, pb, m, n, f, k in ((0, 16, 300, 12281, 6140, 2560), (0, 16, 300, 12288, 6144, 2560), (0, 16, 3000, 4100, 2050, 2560),
                                (0, 4, 513, 12281, 6140, 1280), (1, 32, 300, 12281, 6140, 4096), (1, 32, 300, 12288, 6144, 4096),
                                (1, 32, 3000, 4100, 2050, 5120), (1, 16, 513, 12281, 6140, 2560), (1, 8, 300, 12281, 6140, 3328)):
        yield f"wide_gemm<{FMT[fp4]},MX,RAW,linear,pb{pb}>", fp4, 0, m, n, k
        yield f"wide_gemm<{FMT[fp4]},MX,RAW,gated,pb{pb}>", fp4, 1, m, f, k
    for fp4, pb, m, n, f, k in ((0, 16, 513, 6143, 3071, 7168), (0, 16, 512, 12288, 6144, 7168), (1, 32, 513, 6143, 3071, 16384)):
        yield f"wide_gemm<{FMT[fp4]},MX,RAW,fp32,pb{pb}>+epilogue_reduce<linear", fp4, 0, m, n, k
        yield f"wide_gemm<{FMT[fp4]},MX,RAW,fp32,pb{pb}>+epilogue_reduce<gated", fp4, 1, m, f, k


CASES = [*_ring(), *_ring_split(), *_mid(), *_wide()]


def _operand(qgemm, x, fp4):
    """Codes, scales and the values that they stand for, in 64 bits on the GPU."""
    codes, scale = qgemm.quant_mxfp4(x) if fp4 else qgemm.quant_mxfp8(x)
    if fp4:
        c, table = codes.view(torch.uint8), torch.tensor(FP4, dtype=torch.float64, device=x.device)
        v = torch.stack((table[(c & 15).long()], table[(c >> 4).long()]), -1).reshape(x.shape)
    else:
        v = codes.double()
    return codes, scale, v * torch.exp2(scale.double() - 127).repeat_interleave(32, 1)


def _rand(gpu, seed, *shape, scale=1.0):
    return scale * torch.randn(shape, generator=torch.Generator(gpu).manual_seed(seed), device=gpu)


def _check(got, ref, bound):
    d = (got.double() - ref).abs()
    assert torch.isfinite(got).all() and bool((d <= bound).all()), float((d / bound).max())


def _unit(dtype):
    return 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -22


def _problem(qgemm, gpu, fp4, gated, m, n, k):
    """(call, operands, products in 64 bits [m, rows of B], their slack)."""
    a = _operand(qgemm, _rand(gpu, 1, m, k), fp4)
    w = _rand(gpu, 2, n, k, scale=1.5 / k ** 0.5)
    if gated:
        w = qgemm.interleave_gate_up(w, _rand(gpu, 3, n, k, scale=1.5 / k ** 0.5))
    b = _operand(qgemm, w, fp4)
    p = a[2] @ b[2].t()
    name = ("gated" if gated else "linear") + ("_a4w4_mxfp4" if fp4 else "_a8w8_mxfp8")
    return getattr(qgemm, name), (a[0], b[0], a[1], b[1]), p, float(1e-3 * p.square().mean().sqrt())


def _gelu(v):
    return 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))


def _linear_ref(p, bias, res, slack, dtype):
    p = p + bias.double()
    ref = _gelu(p) + res.double()
    return p, ref, _unit(dtype) * ref.abs() + 1.2 * slack + 2.0 ** -18 * (p.abs() + res.double().abs())


def _gated_ref(qgemm, p, bias, n, slack, dtype):
    p = p + bias.double()
    g, u = (t.t() for t in qgemm.split_gate_up(p.t(), n))
    y = g * torch.sigmoid(g)
    ref = y * u
    return p, ref, (_unit(dtype) * ref.abs() + 1.2 * slack * u.abs() + slack * (y.abs() + 1.2 * slack)
                    + 2.0 ** -18 * (g * u).abs())


def _ids(c):
    return f"{c[0].replace(',MX,RAW', '').rstrip('>')}-{c[3]}x{c[4]}x{c[5]}-{'gated' if c[2] else 'linear'}"


@pytest.mark.parametrize("case", CASES, ids=_ids)
def test_kernel(qgemm, gpu, case):
    kernel, fp4, gated, m, n, k = case
    call, ops, p64, slack = _problem(qgemm, gpu, fp4, gated, m, n, k)
    rows = p64.shape[1]
    for dtype, btype in ((torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)):
        bias = _rand(gpu, 4, rows).to(btype)
        if gated:
            args, kw = (n,), {"bias": bias, "dtype": dtype}
            p, ref, bound = _gated_ref(qgemm, p64, bias, n, slack, dtype)
        else:
            res = _rand(gpu, 5, m, n + 3).to(btype)[:, :n]
            args, kw = (), {"bias": bias, "dtype": dtype, "activation": "gelu", "residual": res}
            p, ref, bound = _linear_ref(p64, bias, res, slack, dtype)
        y, pre = call(*ops, *args, save_pre=True, **kw)
        assert kernel in qgemm.last_launch()
        _check(pre, p, 2.0 ** -8 * p.abs() + slack)
        _check(y, ref, bound)
        assert torch.equal(call(*ops, *args, **kw), y)
        if kernel.startswith("wide_gemm") and "reduce" not in kernel:       # scales as they lie, without a copy in panels
            bare = call(*ops, *args, workspace=False, **kw)
            assert kernel in qgemm.last_launch() and "panels" not in qgemm.last_launch()
            assert torch.equal(bare, y)


# one of each kernel, unsplit and split
PADDED = ["ring_gemm<fp8,MX,RAW,mb2,nb1,", "ring_gemm<fp4,MX,RAW,mb4,nb2,", "ring_gemm<fp8,MX,RAW,mb1,nb4,",
          "mid_gemm<fp8,MX,RAW,linear,st4>", "mid_gemm<fp8,MX,RAW,gated,st4>", "mid_gemm<fp4,MX,RAW,fp32,st4,",
          "wide_gemm<fp8,MX,RAW,linear,pb16>", "wide_gemm<fp8,MX,RAW,gated,pb16>", "wide_gemm<fp4,MX,RAW,linear,pb32>",
          "wide_gemm<fp4,MX,RAW,gated,pb32>", "wide_gemm<fp8,MX,RAW,fp32,pb16>"]


@pytest.mark.parametrize("case", [c for c in CASES if any(c[0].startswith(p) for p in PADDED)], ids=_ids)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nothing_beside_the_rows(qgemm, gpu, case, dtype):
    """The C entry with padded rows of C, pre and the residual: the dense call's bits, and the gaps as they were."""
    kernel, fp4, gated, m, n, k = case
    call, (ac, bc, asc, bsc), p64, _ = _problem(qgemm, gpu, fp4, gated, m, n, k)
    rows = p64.shape[1]
    bias, kb = _rand(gpu, 4, rows), ac.shape[1]
    res = None if gated else _rand(gpu, 5, m, n).bfloat16()
    kw = {} if gated else {"activation": "gelu", "residual": res}
    want, want_pre = call(ac, bc, asc, bsc, *((n,) if gated else ()), bias=bias, dtype=dtype, save_pre=True, **kw)
    mark = 7.0
    for pad, off in ((1, 1), (5, 0), (8, 8)):
        def rows_of(width, t):
            buf = torch.full((off + m * (width + pad) + 8,), mark, dtype=t, device=gpu)
            return buf, buf[off:off + m * (width + pad)].view(m, width + pad)
        cbuf, c = rows_of(n, dtype)
        pbuf, pre = rows_of(rows, torch.bfloat16)
        args = qgemm.Kargs(ac.data_ptr(), bc.data_ptr(), c.data_ptr(), m, rows, k, 1, kb, kb, n + pad, 0, 0, 0, asc.data_ptr(),
                           bsc.data_ptr(), k // 32, k // 32, 0, 0)
        epi = qgemm.Epilogue(bias=bias.data_ptr(), pre=pre.data_ptr(), bias_dtype=0, stride_pre=rows + pad,
                             activation=2 if gated else 3)
        if not gated:
            rbuf, r = rows_of(n, torch.bfloat16)
            r[:, :n] = res
            epi.residual, epi.residual_dtype, epi.stride_residual = r.data_ptr(), 1, n + pad
        lib, entry = qgemm.lib(), ("gemm_a4w4_mxfp4_" if fp4 else "gemm_a8w8_mxfp8_") + ("gated" if gated else "linear")
        need = getattr(lib, entry + "_workspace_bytes")(ctypes.byref(args))
        ws = torch.zeros(need, dtype=torch.uint8, device=gpu) if need else None
        st = getattr(lib, entry)(ctypes.byref(args), ctypes.byref(epi), *((n,) if gated else ()), int(dtype == torch.bfloat16),
                                 ws.data_ptr() if need else None, need,
                                 ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert st == 0 and kernel in qgemm.last_launch()
        torch.cuda.synchronize()
        assert torch.equal(c[:, :n], want) and torch.equal(pre[:, :rows], want_pre)
        for buf, t, width in ((cbuf, c, n), (pbuf, pre, rows)):
            assert bool((t[:, width:] == mark).all()) and bool((buf[:off] == mark).all()) and bool((buf[off + t.numel():] == mark).all())
