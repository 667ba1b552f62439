"""Sizes and row pitches past 31 bits in the quantizers, layouts and products:
refused by the Python wrappers, as the library's 32-bit arguments cannot hold
them.  Meta tensors: a shape and strides, no memory."""
import importlib

import pytest
import torch

FAR = 2 ** 32 + 256       # cut to 32 bits it would be 256


class Reached(Exception):
    pass


@pytest.fixture
def q(qgemm, monkeypatch):
    def reached(*_):
        raise Reached

    for name in ("355_1_trans_amd", "355_1_trans_amd.quant", "355_1_trans_amd.opus"):
        mod = importlib.import_module(name)
        monkeypatch.setattr(mod, "_require_gpu", lambda *t: t[0].device)
        if hasattr(mod, "fast"):
            monkeypatch.setattr(mod, "fast", lambda: qgemm._NoFast)
    monkeypatch.setattr(torch.cuda, "device", reached)
    return qgemm


def _meta(*shape, pitch=None, dtype=torch.uint8):
    if pitch is None:
        return torch.empty(shape, dtype=dtype, device="meta")
    return torch.empty_strided(shape, (pitch, 1), dtype=dtype, device="meta")


def _mx(m, n, k, fp4=False):
    kb = k // 2 if fp4 else k
    return _meta(m, kb), _meta(n, kb), _meta(m, k // 32), _meta(n, k // 32)


def _bs(k, b):
    f = torch.float32
    return _meta(1, k), b, _meta(1, k // 128, dtype=f), _meta(1, k // 128, dtype=f)


def _opus(q):
    return importlib.import_module("355_1_trans_amd.opus")


def _x(ld):
    return _meta(2, 256, pitch=ld, dtype=torch.bfloat16)


CALLS = {
    "quant_mxfp8": lambda q, v: q.quant_mxfp8(_x(v)),
    "quant_mxfp4": lambda q, v: q.quant_mxfp4(_x(v)),
    "quant_fp8_blockscale": lambda q, v: q.quant_fp8_blockscale(_x(v)),
    "quant_fp8_blockscale_weight": lambda q, v: q.quant_fp8_blockscale(_x(v), "128x128"),
    "quant_fp8_e8m0_blockscale": lambda q, v: q.quant_fp8_e8m0_blockscale(_x(v)),
    "quant_rows": lambda q, v: q.quant_mxfp8(_meta(v, 32, dtype=torch.bfloat16)),
    "e8m0_shuffle": lambda q, v: q.e8m0_shuffle(_meta(2, 256, pitch=v)),
    "relayout": lambda q, v: importlib.import_module("355_1_trans_amd.quant").relayout_device(
        "qgemm_shuffle_b_kpanel_device", _meta(2, 256, pitch=v), 512),
    "mxfp8": lambda q, v: q.gemm_a8w8_mxfp8(*_mx(1, 1, v)),
    "mxfp4": lambda q, v: q.gemm_a4w4_mxfp4(*_mx(1, 1, v, True)),
    "kpanel": lambda q, v: q.gemm_a8w8_bpreshuffle(*_bs(v, _meta(v // 128, 1, 128))),
    "reference": lambda q, v: q.reference_gemm("mxfp8", *_mx(1, 1, v)),
    "opus_mxfp8": lambda q, v: _opus(q).gemm_a8w8_mxfp8_opus(*_mx(1, 1, v)),
}


@pytest.mark.parametrize("name", CALLS)
def test_past_31_bits_is_refused(q, name):
    for far in (FAR, 2 ** 31):
        with pytest.raises(ValueError, match=r"below 2\*\*31"):
            CALLS[name](q, far)


@pytest.mark.parametrize("name", CALLS)
def test_in_range_reaches_the_library(q, name):
    with pytest.raises(Reached):
        CALLS[name](q, 512)


def test_one_row_of_any_pitch(q):
    """The pitch of a single row is not used."""
    with pytest.raises(Reached):
        q.quant_mxfp8(_meta(1, 256, pitch=FAR, dtype=torch.bfloat16))
