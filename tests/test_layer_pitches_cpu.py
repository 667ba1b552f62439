"""Sizes and row pitches past 31 bits, which the library's 32-bit arguments
cannot hold: the Python wrappers refuse them before any call.  The tensors are
meta tensors (a shape and strides, no memory); with everything in range the same
calls go on to the library."""
import importlib

import pytest
import torch

FAR = 2 ** 32 + 64        # cut to 32 bits it would be 64, a pitch that fits the rows
BF = torch.bfloat16


class Reached(Exception):
    pass


@pytest.fixture
def layer(qgemm, monkeypatch):
    layer = importlib.import_module("355_1_trans_amd.layer")

    def reached(*_):
        raise Reached

    monkeypatch.setattr(layer, "fast", lambda: qgemm._NoFast)
    monkeypatch.setattr(layer, "_require_gpu", lambda *t: t[0].device)
    monkeypatch.setattr(torch.cuda, "device", reached)
    return layer


def _meta(rows, cols, pitch=None, dtype=BF):
    return torch.empty_strided((rows, cols), (cols if pitch is None else pitch, 1), dtype=dtype, device="meta")


def _vec(n):
    return torch.empty(n, device="meta")


def _mx(m, n, k):
    byte = torch.uint8
    return _meta(m, k, dtype=byte), _meta(n, k, dtype=byte), _meta(m, k // 32, dtype=byte), _meta(n, k // 32, dtype=byte)


CALLS = {
    "norm": lambda q, ld: q.layer_norm(_meta(2, 64, ld)),
    "norm_rows": lambda q, ld: q.layer_norm(_meta(ld, 1)),
    "norm_columns": lambda q, ld: q.layer_norm(_meta(1, ld)),
    "norm_grad_dy": lambda q, ld: q.layer_norm_backward(_meta(2, 64, ld), _meta(2, 64), _vec(2), _vec(2)),
    "norm_grad_x": lambda q, ld: q.layer_norm_backward(_meta(2, 64), _meta(2, 64, ld), _vec(2), _vec(2)),
    "residual": lambda q, ld: q.linear_a8w8_mxfp8(*_mx(2, 64, 128), residual=_meta(2, 64, ld)),
    "linear_columns": lambda q, ld: q.linear_a8w8_mxfp8(*_mx(1, 1, ld * 128)),
    "linear_fp4_columns": lambda q, ld: q.linear_a4w4_mxfp4(
        _meta(1, ld * 64, dtype=torch.uint8), _meta(1, ld * 64, dtype=torch.uint8), _meta(1, ld * 4, dtype=torch.uint8),
        _meta(1, ld * 4, dtype=torch.uint8)),
    "gated_rows": lambda q, ld: q.gated_a8w8_mxfp8(*_mx(ld, 32, 128), 16),
    "grad_dy": lambda q, ld: q.linear_backward(_meta(2, 64, ld), _meta(2, 64), _meta(64, 64)),
    "grad_x": lambda q, ld: q.linear_backward(_meta(2, 64), _meta(2, 64, ld), _meta(64, 64)),
    "grad_w": lambda q, ld: q.linear_backward(_meta(2, 64), _meta(2, 64), _meta(64, 64, ld)),
    "grad_pre": lambda q, ld: q.linear_backward(_meta(2, 64), _meta(2, 64), _meta(64, 64), _meta(2, 64, ld), "silu"),
    "gated_grad_pre": lambda q, ld: q.gated_backward(_meta(2, 32), _meta(2, 64), _meta(64, 64), _meta(2, 64, ld)),
    "gated_grad_rows": lambda q, ld: q.gated_backward(_meta(ld, 16), _meta(ld, 64), _meta(32, 64), _meta(ld, 32)),
}


@pytest.mark.parametrize("name", CALLS)
def test_past_31_bits_is_refused(qgemm, layer, name):
    for far in (FAR, 2 ** 31):
        with pytest.raises(ValueError, match=r"below 2\*\*31"):
            CALLS[name](qgemm, far)


@pytest.mark.parametrize("name", CALLS)
def test_in_range_reaches_the_library(qgemm, layer, name):
    with pytest.raises(Reached):
        CALLS[name](qgemm, 72 if name not in ("linear_columns", "linear_fp4_columns") else 8)
