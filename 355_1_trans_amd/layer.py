"""The layer around the quantised products, PyTorch-facing: layer norm,
linear layers (bias, activation, residual) and gated feed-forward blocks on
MXFP8 / MXFP4 operands, and their gradients.

Calls launch on the current stream and record every tensor on it; there is no
CPU fallback.  Sizes and row pitches (in elements) are below 2**31.  The calls
are not part of autograd: results carry no gradient, also where an input
requires one, and the *_backward calls are made by hand, with the tensors that
the forward call used and returned; nothing is kept between calls.
"""
import ctypes

import torch

from . import (_WORKSPACES, Epilogue, Kargs, LayerGrad, _check, _int32, _out, _out_code, _record, _require_gpu,
               _stream, _workspace_of, _ws_tensor, fast, lib)

_TYPES = {torch.float32: 0, torch.bfloat16: 1}
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def _activation(name):
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}")
    return ACTIVATIONS[name]


def _rows(t, name, like=None):
    """dtype code and row pitch of a 2-D fp32 / bf16 tensor with contiguous rows."""
    if t.dim() != 2 or t.dtype not in _TYPES:
        raise ValueError(f"{name} must be a 2-D float32 or bfloat16 GPU tensor")
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype):
        raise ValueError(f"{name} must have the shape and dtype of the tensor beside it")
    if t.shape[1] == 0 or (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{name} needs at least one column and contiguous rows that do not overlap")
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    _int32(name, *t.shape, ld)
    return _TYPES[t.dtype], ld


def _vectors(n, *pairs):
    """The one dtype code of the given [n] vectors (name, tensor or None)."""
    code = None
    for name, v in pairs:
        if v is None:
            continue
        if v.shape != (n,) or v.dtype not in _TYPES or not v.is_contiguous():
            raise ValueError(f"{name} must be a contiguous float32 or bfloat16 vector of {n} elements")
        if code not in (None, _TYPES[v.dtype]):
            raise ValueError("weight and bias must have one dtype")
        code = _TYPES[v.dtype]
    return 0 if code is None else code


def _ptr(t):
    return None if t is None else t.data_ptr()


def layer_norm(x, weight=None, bias=None, eps=1e-5, stats=False, out=None):
    """Layer norm over the rows of x [M, N] (fp32 or bf16, contiguous rows of
    any pitch and length), weight and bias [N] fp32 or bf16 (None: ones,
    zeros): y like x, rounded once from fp32.  ``stats``: (y, mean, rstd),
    fp32 [M], as layer_norm_backward takes them."""
    if out is None:
        y = fast().norm(x, weight, bias, eps, stats)
        if y is not None:
            return y
    dev = _require_gpu(x, *(t for t in (weight, bias) if t is not None))
    code, ldx = _rows(x, "x")
    m, n = x.shape
    wcode = _vectors(n, ("weight", weight), ("bias", bias))
    y = _out(out, (m, n), x.dtype, dev)
    mean = torch.empty(m, dtype=torch.float32, device=dev) if stats else None
    rstd = torch.empty(m, dtype=torch.float32, device=dev) if stats else None
    if m:
        with torch.cuda.device(dev):
            s = _stream(dev)
            st = lib().qgemm_layer_norm(x.data_ptr(), code, m, n, ldx, _ptr(weight), _ptr(bias), wcode, float(eps),
                                        y.data_ptr(), n, _ptr(mean), _ptr(rstd), ctypes.c_void_p(s.cuda_stream))
            _record(s, x, weight, bias, y, mean, rstd)
        _check(st, "qgemm_layer_norm")
    return (y, mean, rstd) if stats else y


def layer_norm_backward(dy, x, mean, rstd, weight=None, weight_grad=True, workspace=None):
    """(dx, dweight, dbias) of layer_norm: dx like x, dweight and dbias [N] of
    weight's dtype (fp32 without a weight; None, None without
    ``weight_grad``).  mean and rstd come from layer_norm(..., stats=True).
    ``workspace``: None for the cached one, or a uint8 tensor of at least
    qgemm_layer_norm_backward_workspace_bytes."""
    if weight_grad and workspace is None:
        grads = fast().norm_grad(dy, x, mean, rstd, weight, _WORKSPACES)
        if grads is not None:
            return grads
    dev = _require_gpu(dy, x, mean, rstd, *(() if weight is None else (weight,)))
    code, ldx = _rows(x, "x")
    _, lddy = _rows(dy, "dy", x)
    m, n = x.shape
    for name, v in (("mean", mean), ("rstd", rstd)):
        if v.shape != (m,) or v.dtype != torch.float32 or not v.is_contiguous():
            raise ValueError(f"{name} must be a contiguous float32 vector of {m} elements")
    wcode = _vectors(n, ("weight", weight))
    wtype = torch.float32 if weight is None else weight.dtype
    dx = torch.empty((m, n), dtype=x.dtype, device=dev)
    make = torch.empty if m else torch.zeros
    dweight = make(n, dtype=wtype, device=dev) if weight_grad else None
    dbias = make(n, dtype=wtype, device=dev) if weight_grad else None
    if m:
        with torch.cuda.device(dev):
            s = _stream(dev)
            need = lib().qgemm_layer_norm_backward_workspace_bytes(m, n) if weight_grad else 0
            wp, wb = _workspace_of(need, workspace, dev, s)
            st = lib().qgemm_layer_norm_backward(dy.data_ptr(), lddy, x.data_ptr(), ldx, code, m, n, mean.data_ptr(),
                                                 rstd.data_ptr(), _ptr(weight), wcode, dx.data_ptr(), n,
                                                 _ptr(dweight), _ptr(dbias), wp, wb, ctypes.c_void_p(s.cuda_stream))
            _record(s, dy, x, mean, rstd, weight, dx, dweight, dbias,
                    workspace if isinstance(workspace, torch.Tensor) else None)
        _check(st, "qgemm_layer_norm_backward")
    return dx, dweight, dbias


def _mx_operands(A, B, A_scale, B_scale, fp4):
    """(device, m, n, kargs without C) of row-major MX operands."""
    dev = _require_gpu(A, B, A_scale, B_scale)
    step = 256 if fp4 else 128
    for t in (A, B, A_scale, B_scale):
        if t.dim() != 2 or t.element_size() != 1 or not t.is_contiguous():
            raise ValueError("A, B and scales must be contiguous 2-D byte tensors")
    m, kb = A.shape
    n, k = B.shape[0], 2 * kb if fp4 else kb
    if B.shape[1] != kb or k % step or k == 0 or n == 0:
        raise ValueError(f"requires matching K with K % {step} == 0 and at least one row of B")
    if A_scale.shape != (m, k // 32) or B_scale.shape != (n, k // 32):
        raise ValueError("requires A_scale [M,K/32] and B_scale [N,K/32]")
    _int32("A, B", m, n, k)
    kg = k // 32
    args = Kargs(A.data_ptr(), B.data_ptr(), None, m, n, k, 1, kb, kb, 0, 0, 0, 0, A_scale.data_ptr(),
                 B_scale.data_ptr(), kg, kg, 0, 0)
    return dev, m, n, args


def _product(name, tensors, args, dev, cols, features, bias, activation, residual, dtype, save_pre, out, workspace):
    """C = epilogue(A B^T) [m, cols] through the entry `name`."""
    m, n = args.m, args.n
    epi = Epilogue(activation=_activation(activation))
    out_code = _out_code(dtype)
    if bias is not None:
        epi.bias_dtype = _vectors(n, ("bias", bias))
        epi.bias = bias.data_ptr()
    if residual is not None:
        if residual.shape != (m, cols):
            raise ValueError("residual must have the output's shape")
        if m:
            epi.residual_dtype, epi.stride_residual = _rows(residual, "residual")
            epi.residual = residual.data_ptr()
    for t in (bias, residual):
        if t is not None and t.device != dev:
            raise ValueError("all tensors must be on the same GPU")
    out = _out(out, (m, cols), dtype, dev)
    pre = torch.empty((m, n), dtype=torch.bfloat16, device=dev) if save_pre else None
    if m:
        args.ptr_c, args.stride_c = out.data_ptr(), cols
        epi.pre, epi.stride_pre = (pre.data_ptr() if save_pre else None), n
        extra = () if features is None else (features,)
        with torch.cuda.device(dev):
            s = _stream(dev)
            need = getattr(lib(), name + "_workspace_bytes")(ctypes.byref(args)) if workspace is not False else 0
            wp, wb = _workspace_of(need, None if workspace is False else workspace, dev, s)
            st = getattr(lib(), name)(ctypes.byref(args), ctypes.byref(epi), *extra, out_code, wp, wb,
                                      ctypes.c_void_p(s.cuda_stream))
            _record(s, *tensors, bias, residual, out, pre, _ws_tensor(workspace))
        _check(st, name)
    return (out, pre) if save_pre else out


def _linear(fp4, A, B, A_scale, B_scale, bias, activation, residual, dtype, save_pre, out, workspace):
    if out is None and workspace is None:
        y = fast().product(fp4, A, B, A_scale, B_scale, 0, bias, ACTIVATIONS.get(activation, -1), residual, dtype,
                           save_pre, _WORKSPACES)
        if y is not None:
            return y
    dev, m, n, args = _mx_operands(A, B, A_scale, B_scale, fp4)
    return _product("gemm_a4w4_mxfp4_linear" if fp4 else "gemm_a8w8_mxfp8_linear", (A, B, A_scale, B_scale), args, dev,
                    n, None, bias, activation, residual, dtype, save_pre, out, workspace)


def linear_a8w8_mxfp8(A, B, A_scale, B_scale, bias=None, activation="none", residual=None, dtype=torch.bfloat16,
                      save_pre=False, out=None, workspace=None):
    """act(A B^T + bias) + residual in one pass: operands as gemm_a8w8_mxfp8 takes
    them; bias [N] and residual [M, N] fp32 or bf16; activation "none", "relu",
    "silu", "gelu" (v Phi(v)) or "gelu_tanh".  ``save_pre``: (y, A B^T + bias as
    bf16), which linear_backward reads.  ``out`` may be the residual."""
    return _linear(False, A, B, A_scale, B_scale, bias, activation, residual, dtype, save_pre, out, workspace)


def linear_a4w4_mxfp4(A, B, A_scale, B_scale, bias=None, activation="none", residual=None, dtype=torch.bfloat16,
                      save_pre=False, out=None, workspace=None):
    """linear_a8w8_mxfp8 on gemm_a4w4_mxfp4's operands."""
    return _linear(True, A, B, A_scale, B_scale, bias, activation, residual, dtype, save_pre, out, workspace)


def interleave_gate_up(gate, up):
    """The weight of a gated block from its gate and up projections [F, K]:
    [2 * (F rounded up to 16), K], 16 rows of gate, 16 of up, and so on; rows
    past F are zero.  (Any dtype; for a bias, [F] -> [2 * ...].)"""
    if gate.shape != up.shape or gate.dtype != up.dtype:
        raise ValueError("gate and up must have one shape and dtype")
    f = gate.shape[0]
    out = torch.zeros(((f + 15) // 16, 2, 16, *gate.shape[1:]), dtype=gate.dtype, device=gate.device)
    for i, part in enumerate((gate, up)):
        full = f // 16 * 16
        out[: f // 16, i] = part[:full].reshape(f // 16, 16, *gate.shape[1:])
        if f % 16:
            out[f // 16, i, : f % 16] = part[full:]
    return out.reshape(-1, *gate.shape[1:])


def split_gate_up(w, features):
    """(gate, up) [features, ...] of a tensor in interleave_gate_up's row order."""
    if w.shape[0] != 2 * ((features + 15) // 16 * 16):
        raise ValueError("w must have 2 * (features rounded up to 16) rows")
    parts = w.reshape(-1, 2, 16, *w.shape[1:])
    return tuple(parts[:, i].reshape(-1, *w.shape[1:])[:features] for i in (0, 1))


def _gated(fp4, A, B, A_scale, B_scale, features, bias, activation, dtype, save_pre, out, workspace):
    if out is None and workspace is None and features:
        h = fast().product(fp4, A, B, A_scale, B_scale, features, bias, ACTIVATIONS.get(activation, -1), None, dtype,
                           save_pre, _WORKSPACES)
        if h is not None:
            return h
    dev, m, n, args = _mx_operands(A, B, A_scale, B_scale, fp4)
    features = int(features)
    if features < 1 or n != 2 * ((features + 15) // 16 * 16):
        raise ValueError("B must have 2 * (features rounded up to 16) rows (interleave_gate_up)")
    return _product("gemm_a4w4_mxfp4_gated" if fp4 else "gemm_a8w8_mxfp8_gated", (A, B, A_scale, B_scale), args, dev,
                    features, features, bias, activation, None, dtype, save_pre, out, workspace)


def gated_a8w8_mxfp8(A, B, A_scale, B_scale, features, bias=None, activation="silu", dtype=torch.bfloat16,
                     save_pre=False, out=None, workspace=None):
    """act(A G^T) * (A U^T) [M, features] in one pass: B is the quantised
    interleave_gate_up(G, U), bias in the same row order.  ``save_pre``: (h,
    pre), pre [M, B's rows] bf16 as gated_backward reads it."""
    return _gated(False, A, B, A_scale, B_scale, features, bias, activation, dtype, save_pre, out, workspace)


def gated_a4w4_mxfp4(A, B, A_scale, B_scale, features, bias=None, activation="silu", dtype=torch.bfloat16,
                     save_pre=False, out=None, workspace=None):
    """gated_a8w8_mxfp8 on gemm_a4w4_mxfp4's operands."""
    return _gated(True, A, B, A_scale, B_scale, features, bias, activation, dtype, save_pre, out, workspace)


def _bf16(t, name, shape):
    if t.dtype != torch.bfloat16 or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be bfloat16 of shape {tuple(shape)}")
    return _rows(t, name)[1] if shape[0] else shape[1]


def _operand16(t, name, shape):
    """Row pitch of an operand that the products load in 16-byte pieces."""
    ld = _bf16(t, name, shape)
    if shape[0] and (t.data_ptr() % 16 or ld % 8):
        raise ValueError(f"{name}'s rows must start on 16 bytes")
    return ld


def _backward(dy, x, w, pre, features, activation, bias_grad, workspace):
    if workspace is None:
        grads = fast().layer_grad(dy, x, w, pre, features, ACTIVATIONS.get(activation, -1), bias_grad, _WORKSPACES)
        if grads is not None:
            return grads
    dev = _require_gpu(dy, x, w, *(() if pre is None else (pre,)))
    if x.dim() != 2 or w.dim() != 2:
        raise ValueError("x and w must be 2-D")
    (m, k), n = x.shape, w.shape[0]
    if k == 0 or k % 8 or n == 0:
        raise ValueError("requires K % 8 == 0, at least one column and one row of w")
    _int32("x, w", m, n, k)
    act = _activation(activation)
    if pre is None and (features or act):
        raise ValueError("pre (the forward call's save_pre) is needed")
    g = LayerGrad(m=m, n=n, k=k, features=features, dbias_dtype=1, activation=act)
    g.stride_dy = _bf16(dy, "dy", (m, features or n))
    g.stride_x, g.stride_w = _operand16(x, "x", (m, k)), _operand16(w, "w", (n, k))
    if pre is not None:
        g.stride_pre = _bf16(pre, "pre", (m, n))
    make = torch.empty if m else torch.zeros
    dx = torch.empty((m, k), dtype=torch.bfloat16, device=dev)
    dw = make((n, k), dtype=torch.bfloat16, device=dev)
    db = make(n, dtype=torch.bfloat16, device=dev) if bias_grad else None
    if m:
        g.dy, g.pre, g.x, g.w = dy.data_ptr(), _ptr(pre), x.data_ptr(), w.data_ptr()
        g.dx, g.dw, g.dbias, g.stride_dx, g.stride_dw = dx.data_ptr(), dw.data_ptr(), _ptr(db), k, k
        with torch.cuda.device(dev):
            s = _stream(dev)
            wp, wb = _workspace_of(lib().qgemm_layer_backward_workspace_bytes(ctypes.byref(g)), workspace, dev, s)
            st = lib().qgemm_layer_backward(ctypes.byref(g), wp, wb, ctypes.c_void_p(s.cuda_stream))
            _record(s, dy, x, w, pre, dx, dw, db, _ws_tensor(workspace))
        _check(st, "qgemm_layer_backward")
    return dx, dw, db


def linear_backward(dy, x, w, pre=None, activation="none", bias_grad=True, workspace=None):
    """(dx [M, K], dw [N, K], dbias [N] or None) of y = act(x w^T + bias): dy
    [M, N], x [M, K], w [N, K] and pre (linear_*'s save_pre; not read for
    activation "none") bf16, results bf16.  The quantisation of a linear_* call
    counts as the identity; the residual's gradient is dy itself.
    ``workspace``: None for the cached one, or a uint8 tensor of at least
    qgemm_layer_backward_workspace_bytes."""
    return _backward(dy, x, w, pre, 0, activation, bias_grad, workspace)


def gated_backward(dy, x, w, pre, activation="silu", bias_grad=False, workspace=None):
    """(dx [M, K], dw) of h = act(x G^T) * (x U^T), with ``bias_grad`` (dx, dw,
    dbias): dy [M, features], w and pre (gated_*'s save_pre) in
    interleave_gate_up's order, dw and dbias in the same order."""
    features = dy.shape[1] if dy.dim() == 2 else 0
    if features < 1 or w.dim() != 2 or w.shape[0] != 2 * ((features + 15) // 16 * 16):
        raise ValueError("w must have 2 * (features rounded up to 16) rows for dy [M, features]")
    dx, dw, db = _backward(dy, x, w, pre, features, activation, bias_grad, workspace)
    return (dx, dw, db) if bias_grad else (dx, dw)
