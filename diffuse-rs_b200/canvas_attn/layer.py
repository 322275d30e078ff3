"""What a layer does around its attention block, on the GPU: the residual
addition and RMS norm of its rows (rms_norm_inplace, src/model/ops.rs:107-114),
products of 8-bit rows, and the gated first half of the feed-forward block
(ffn_block, src/model/forward.rs:354-370, :439-461).

  rms_norm       rows to bf16, fp32 or e4m3 with a scale a row  (ca_rms_norm)
  quantize_rows  the same without the norm                      (ca_rms_norm)
  linear_q8      act . W^T of e4m3 rows, bias, residual         (ca_linear_q8)
  gated_linear   activation(act . Wgate^T) * (act . Wup^T)      (ca_gated_linear)

Each call has a `make_*_args` form for programs that keep their buffers: the
argument block is built once and `*_args(a, stream)` launches it. Calls are
asynchronous on `stream` (None: the legacy default stream) of the tensors'
device, which has to be the current one, and allocate nothing. Like every
tensor of a call, the arguments are to be kept until the work that was
launched with them is done.
"""
from __future__ import annotations

import ctypes

from . import _check, _ptr, _stream, lib

BF16, F32, E4M3 = 0, 1, 2
ACTIVATIONS = {"silu": 0, "gelu": 1}
_TYPES = {"torch.bfloat16": BF16, "torch.float32": F32, "torch.float8_e4m3fn": E4M3}


class CaRmsNormArgs(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("x_type", ctypes.c_int32), ("x_stride", ctypes.c_int64),
                ("residual", ctypes.c_void_p), ("residual_type", ctypes.c_int32),
                ("residual_stride", ctypes.c_int64), ("sum_out", ctypes.c_void_p),
                ("sum_stride", ctypes.c_int64), ("w", ctypes.c_void_p), ("norm", ctypes.c_int32),
                ("eps", ctypes.c_float), ("out", ctypes.c_void_p), ("out_type", ctypes.c_int32),
                ("out_stride", ctypes.c_int64), ("out_scale", ctypes.c_void_p),
                ("rows", ctypes.c_int64), ("cols", ctypes.c_int64)]


class CaLinearQ8Args(ctypes.Structure):
    _fields_ = [("act", ctypes.c_void_p), ("act_stride", ctypes.c_int64),
                ("act_scale", ctypes.c_void_p), ("w", ctypes.c_void_p),
                ("w_scale", ctypes.c_void_p), ("bias", ctypes.c_void_p),
                ("residual", ctypes.c_void_p), ("residual_stride", ctypes.c_int64),
                ("out", ctypes.c_void_p), ("out_f32", ctypes.c_int32),
                ("out_stride", ctypes.c_int64), ("n", ctypes.c_int64), ("rows", ctypes.c_int64),
                ("cols", ctypes.c_int64), ("status", ctypes.c_void_p)]


class CaGatedLinearArgs(ctypes.Structure):
    _fields_ = [("act", ctypes.c_void_p), ("type", ctypes.c_int32), ("act_stride", ctypes.c_int64),
                ("act_scale", ctypes.c_void_p), ("w_gate", ctypes.c_void_p),
                ("w_up", ctypes.c_void_p), ("gate_scale", ctypes.c_void_p),
                ("up_scale", ctypes.c_void_p), ("activation", ctypes.c_int32),
                ("out", ctypes.c_void_p), ("out_f32", ctypes.c_int32),
                ("out_stride", ctypes.c_int64), ("n", ctypes.c_int64), ("rows", ctypes.c_int64),
                ("cols", ctypes.c_int64), ("status", ctypes.c_void_p)]


for _name, _args in (("ca_rms_norm", CaRmsNormArgs), ("ca_linear_q8", CaLinearQ8Args),
                     ("ca_gated_linear", CaGatedLinearArgs)):
    _f = getattr(lib, _name)
    _f.argtypes = [ctypes.POINTER(_args), ctypes.c_void_p]
    _f.restype = ctypes.c_int


def _matrix(name, x, types, shape=None):
    """Checks a [rows, cols] tensor (rows of any stride) and returns its type
    and row stride."""
    kind = _TYPES.get(str(x.dtype))
    if kind not in types:
        raise ValueError(f"{name}: {x.dtype} is not taken here")
    if x.dim() != 2 or (shape is not None and tuple(x.shape) != tuple(shape)):
        raise ValueError(f"{name} must be {list(shape) if shape else '[rows, cols]'}, "
                         f"got {list(x.shape)}")
    if x.shape[1] > 1 and x.stride(1) != 1:
        raise ValueError(f"{name}: columns must be next to one another")
    if x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        raise ValueError(f"{name}: rows must not overlap")
    return kind, int(x.stride(0)) if x.shape[0] > 1 else 0


def _vector(name, x, n):
    if x is None:
        return
    if str(x.dtype) != "torch.float32" or x.numel() != n or not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous float32 with {n} entries")


def _status(x):
    if x is not None and (str(x.dtype) != "torch.int32" or x.numel() < 1):
        raise ValueError("status must be int32")


def one_device(*xs):
    """The tensors of a call are on one device, a GPU where there is one, and
    that is the current one."""
    devices = {x.device for x in xs if x is not None}
    if len(devices) > 1:
        raise ValueError(f"tensors of one call are on {sorted(map(str, devices))}")
    dev = devices.pop()
    import torch
    if dev.type != "cuda" and torch.cuda.is_available():
        raise ValueError(f"tensors are on {dev}")
    if dev.type == "cuda":
        if dev.index not in (None, torch.cuda.current_device()):
            raise ValueError(f"tensors are on {dev}, which is not the current device")


def make_rms_norm_args(x, out, *, w=None, eps: float = 1e-6, norm: bool = True, residual=None,
                       sum_out=None, out_scale=None) -> CaRmsNormArgs:
    """x: bf16 or fp32 [rows, cols]; residual: bf16 or fp32, added to x, and
    sum_out (default: the residual itself) takes the sum; w: fp32 [cols] gain;
    out: bf16, fp32 or e4m3 (then out_scale: fp32 [rows]). norm=False: the rows
    as they are. Rows may have any stride."""
    shape = tuple(x.shape)
    xt, xs = _matrix("x", x, (BF16, F32))
    ot, os_ = _matrix("out", out, (BF16, F32, E4M3), shape)
    rt = rs = ss = 0
    if residual is not None:
        rt, rs = _matrix("residual", residual, (BF16, F32), shape)
        sum_out = residual if sum_out is None else sum_out
        st, ss = _matrix("sum_out", sum_out, (BF16, F32), shape)
        if st != rt:
            raise ValueError("sum_out must have the residual's type")
    elif sum_out is not None:
        raise ValueError("sum_out goes with a residual")
    _vector("w", w, shape[1])
    _vector("out_scale", out_scale, shape[0])
    if ot == E4M3 and out_scale is None:
        raise ValueError("an e4m3 output needs out_scale")
    one_device(x, out, residual, sum_out, w, out_scale)
    a = CaRmsNormArgs(_ptr(x), xt, xs, _ptr(residual), rt, rs, _ptr(sum_out), ss, _ptr(w),
                      1 if norm else 0, float(eps), _ptr(out), ot, os_, _ptr(out_scale),
                      shape[0], shape[1])
    a._keep = (x, out, residual, sum_out, w, out_scale)
    return a


def rms_norm_args(a: CaRmsNormArgs, stream=None) -> None:
    _check(lib.ca_rms_norm(ctypes.byref(a), _stream(stream)), "ca_rms_norm")


def rms_norm(x, out, *, stream=None, **kw) -> None:
    """ca_rms_norm: residual addition and RMS norm of rows (see
    make_rms_norm_args)."""
    rms_norm_args(make_rms_norm_args(x, out, **kw), stream)


def quantize_rows(x, out, out_scale, *, stream=None) -> None:
    """Rows of bf16 or fp32 as e4m3 with a power-of-two scale each: operands of
    linear_q8 and gated_linear."""
    rms_norm_args(make_rms_norm_args(x, out, norm=False, out_scale=out_scale), stream)


def _weights(name, w, types, cols, rows=None):
    kind, _ = _matrix(name, w, types)
    if w.shape[1] != cols or (rows is not None and w.shape[0] != rows) or not w.is_contiguous():
        raise ValueError(f"{name} must be contiguous [rows, {cols}], got {list(w.shape)}")
    return kind


def make_linear_q8_args(act, act_scale, w, w_scale, out, *, bias=None, residual=None,
                        status=None) -> CaLinearQ8Args:
    """act: e4m3 [n, cols], act_scale: fp32 [n] or None; w: e4m3 [rows, cols],
    w_scale: fp32 [rows] or None; out: bf16 or fp32 [n, rows]; bias: fp32
    [rows]; residual: [n, rows] of out's type (may be out). act, out and
    residual may have any stride between rows (act's a multiple of 16)."""
    n, cols = int(act.shape[0]), int(act.shape[1])
    _, as_ = _matrix("act", act, (E4M3,))
    _weights("w", w, (E4M3,), cols)
    rows = int(w.shape[0])
    ot, os_ = _matrix("out", out, (BF16, F32), (n, rows))
    rs = 0
    if residual is not None:
        rt, rs = _matrix("residual", residual, (BF16, F32), (n, rows))
        if rt != ot:
            raise ValueError("residual must have out's type")
    _vector("act_scale", act_scale, n)
    _vector("w_scale", w_scale, rows)
    _vector("bias", bias, rows)
    _status(status)
    one_device(act, act_scale, w, w_scale, out, bias, residual, status)
    a = CaLinearQ8Args(_ptr(act), as_, _ptr(act_scale), _ptr(w), _ptr(w_scale), _ptr(bias),
                       _ptr(residual), rs, _ptr(out), 1 if ot == F32 else 0, os_, n, rows, cols,
                       _ptr(status))
    a._keep = (act, act_scale, w, w_scale, out, bias, residual, status)
    return a


def linear_q8_args(a: CaLinearQ8Args, stream=None) -> None:
    _check(lib.ca_linear_q8(ctypes.byref(a), _stream(stream)), "ca_linear_q8")


def linear_q8(act, act_scale, w, w_scale, out, *, stream=None, **kw) -> None:
    """ca_linear_q8: out = act . w^T (+ bias) (+ residual) over 8-bit operands
    (see make_linear_q8_args)."""
    linear_q8_args(make_linear_q8_args(act, act_scale, w, w_scale, out, **kw), stream)


def make_gated_linear_args(act, w_gate, w_up, out, *, activation: str = "silu",
                           act_scale=None, gate_scale=None, up_scale=None,
                           status=None) -> CaGatedLinearArgs:
    """act: bf16 or e4m3 [n, cols]; w_gate, w_up: [rows, cols] of the same type;
    scales (e4m3): fp32 [n], [rows], [rows] or None; out: bf16 or fp32
    [n, rows]. act and out may have any stride between rows (act's a multiple
    of 16 bytes)."""
    n, cols = int(act.shape[0]), int(act.shape[1])
    kind, as_ = _matrix("act", act, (BF16, E4M3))
    _weights("w_gate", w_gate, (kind,), cols)
    rows = int(w_gate.shape[0])
    _weights("w_up", w_up, (kind,), cols, rows)
    ot, os_ = _matrix("out", out, (BF16, F32), (n, rows))
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}")
    if kind == BF16 and any(s is not None for s in (act_scale, gate_scale, up_scale)):
        raise ValueError("scales go with e4m3 operands")
    _vector("act_scale", act_scale, n)
    _vector("gate_scale", gate_scale, rows)
    _vector("up_scale", up_scale, rows)
    _status(status)
    one_device(act, act_scale, w_gate, w_up, gate_scale, up_scale, out, status)
    a = CaGatedLinearArgs(_ptr(act), kind, as_, _ptr(act_scale), _ptr(w_gate), _ptr(w_up),
                          _ptr(gate_scale), _ptr(up_scale), ACTIVATIONS[activation], _ptr(out),
                          1 if ot == F32 else 0, os_, n, rows, cols, _ptr(status))
    a._keep = (act, act_scale, w_gate, w_up, gate_scale, up_scale, out, status)
    return a


def gated_linear_args(a: CaGatedLinearArgs, stream=None) -> None:
    _check(lib.ca_gated_linear(ctypes.byref(a), _stream(stream)), "ca_gated_linear")


def gated_linear(act, w_gate, w_up, out, *, stream=None, **kw) -> None:
    """ca_gated_linear: activation(act . w_gate^T) * (act . w_up^T) (see
    make_gated_linear_args)."""
    gated_linear_args(make_gated_linear_args(act, w_gate, w_up, out, **kw), stream)
