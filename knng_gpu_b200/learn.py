"""The projection that makes the searched rows, and the loss that trains it.

Device operators on CUDA torch tensors, through ``libknng_gpu.so``:

* :func:`linear`, :func:`linear_backward` -- ``act(x w^T + bias) + residual``
  and its gradients;
* :func:`softmax_xent`, :func:`softmax_xent_backward` -- softmax cross entropy
  over the inner products of ``x`` with every row of ``w`` (classes, or the
  base rows of a search), without the (m, n) scores in memory, and its
  gradients.

Matrices are 2-D, bfloat16, float16 or float32, with any row stride (the last
dimension contiguous). Calls are asynchronous on ``stream`` (default: torch's
current stream). With another stream, make it wait for the inputs first, as
for any torch operation; tensors made here belong to that stream. ``workspace``
is a uint8 CUDA tensor of at least the call's ``*_workspace_bytes`` bytes (the
C ABI's), allocated here when not given. The operators build no autograd graph.
"""
from __future__ import annotations

from contextlib import nullcontext
from struct import Struct

import torch

from ._native import gpu_lib
from .api import InvalidArgument, check

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_current_scope = nullcontext()


class _Operator:
    """One C entry point: its argument structure as a byte format (the mirrors
    in _native spell the fields out), its two functions once loaded."""

    def __init__(self, name: str, fields: str):
        self.name, self.fields = name, Struct(fields)
        self.size = self.call = None

    def run(self, device, workspace, *values) -> None:
        """On the current device and stream of the caller's :func:`_scope`."""
        if self.call is None:
            lib = gpu_lib()
            self.size = getattr(lib, f"knng_gpu_{self.name}_workspace_bytes")
            self.call = getattr(lib, f"knng_gpu_{self.name}")
        args = self.fields.pack(*values)
        if workspace is None:
            need = self.size(args)
            if need:
                workspace = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=device)
        stream = torch.cuda.current_stream(device).cuda_stream if _raw_stream is None else _raw_stream(device.index)
        if workspace is None:
            status = self.call(args, None, 0, stream)
        else:
            status = self.call(args, workspace.data_ptr(), workspace.numel(), stream)
        if status:
            check(status)


# The current stream's handle without making a Stream object (2 us), where torch offers it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)

_LINEAR = _Operator("linear", "14Q3i4x")
_LINEAR_BACKWARD = _Operator("linear_backward", "14Q2i")
_XENT = _Operator("softmax_xent", "10Qf2i4x")
_XENT_BACKWARD = _Operator("softmax_xent_backward", "12Qf2i4x")


def _dtype_id(op: str, dtype) -> int:
    d = _DTYPES.get(dtype)
    if d is None:
        raise InvalidArgument(f"knng::gpu::{op}: dtype must be float32, bfloat16 or float16, not {dtype}")
    return d


def _stride(op: str, name: str, t, rows: int, cols: int) -> int:
    """Row stride of a 2-D CUDA tensor of that shape, after its checks."""
    if t.dim() != 2 or not t.is_cuda:
        raise InvalidArgument(f"knng::gpu::{op}: {name} must be a 2-D CUDA tensor")
    if t.shape != (rows, cols):
        raise InvalidArgument(f"knng::gpu::{op}: {name} is {tuple(t.shape)}, expected ({rows}, {cols})")
    s0, s1 = t.stride()
    if s1 != 1 and cols > 1:
        raise InvalidArgument(f"knng::gpu::{op}: the rows of {name} must be contiguous")
    if rows <= 1:
        return cols
    if s0 < cols:
        raise InvalidArgument(f"knng::gpu::{op}: the rows of {name} overlap")
    return s0


def _operands(op: str, x, w):
    """Sizes, strides and type of x (m, k) and w (n, k)."""
    if x.dim() != 2 or w.dim() != 2:
        raise InvalidArgument(f"knng::gpu::{op}: x and w must be 2-D CUDA tensors")
    m, k = x.shape
    n = w.shape[0]
    _same(op, "w", w, x)
    return m, k, n, _stride(op, "x", x, m, k), _stride(op, "w", w, n, k), _dtype_id(op, x.dtype)


def _same(op: str, name: str, t, x) -> None:
    if t.dtype != x.dtype or t.device != x.device:
        raise InvalidArgument(f"knng::gpu::{op}: {name} must have the dtype and device of x")


def _vector(op: str, name: str, t, n: int, dtype, device) -> int:
    """Address of a dense vector."""
    if t.dim() != 1 or t.shape[0] != n or t.dtype != dtype or t.device != device:
        raise InvalidArgument(f"knng::gpu::{op}: {name} must be a {dtype} vector of {n} values on {device}")
    if n > 1 and t.stride(0) != 1:
        raise InvalidArgument(f"knng::gpu::{op}: {name} must be contiguous")
    return t.data_ptr()


def _labels(op: str, t, m: int, device):
    """Address and whether int64."""
    if t.dtype not in (torch.int64, torch.int32):
        raise InvalidArgument(f"knng::gpu::{op}: labels must be int64 or int32")
    return _vector(op, "labels", t, m, t.dtype, device), int(t.dtype == torch.int64)


def _activation(op: str, name: str) -> int:
    act = ACTIVATIONS.get(name)
    if act is None:
        raise InvalidArgument(f"knng::gpu::{op}: unknown activation {name!r}")
    return act


def _scope(device, stream, *inputs):
    """Allocations and launches on the tensors' device and the call's stream.
    On another stream than the current one the allocator learns that the
    inputs are in use there, so that they may be dropped after the call."""
    if stream is not None:
        for t in inputs:
            if t is not None:
                t.record_stream(stream)
        return torch.cuda.stream(stream)
    if device.index != torch.cuda.current_device():
        return torch.cuda.device(device)
    return _current_scope


def _rows(rows: int, cols: int, dtype, device):
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def linear(x, w, bias=None, residual=None, activation="none", out_dtype=None, out=None, save_pre=False,
           workspace=None, stream=None):
    """``act(x w^T + bias) + residual`` for x (m, k), w (n, k).

    ``activation``: "none", "relu", "gelu", "gelu_tanh" or "silu".
    ``out_dtype`` may be float32 (rows for :func:`brute_force_knn_device`)
    instead of x's. With ``save_pre`` returns ``(out, pre)``, pre = x w^T +
    bias in x's dtype, which :func:`linear_backward` takes.
    """
    op = "linear"
    m, k, n, ldx, ldw, dtype = _operands(op, x, w)
    act = _activation(op, activation)
    device = x.device
    ldr = 0
    if bias is not None:
        _vector(op, "bias", bias, n, x.dtype, device)
    if residual is not None:
        _same(op, "residual", residual, x)
        ldr = _stride(op, "residual", residual, m, n)
    if out is not None and (out.device != device or (out_dtype is not None and out.dtype != out_dtype)):
        raise InvalidArgument("knng::gpu::linear: out has another dtype or device than asked for")
    with _scope(device, stream, x, w, bias, residual, out, workspace):
        if out is None:
            out, ldo = _rows(m, n, out_dtype or x.dtype, device), n
        else:
            ldo = _stride(op, "out", out, m, n)
        pre = _rows(m, n, x.dtype, device) if save_pre else None
        _LINEAR.run(device, workspace, m, k, n, x.data_ptr(), ldx, w.data_ptr(), ldw, _ptr(bias), _ptr(residual), ldr,
                    out.data_ptr(), ldo, _ptr(pre), n, dtype, _dtype_id(op, out.dtype), act)
    return (out, pre) if save_pre else out


def linear_backward(dy, x, w, pre=None, activation="none", need_dx=True, need_dw=True, need_db=False,
                    workspace=None, stream=None):
    """Gradients of :func:`linear` from ``dy`` (m, n): ``(dx, dw, db)``, None
    where not needed. ``pre`` is what the forward call saved (not needed
    without an activation). The residual's gradient is ``dy``."""
    op = "linear_backward"
    m, k, n, ldx, ldw, dtype = _operands(op, x, w)
    act = _activation(op, activation)
    _same(op, "dy", dy, x)
    lddy, ldp = _stride(op, "dy", dy, m, n), 0
    if pre is not None:
        _same(op, "pre", pre, x)
        ldp = _stride(op, "pre", pre, m, n)
    elif act:
        raise InvalidArgument("knng::gpu::linear_backward: pre is needed with an activation")
    device = x.device
    with _scope(device, stream, dy, x, w, pre, workspace):
        dx = _rows(m, k, x.dtype, device) if need_dx else None
        dw = _rows(n, k, x.dtype, device) if need_dw else None
        db = torch.empty(n, dtype=x.dtype, device=device) if need_db else None
        _LINEAR_BACKWARD.run(device, workspace, m, k, n, dy.data_ptr(), lddy, x.data_ptr(), ldx, w.data_ptr(), ldw,
                             _ptr(pre), ldp, _ptr(dx), _ptr(dw), _ptr(db), dtype, act)
    return dx, dw, db


def softmax_xent(x, w, labels, scale=1.0, workspace=None, stream=None):
    """Per-row softmax cross entropy over ``scale * x w^T``: ``(loss, lse)``,
    float32 (m,). ``labels`` (m,) int64 or int32 name a row of w; a label
    outside [0, n) leaves its row out (loss 0; lse is still that row's)."""
    op = "softmax_xent"
    m, k, n, ldx, ldw, dtype = _operands(op, x, w)
    device = x.device
    y, i64 = _labels(op, labels, m, device)
    with _scope(device, stream, x, w, labels, workspace):
        loss = torch.empty_strided((m,), (1,), dtype=torch.float32, device=device)
        lse = torch.empty_strided((m,), (1,), dtype=torch.float32, device=device)
        _XENT.run(device, workspace, m, k, n, x.data_ptr(), ldx, w.data_ptr(), ldw, y, loss.data_ptr(), lse.data_ptr(),
                  scale, dtype, i64)
    return loss, lse


def softmax_xent_backward(dloss, x, w, labels, lse, scale=1.0, need_dx=True, need_dw=True, workspace=None,
                          stream=None):
    """Gradients of :func:`softmax_xent` from ``dloss`` (m,) float32 and the
    forward call's ``lse``: ``(dx, dw)`` in x's dtype, None where not needed.
    A row without a label has dx 0 and adds nothing to dw, whatever it holds."""
    op = "softmax_xent_backward"
    m, k, n, ldx, ldw, dtype = _operands(op, x, w)
    device = x.device
    y, i64 = _labels(op, labels, m, device)
    at_dloss = _vector(op, "dloss", dloss, m, torch.float32, device)
    at_lse = _vector(op, "lse", lse, m, torch.float32, device)
    with _scope(device, stream, dloss, x, w, labels, lse, workspace):
        dx = _rows(m, k, x.dtype, device) if need_dx else None
        dw = _rows(n, k, x.dtype, device) if need_dw else None
        _XENT_BACKWARD.run(device, workspace, m, k, n, at_dloss, x.data_ptr(), ldx, w.data_ptr(), ldw, y, at_lse,
                           _ptr(dx), _ptr(dw), scale, dtype, i64)
    return dx, dw
