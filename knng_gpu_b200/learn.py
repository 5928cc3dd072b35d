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

import ctypes
from contextlib import nullcontext

from . import _native
from ._native import gpu_lib
from .api import InvalidArgument, check

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_dtypes: dict = {}


def _dtype_id(op: str, dtype) -> int:
    if not _dtypes:
        import torch

        _dtypes.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
    if dtype not in _dtypes:
        raise InvalidArgument(f"knng::gpu::{op}: dtype must be float32, bfloat16 or float16, not {dtype}")
    return _dtypes[dtype]


def _matrix(op: str, name: str, t, rows: int | None, cols: int | None, like=None):
    """Row stride of a 2-D tensor after its checks (None sizes are free)."""
    if t.dim() != 2 or not t.is_cuda:
        raise InvalidArgument(f"knng::gpu::{op}: {name} must be a 2-D CUDA tensor")
    r, c = t.shape
    if (rows is not None and r != rows) or (cols is not None and c != cols):
        raise InvalidArgument(f"knng::gpu::{op}: {name} is {tuple(t.shape)}, expected "
                              f"({'any' if rows is None else rows}, {'any' if cols is None else cols})")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise InvalidArgument(f"knng::gpu::{op}: {name} must have the dtype and device of the other operands")
    s0, s1 = t.stride()
    if c > 1 and s1 != 1:
        raise InvalidArgument(f"knng::gpu::{op}: the rows of {name} must be contiguous")
    if r <= 1:
        return c
    if s0 < c:
        raise InvalidArgument(f"knng::gpu::{op}: the rows of {name} overlap")
    return s0


def _vector(op: str, name: str, t, n: int, dtype, device):
    if t.dim() != 1 or t.shape[0] != n or t.dtype != dtype or t.device != device:
        raise InvalidArgument(f"knng::gpu::{op}: {name} must be a {dtype} vector of {n} values on {device}")
    if n > 1 and t.stride(0) != 1:
        raise InvalidArgument(f"knng::gpu::{op}: {name} must be contiguous")


def _labels(op: str, t, m: int, device) -> int:
    import torch

    if t.dtype not in (torch.int64, torch.int32):
        raise InvalidArgument(f"knng::gpu::{op}: labels must be int64 or int32")
    _vector(op, "labels", t, m, t.dtype, device)
    return int(t.dtype == torch.int64)


def _scope(device, stream):
    """Allocations and launches on the tensors' device and the call's stream."""
    import torch

    if stream is not None:
        return torch.cuda.stream(stream)
    if device.index is not None and device.index != torch.cuda.current_device():
        return torch.cuda.device(device)
    return nullcontext()


def _run(name: str, args, device, workspace) -> None:
    """Inside :func:`_scope`."""
    import torch

    lib = gpu_lib()
    ref = ctypes.byref(args)
    ws, have = None, 0
    if workspace is None:
        need = getattr(lib, f"knng_gpu_{name}_workspace_bytes")(ref)
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
    if workspace is not None:
        ws, have = workspace.data_ptr(), workspace.numel()
    check(getattr(lib, f"knng_gpu_{name}")(ref, ws, have, torch.cuda.current_stream(device).cuda_stream))


def linear(x, w, bias=None, residual=None, activation="none", out_dtype=None, out=None, save_pre=False,
           workspace=None, stream=None):
    """``act(x w^T + bias) + residual`` for x (m, k), w (n, k).

    ``activation``: "none", "relu", "gelu", "gelu_tanh" or "silu".
    ``out_dtype`` may be float32 (rows for :func:`brute_force_knn_device`)
    instead of x's. With ``save_pre`` returns ``(out, pre)``, pre = x w^T +
    bias in x's dtype, which :func:`linear_backward` takes.
    """
    import torch

    op = "linear"
    dtype = _dtype_id(op, x.dtype)
    ldx = _matrix(op, "x", x, None, None)
    m, k = x.shape
    ldw = _matrix(op, "w", w, None, k, x)
    n = w.shape[0]
    if activation not in ACTIVATIONS:
        raise InvalidArgument(f"knng::gpu::linear: unknown activation {activation!r}")
    device = x.device
    ldr = 0
    if bias is not None:
        _vector(op, "bias", bias, n, x.dtype, device)
    if residual is not None:
        ldr = _matrix(op, "residual", residual, m, n, x)
    if out is not None:
        if out_dtype is not None and out.dtype != out_dtype:
            raise InvalidArgument("knng::gpu::linear: out has another dtype than out_dtype")
        if out.device != device:
            raise InvalidArgument("knng::gpu::linear: out is on another device")
        _matrix(op, "out", out, m, n)
    with _scope(device, stream):
        if out is None:
            out = torch.empty((m, n), dtype=out_dtype or x.dtype, device=device)
        pre = torch.empty((m, n), dtype=x.dtype, device=device) if save_pre else None
        args = _native.LinearArgs(
            m, k, n, x.data_ptr(), ldx, w.data_ptr(), ldw, None if bias is None else bias.data_ptr(),
            None if residual is None else residual.data_ptr(), ldr, out.data_ptr(), _matrix(op, "out", out, m, n),
            None if pre is None else pre.data_ptr(), n, dtype, _dtype_id(op, out.dtype), ACTIVATIONS[activation])
        _run(op, args, device, workspace)
    return (out, pre) if save_pre else out


def linear_backward(dy, x, w, pre=None, activation="none", need_dx=True, need_dw=True, need_db=False,
                    workspace=None, stream=None):
    """Gradients of :func:`linear` from ``dy`` (m, n): ``(dx, dw, db)``, None
    where not needed. ``pre`` is what the forward call saved (not needed
    without an activation). The residual's gradient is ``dy``."""
    import torch

    op = "linear_backward"
    dtype = _dtype_id(op, x.dtype)
    ldx = _matrix(op, "x", x, None, None)
    m, k = x.shape
    ldw = _matrix(op, "w", w, None, k, x)
    n = w.shape[0]
    lddy = _matrix(op, "dy", dy, m, n, x)
    if activation not in ACTIVATIONS:
        raise InvalidArgument(f"knng::gpu::linear_backward: unknown activation {activation!r}")
    ldp = 0
    if pre is not None:
        ldp = _matrix(op, "pre", pre, m, n, x)
    elif activation != "none":
        raise InvalidArgument("knng::gpu::linear_backward: pre is needed with an activation")
    device = x.device
    with _scope(device, stream):
        dx = torch.empty((m, k), dtype=x.dtype, device=device) if need_dx else None
        dw = torch.empty((n, k), dtype=x.dtype, device=device) if need_dw else None
        db = torch.empty(n, dtype=x.dtype, device=device) if need_db else None
        args = _native.LinearBackwardArgs(
            m, k, n, dy.data_ptr(), lddy, x.data_ptr(), ldx, w.data_ptr(), ldw,
            None if pre is None else pre.data_ptr(), ldp, None if dx is None else dx.data_ptr(),
            None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(), dtype,
            ACTIVATIONS[activation])
        _run(op, args, device, workspace)
    return dx, dw, db


def softmax_xent(x, w, labels, scale=1.0, workspace=None, stream=None):
    """Per-row softmax cross entropy over ``scale * x w^T``: ``(loss, lse)``,
    float32 (m,). ``labels`` (m,) int64 or int32 name a row of w; a label
    outside [0, n) leaves its row out (loss 0; lse is still that row's)."""
    import torch

    op = "softmax_xent"
    dtype = _dtype_id(op, x.dtype)
    ldx = _matrix(op, "x", x, None, None)
    m, k = x.shape
    ldw = _matrix(op, "w", w, None, k, x)
    device = x.device
    i64 = _labels(op, labels, m, device)
    with _scope(device, stream):
        loss = torch.empty(m, dtype=torch.float32, device=device)
        lse = torch.empty(m, dtype=torch.float32, device=device)
        args = _native.SoftmaxXentArgs(m, k, w.shape[0], x.data_ptr(), ldx, w.data_ptr(), ldw, labels.data_ptr(),
                                       loss.data_ptr(), lse.data_ptr(), scale, dtype, i64)
        _run(op, args, device, workspace)
    return loss, lse


def softmax_xent_backward(dloss, x, w, labels, lse, scale=1.0, need_dx=True, need_dw=True, workspace=None,
                          stream=None):
    """Gradients of :func:`softmax_xent` from ``dloss`` (m,) float32 and the
    forward call's ``lse``: ``(dx, dw)`` in x's dtype, None where not needed.
    A row without a label has dx 0 and adds nothing to dw, whatever it holds."""
    import torch

    op = "softmax_xent_backward"
    dtype = _dtype_id(op, x.dtype)
    ldx = _matrix(op, "x", x, None, None)
    m, k = x.shape
    ldw = _matrix(op, "w", w, None, k, x)
    n = w.shape[0]
    device = x.device
    i64 = _labels(op, labels, m, device)
    _vector(op, "dloss", dloss, m, torch.float32, device)
    _vector(op, "lse", lse, m, torch.float32, device)
    with _scope(device, stream):
        dx = torch.empty((m, k), dtype=x.dtype, device=device) if need_dx else None
        dw = torch.empty((n, k), dtype=x.dtype, device=device) if need_dw else None
        args = _native.SoftmaxXentBackwardArgs(
            m, k, n, dloss.data_ptr(), x.data_ptr(), ldx, w.data_ptr(), ldw, labels.data_ptr(), lse.data_ptr(),
            None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(), scale, dtype, i64)
        _run(op, args, device, workspace)
    return dx, dw
