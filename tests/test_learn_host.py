"""Refusals and workspace sizes of the projection and softmax-loss entry
points: what the host decides, without a GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

import knng_gpu_b200 as kg
from knng_gpu_b200 import _native
from learn_refs import act64, linear64, linear_backward64, xent64, xent_backward64

INVALID, NOT_SUPPORTED, WORKSPACE = 1, 4, 6
A = 4096  # an aligned address that is never read: the calls below are refused before any launch


def call(name, args, ws=None, have=0):
    lib = _native.gpu_lib()
    st = getattr(lib, f"knng_gpu_{name}")(ctypes.byref(args), ws, have, None)
    return st, lib.knng_gpu_last_error().decode()


def linear_args(**kw):
    v = dict(m=300, k=64, n=200, x=A, ldx=64, w=A, ldw=64, bias=None, residual=None, ldr=0, out=A, ldo=200, pre=None,
             ldp=0, dtype=1, out_dtype=1, activation=0)
    v.update(kw)
    return _native.LinearArgs(**v)


def backward_args(**kw):
    v = dict(m=300, k=64, n=200, dy=A, lddy=200, x=A, ldx=64, w=A, ldw=64, pre=A, ldp=200, dx=A, dw=A, db=A, dtype=1,
             activation=2)
    v.update(kw)
    return _native.LinearBackwardArgs(**v)


def xent_args(**kw):
    v = dict(m=300, k=64, n=200, x=A, ldx=64, w=A, ldw=64, labels=A, loss=A, lse=A, scale=1.0, dtype=1, labels_i64=1)
    v.update(kw)
    return _native.SoftmaxXentArgs(**v)


def xent_backward_args(**kw):
    v = dict(m=300, k=64, n=200, dloss=A, x=A, ldx=64, w=A, ldw=64, labels=A, lse=A, dx=A, dw=A, scale=1.0, dtype=1,
             labels_i64=1)
    v.update(kw)
    return _native.SoftmaxXentBackwardArgs(**v)


MAKE = {"linear": linear_args, "linear_backward": backward_args, "softmax_xent": xent_args,
        "softmax_xent_backward": xent_backward_args}


@pytest.mark.parametrize("name", MAKE)
def test_sizes_and_types_are_checked(name):
    make = MAKE[name]
    for kw, status, words in [
        (dict(k=0), INVALID, "k must be > 0"),
        (dict(n=0), INVALID, "n must be > 0"),
        (dict(dtype=3), INVALID, "unknown dtype"),
        (dict(dtype=-1), INVALID, "unknown dtype"),
        (dict(n=1 << 31), NOT_SUPPORTED, "2^31"),
        (dict(m=1 << 31), NOT_SUPPORTED, "2^31"),
        (dict(k=(1 << 20) + 1), NOT_SUPPORTED, "2^20"),
        (dict(ldx=63), INVALID, "row stride of x"),
        (dict(ldw=63), INVALID, "row stride of w"),
        (dict(x=None), INVALID, "x is NULL"),
        (dict(w=None), INVALID, "w is NULL"),
        (dict(x=A + 1), INVALID, "not aligned to its elements"),
    ]:
        st, msg = call(name, make(**kw))
        assert st == status and words in msg and msg.startswith(f"knng::gpu::{name}"), (kw, st, msg)
    lib = _native.gpu_lib()
    assert getattr(lib, f"knng_gpu_{name}")(None, None, 0, None) == INVALID
    assert getattr(lib, f"knng_gpu_{name}_workspace_bytes")(None) == 0


def test_arguments_of_one_operator_are_checked():
    for name, args, words in [
        ("linear", linear_args(out_dtype=2), "out_dtype"),
        ("linear", linear_args(activation=5), "unknown activation"),
        ("linear", linear_args(out=None), "out is NULL"),
        ("linear", linear_args(ldo=199), "row stride of out"),
        ("linear", linear_args(residual=A, ldr=10), "row stride of residual"),
        ("linear", linear_args(pre=A, ldp=10), "row stride of pre"),
        ("linear_backward", backward_args(pre=None), "pre is NULL"),
        ("linear_backward", backward_args(activation=-1), "unknown activation"),
        ("linear_backward", backward_args(lddy=10), "row stride of dy"),
        ("softmax_xent", xent_args(scale=0.0), "scale"),
        ("softmax_xent", xent_args(scale=float("inf")), "scale"),
        ("softmax_xent", xent_args(labels=None), "labels"),
        ("softmax_xent_backward", xent_backward_args(scale=-2.0), "scale"),
        ("softmax_xent_backward", xent_backward_args(dloss=None), "dloss"),
    ]:
        st, msg = call(name, args)
        assert st == INVALID and words in msg, (name, words, st, msg)


@pytest.mark.parametrize("name", MAKE)
def test_workspace_is_checked(name):
    lib = _native.gpu_lib()
    args = MAKE[name](dtype=0, **({"out_dtype": 0} if name == "linear" else {}))
    need = getattr(lib, f"knng_gpu_{name}_workspace_bytes")(ctypes.byref(args))
    assert need > 0
    st, msg = call(name, args, A, need - 1)
    assert st == WORKSPACE and str(need) in msg
    st, msg = call(name, args, None, need)
    assert st == WORKSPACE
    st, msg = call(name, args, A + 16, need)
    assert st == INVALID and "256-byte" in msg


def test_an_aligned_product_needs_no_workspace():
    lib = _native.gpu_lib()
    args = linear_args(m=65536, k=256, n=1024, ldx=256, ldw=256, ldo=1024)
    assert lib.knng_gpu_linear_workspace_bytes(ctypes.byref(args)) == 0
    odd = linear_args(m=65536, k=255, n=1024, ldx=255, ldw=255, ldo=1024)
    # Rows of 255 values are staged at a pitch of 256.
    assert lib.knng_gpu_linear_workspace_bytes(ctypes.byref(odd)) == (65536 + 1024) * 512


def test_an_empty_batch_needs_nothing():
    for name in ("linear", "softmax_xent"):
        assert call(name, MAKE[name](m=0, x=None))[0] == 0


def test_scores_are_never_kept():
    lib = _native.gpu_lib()
    m, n = 8192, 1000000
    fwd = lib.knng_gpu_softmax_xent_workspace_bytes(ctypes.byref(xent_args(m=m, n=n)))
    bwd = lib.knng_gpu_softmax_xent_backward_workspace_bytes(ctypes.byref(xent_backward_args(m=m, n=n)))
    assert fwd < m * n * 2 / 100 and bwd < m * n * 2 / 50


def test_cpu_tensors_are_refused():
    x, w = torch.zeros((4, 8)), torch.zeros((6, 8))
    y, f = torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    for fn in (lambda: kg.linear(x, w), lambda: kg.linear_backward(torch.zeros((4, 6)), x, w),
               lambda: kg.softmax_xent(x, w, y), lambda: kg.softmax_xent_backward(f, x, w, y, f)):
        with pytest.raises(kg.InvalidArgument, match="CUDA tensor"):
            fn()


def test_definitions_agree_with_autograd():
    """The 64-bit formulas the GPU tests use, against torch's own derivatives."""
    g = torch.Generator().manual_seed(1)
    x, w, b = (torch.randn(s, generator=g, dtype=torch.float32) for s in ((9, 7), (5, 7), (5,)))
    dy = torch.randn((9, 5), generator=g)
    for act in ("none", "relu", "gelu", "gelu_tanh", "silu"):
        xd, wd, bd = (t.double().requires_grad_() for t in (x, w, b))
        z = xd @ wd.t() + bd
        (act64(z, act)[0] * dy.double()).sum().backward()
        got = linear_backward64(dy, x, w, z.detach(), act)
        for (v, bound), want in zip(got, (xd.grad, wd.grad, bd.grad)):
            assert torch.allclose(v, want, atol=1e-12) and (bound > 0).all()
    (y, _), (z, _) = linear64(x, w, b, dy, "silu", torch.float32)
    ref = torch.nn.functional.silu(torch.nn.functional.linear(x.double(), w.double(), b.double()))
    assert torch.allclose(y, ref + dy.double(), atol=1e-12)
    labels = torch.tensor([0, 4, -1, 2, 5, 1, 3, 3, -100])
    keep = (labels >= 0) & (labels < 5)
    xd, wd = x.double().requires_grad_(), w.double().requires_grad_()
    rows = torch.nn.functional.cross_entropy(2.5 * xd @ wd.t(), torch.where(keep, labels, -1), ignore_index=-1,
                                             reduction="none")
    dloss = torch.rand(9, generator=g)
    (rows * dloss.double()).sum().backward()
    (loss, _), (lse, _), _, _ = xent64(x, w, labels, 2.5)
    assert torch.allclose(loss, rows.detach(), atol=1e-12)
    (dx, _), (dw, _) = xent_backward64(dloss, x, w, labels, lse, 2.5)
    # lse reaches the gradient in fp32 in use; here it is the 64-bit one.
    assert torch.allclose(dx, xd.grad, atol=1e-12) and torch.allclose(dw, wd.grad, atol=1e-12)


def test_argument_formats_match_the_structures():
    from knng_gpu_b200 import learn

    for op, args in ((learn._LINEAR, _native.LinearArgs), (learn._LINEAR_BACKWARD, _native.LinearBackwardArgs),
                     (learn._XENT, _native.SoftmaxXentArgs), (learn._XENT_BACKWARD, _native.SoftmaxXentBackwardArgs)):
        values = [1.5 if t is ctypes.c_float else i + 1 for i, (_, t) in enumerate(args._fields_)]
        assert op.fields.pack(*values) == bytes(args(*values)), op.name
