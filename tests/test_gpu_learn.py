"""linear, softmax_xent and their gradients on the GPU against their 64-bit
definitions (learn_refs.py derives the bounds)."""
from __future__ import annotations

import pytest
import torch

import knng_gpu_b200 as kg
from learn_refs import act64, linear64, linear_backward64, xent64, xent_backward64

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def rows(gen, m, k, dtype, pad=0, scale=1.0, shift=0):
    """(m, k) rows of a wider table whose other values are NaN; `shift`
    elements move the first row off its alignment."""
    t = torch.full((m * (k + pad) + shift,), float("nan"), device="cuda", dtype=dtype)
    v = t[shift:].view(m, k + pad)[:, :k]
    v.copy_((torch.randn((m, k), generator=gen, device="cuda") * scale).to(dtype))
    return v


def make_gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def check(got, want, bound, what):
    assert got.shape == want.shape, what
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((off / bound).nan_to_num(float("inf")).max()))


# Tiles are 128 or 256 wide, K blocks 64, boxes 32 and 64: each size sits at, before or behind one of these.
LINEAR = [
    (1, 1, 1), (1, 960, 1024), (2, 17, 33), (31, 64, 128), (33, 785, 300), (128, 128, 128), (129, 65, 127),
    (256, 192, 512), (257, 1000, 255), (777, 300, 1025), (2049, 784, 1024), (5000, 130, 16),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,k,n", LINEAR)
def test_linear(cuda_ok, m, k, n, dtype):
    i = LINEAR.index((m, k, n))
    act, pad, shift = ACTS[i % 5], (0, 3, 8)[i % 3], (0, 0, 1)[i % 3]
    g = make_gen(i)
    x, w = rows(g, m, k, dtype, pad, shift=shift), rows(g, n, k, dtype, (8, 0)[i % 2], k ** -0.5)
    bias = rows(g, 1, n, dtype)[0] if i % 4 else None
    res = rows(g, m, n, dtype, pad) if i % 2 else None
    for out_dtype in dict.fromkeys((dtype, F32)):
        (y, by), (z, bz) = linear64(x, w, bias, res, act, out_dtype)
        out, pre = kg.linear(x, w, bias, res, act, out_dtype=out_dtype, save_pre=True)
        assert out.dtype == out_dtype and pre.dtype == dtype
        check(out, y, by, "out")
        check(pre, z, bz, "pre")
    check(kg.linear(x, w, bias, res, act), *linear64(x, w, bias, res, act, dtype)[0], "out without pre")


def test_linear_into_strided_out(cuda_ok):
    g = make_gen(50)
    x, w = rows(g, 300, 96, BF16), rows(g, 200, 96, BF16)
    for wide in (201, 208):
        table = torch.full((300, wide), 7.0, device="cuda", dtype=BF16)
        got = kg.linear(x, w, activation="relu", out=table[:, :200])
        assert got.data_ptr() == table.data_ptr()
        check(table[:, :200], *linear64(x, w, None, None, "relu", BF16)[0], "out")
        assert (table[:, 200:] == 7.0).all()


@pytest.mark.parametrize("act", ACTS)
def test_activation_over_its_range(cuda_ok, act):
    # One row per value: x w^T is the value itself.
    v = torch.linspace(-30, 30, 4001, device="cuda")
    x = torch.stack([v, torch.zeros_like(v)], 1).contiguous()
    w = torch.tensor([[1.0, 0.0]], device="cuda")
    out = kg.linear(x, w, activation=act)
    want = act64(v.double()[:, None], act)[0]
    check(out, want, 2.0 ** -20 * v.double().abs()[:, None] + 2.0 ** -23, act)
    dy = torch.ones_like(out)
    dx, _, _ = kg.linear_backward(dy, x, w, pre=v[:, None].contiguous(), activation=act, need_dw=False)
    check(dx[:, :1], act64(v.double()[:, None], act)[1], torch.full_like(want, 2.0 ** -18), act)


def test_linear_infinity_and_nan_stay_in_their_row(cuda_ok):
    g = make_gen(51)
    for dtype in (BF16, F16):
        x, w = rows(g, 40, 64, dtype), rows(g, 50, 64, dtype)
        clean = kg.linear(x, w, activation="silu")
        x[7, 3], x[30, 0] = float("nan"), float("inf")
        got = kg.linear(x, w, activation="silu")
        keep = torch.ones(40, dtype=torch.bool, device="cuda")
        keep[[7, 30]] = False
        assert torch.equal(got[keep], clean[keep])
        assert got[7].isnan().all() and not got[30].isfinite().all()


BACKWARD = [(1, 8, 8), (3, 785, 300), (130, 17, 1000), (500, 128, 129), (1537, 960, 300), (4100, 784, 520), (20000, 40, 24)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,k,n", BACKWARD)
def test_linear_backward(cuda_ok, m, k, n, dtype):
    i = BACKWARD.index((m, k, n))
    g = make_gen(100 + i)
    pad = (0, 3, 8)[i % 3]
    x, w, dy = rows(g, m, k, dtype, pad), rows(g, n, k, dtype, 0, k ** -0.5), rows(g, m, n, dtype, pad, 0.1)
    pre = rows(g, m, n, dtype, pad)
    for act in ("none", ACTS[1 + i % 4]):
        want = linear_backward64(dy, x, w, pre, act)
        got = kg.linear_backward(dy, x, w, pre=None if act == "none" else pre, activation=act, need_db=True)
        for a, (v, b), name in zip(got, want, ("dx", "dw", "db")):
            check(a, v, b, (name, act))
    dx, dw, db = kg.linear_backward(dy, x, w, need_dx=False)
    assert dx is None and db is None
    check(dw, *linear_backward64(dy, x, w, None, "none")[1], "dw alone")
    dx, dw, db = kg.linear_backward(dy, x, w, need_dx=False, need_dw=False, need_db=True)
    assert dx is None and dw is None
    check(db, *linear_backward64(dy, x, w, None, "none")[2], "db alone")


def test_linear_gradient_against_differences(cuda_ok):
    g = make_gen(150)
    x, w, b = rows(g, 24, 40, F32), rows(g, 30, 40, F32, scale=0.2), rows(g, 1, 30, F32)[0]
    dy = rows(g, 24, 30, F32)
    for act in ("gelu", "gelu_tanh", "silu"):
        _, pre = kg.linear(x, w, b, activation=act, save_pre=True)
        grads = kg.linear_backward(dy, x, w, pre=pre, activation=act, need_db=True)
        for which in range(3):
            base = (x, w, b)
            step = rows(g, 1, base[which].numel(), F32)[0].view_as(base[which])
            h = 2.0 ** -7
            f = []
            for sign in (1, -1):
                moved = list(base)
                moved[which] = base[which] + sign * h * step
                f.append((kg.linear(*moved, activation=act).double() * dy.double()).sum())
            diff = (f[0] - f[1]) / (2 * h)
            want = (grads[which].double() * step.double()).sum()
            # h^2 / 6 times a third derivative along the step, plus the values' rounding over h.
            size = (dy.abs().double().sum() * float(step.abs().max()))
            assert abs(float(diff - want)) <= float(size) * (h * h * 8 + 2.0 ** -20 / h), (act, which)


XENT = [(1, 1, 1), (1, 128, 10000), (2, 17, 3), (33, 785, 300), (128, 64, 129), (129, 960, 1000), (256, 128, 4096),
        (300, 300, 30011), (1000, 128, 777), (2500, 24, 5000)]


def xent_case(m, k, n, dtype, seed, pad=0):
    g = make_gen(seed)
    w = rows(g, n, k, dtype, pad)
    w.copy_(torch.nn.functional.normalize(w.float(), dim=1).to(dtype))
    labels = torch.randint(0, n, (m,), generator=g, device="cuda")
    x = rows(g, m, k, dtype, pad)
    x.copy_(torch.nn.functional.normalize(w[labels].float() + x.float() * k ** -0.5, dim=1).to(dtype))
    return x, w, labels


def some_ignored(labels, n):
    labels = labels.clone()
    labels[1::3] = -1
    labels[2::7] = n
    labels[5::11] = -100
    return labels


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,k,n", XENT)
def test_softmax_xent_and_gradient(cuda_ok, m, k, n, dtype):
    i = XENT.index((m, k, n))
    x, w, labels = xent_case(m, k, n, dtype, 200 + i, (0, 3, 8)[i % 3])
    scale = (1.0, 20.0, 7.5)[i % 3]
    if i % 2:
        labels = some_ignored(labels, n)
    if i % 4 == 1:
        labels = labels.int()
    (loss, bl), (lse, be), _, _ = xent64(x, w, labels, scale)
    got_loss, got_lse = kg.softmax_xent(x, w, labels, scale)
    check(got_loss, loss, bl, "loss")
    check(got_lse, lse, be, "lse")
    g = make_gen(300 + i)
    dloss = torch.randn(m, generator=g, device="cuda") / m
    lse32 = lse.float()
    (dx, bx), (dw, bw) = xent_backward64(dloss, x, w, labels, lse32, scale)
    got_dx, got_dw = kg.softmax_xent_backward(dloss, x, w, labels, lse32, scale)
    check(got_dx, dx, bx, "dx")
    check(got_dw, dw, bw, "dw")
    only, none = kg.softmax_xent_backward(dloss, x, w, labels, lse32, scale, need_dw=False)
    assert none is None and torch.equal(only, got_dx)
    none, only = kg.softmax_xent_backward(dloss, x, w, labels, lse32, scale, need_dx=False)
    assert none is None and torch.equal(only, got_dw)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_softmax_xent_gradient_in_several_pieces(cuda_ok, dtype):
    # Enough rows that w is taken in pieces, the last one narrower.
    x, w, labels = xent_case(20000, 24, 5001, dtype, 400)
    labels = some_ignored(labels, 5001)
    dloss = torch.full((20000,), 1.0 / 20000, device="cuda")
    lse = xent64(x, w, labels, 9.0)[1][0].float()
    got = kg.softmax_xent_backward(dloss, x, w, labels, lse, 9.0)
    for a, (v, b), name in zip(got, xent_backward64(dloss, x, w, labels, lse, 9.0), ("dx", "dw")):
        check(a, v, b, name)


def test_fp32_results_are_fp32_good(cuda_ok):
    # In the norm, not only within worst-case bounds: long sums stay at fp32's own error.
    g = make_gen(450)
    x, w, dy = rows(g, 30000, 300, F32), rows(g, 200, 300, F32), rows(g, 30000, 200, F32)
    got = kg.linear_backward(dy, x, w, need_db=True)
    for a, (v, _), name in zip(got, linear_backward64(dy, x, w, None, "none"), ("dx", "dw", "db")):
        assert float((a.double() - v).norm() / v.norm()) < 1e-6, name
    xs, ws, labels = xent_case(500, 960, 3000, F16, 451)
    (loss, _), (lse, _), _, _ = xent64(xs, ws, labels, 16.0)
    got = kg.softmax_xent(xs, ws, labels, 16.0)
    assert float((got[0].double() - loss).norm() / loss.norm()) < 4e-6
    assert float((got[1].double() - lse).norm() / lse.norm()) < 1e-6


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_without_label_may_hold_anything(cuda_ok, dtype):
    x, w, labels = xent_case(200, 48, 500, dtype, 500)
    labels[::4] = -1
    dloss = torch.full((200,), 0.01, device="cuda")
    loss, lse = kg.softmax_xent(x, w, labels, 5.0)
    dx, dw = kg.softmax_xent_backward(dloss, x, w, labels, lse, 5.0)
    x[::8], x[4::8] = float("nan"), float("inf")
    dloss[::4] = float("nan")
    loss2, lse2 = kg.softmax_xent(x, w, labels, 5.0)
    dx2, dw2 = kg.softmax_xent_backward(dloss, x, w, labels, lse2, 5.0)
    assert torch.equal(loss, loss2) and torch.equal(dx, dx2) and torch.equal(dw, dw2)
    assert (loss2[::4] == 0).all() and (dx2[::4] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_no_row_has_a_label(cuda_ok, dtype):
    x, w, labels = xent_case(70, 32, 90, dtype, 501)
    labels.fill_(-1)
    loss, lse = kg.softmax_xent(x, w, labels, 5.0)
    assert (loss == 0).all() and lse.isfinite().all()
    dx, dw = kg.softmax_xent_backward(torch.ones(70, device="cuda"), x, w, labels, lse, 5.0)
    assert (dx == 0).all() and (dw == 0).all()


def test_masked_classes_and_large_scores(cuda_ok):
    # Classes at -inf have no weight; scores far beyond exp's range stay finite.
    x = torch.ones((3, 16), device="cuda", dtype=BF16)
    w = torch.zeros((300, 16), device="cuda", dtype=BF16)
    w[1::2] = float("-inf")
    labels = torch.tensor([0, 2, 298], device="cuda")
    loss, lse = kg.softmax_xent(x, w, labels, 2.0)
    assert torch.allclose(lse.double(), torch.full((3,), 150.0, device="cuda", dtype=torch.float64).log(), atol=1e-5)
    assert torch.allclose(loss, lse)
    w.fill_(float("-inf"))
    loss, lse = kg.softmax_xent(x, w, torch.full_like(labels, -1), 2.0)
    assert (lse == float("-inf")).all() and (loss == 0).all()
    w.zero_()
    w[7] = 1000.0
    loss, lse = kg.softmax_xent(x, w, torch.tensor([7, 7, 8], device="cuda"), 100.0)
    assert loss[:2].abs().max() == 0 and float(loss[2]) == pytest.approx(1.6e6) and float(lse[0]) == pytest.approx(1.6e6)


def test_xent_gradient_against_differences(cuda_ok):
    x, w, labels = xent_case(20, 24, 130, F32, 502)
    labels[3] = -1
    g = make_gen(503)
    dloss = torch.rand(20, generator=g, device="cuda")
    _, lse = kg.softmax_xent(x, w, labels, 3.0)
    grads = kg.softmax_xent_backward(dloss, x, w, labels, lse, 3.0)
    for which in range(2):
        base = (x, w)
        step = torch.randn(base[which].shape, generator=g, device="cuda")
        h, f = 2.0 ** -8, []
        for sign in (1, -1):
            moved = list(base)
            moved[which] = base[which] + sign * h * step
            f.append((kg.softmax_xent(*moved, labels, 3.0)[0].double() * dloss.double()).sum())
        want = (grads[which].double() * step.double()).sum()
        # Third derivative of a row's loss along the step: at most 6 (scale |x||step| or |w||step|)^3.
        reach = (3.0 * float(step.norm(dim=1).max()) * 1.0) ** 3
        tol = float(dloss.sum()) * (h * h * reach + 2.0 ** -19 / h)
        assert abs(float((f[0] - f[1]) / (2 * h) - want)) <= tol


def test_calls_repeat_bit_for_bit(cuda_ok):
    x, w, labels = xent_case(3000, 200, 9000, BF16, 504)
    dloss = torch.rand(3000, device="cuda")
    _, lse = kg.softmax_xent(x, w, labels, 9.0)
    one = (*kg.softmax_xent(x, w, labels, 9.0), *kg.softmax_xent_backward(dloss, x, w, labels, lse, 9.0),
           *kg.linear_backward(x, x[:, :100], w[:200, :100].contiguous(), need_db=True))
    two = (*kg.softmax_xent(x, w, labels, 9.0), *kg.softmax_xent_backward(dloss, x, w, labels, lse, 9.0),
           *kg.linear_backward(x, x[:, :100], w[:200, :100].contiguous(), need_db=True))
    for a, b in zip(one, two):
        assert torch.equal(a, b)


def test_empty_batches(cuda_ok):
    w = torch.randn((50, 16), device="cuda", dtype=BF16)
    x = torch.empty((0, 16), device="cuda", dtype=BF16)
    out, pre = kg.linear(x, w, save_pre=True)
    assert out.shape == (0, 50) and pre.shape == (0, 50)
    dx, dw, db = kg.linear_backward(out, x, w, pre=pre, activation="gelu", need_db=True)
    assert dx.shape == (0, 16) and (dw == 0).all() and (db == 0).all()
    labels = torch.empty(0, device="cuda", dtype=torch.int64)
    loss, lse = kg.softmax_xent(x, w, labels)
    dx, dw = kg.softmax_xent_backward(loss, x, w, labels, lse)
    assert loss.shape == (0,) and dx.shape == (0, 16) and (dw == 0).all()


def test_another_stream_and_own_workspace(cuda_ok):
    import ctypes

    from knng_gpu_b200 import _native

    x, w, labels = xent_case(400, 128, 1000, BF16, 505)
    want = kg.softmax_xent(x, w, labels, 4.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = kg.softmax_xent(x, w, labels, 4.0, stream=side)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    args = _native.SoftmaxXentArgs(400, 128, 1000, x.data_ptr(), 128, w.data_ptr(), 128, labels.data_ptr(),
                                   got[0].data_ptr(), got[1].data_ptr(), 4.0, 1, 1)
    need = _native.gpu_lib().knng_gpu_softmax_xent_workspace_bytes(ctypes.byref(args))
    ws = torch.full((need + 64,), 255, device="cuda", dtype=torch.uint8)
    got = kg.softmax_xent(x, w, labels, 4.0, workspace=ws[:need])
    assert torch.equal(got[0], want[0]) and (ws[need:] == 255).all()
    with pytest.raises(kg.KnngGpuError, match="WORKSPACE_TOO_SMALL"):
        kg.softmax_xent(x, w, labels, 4.0, workspace=ws[: need - 1])


def test_operators_in_a_graph(cuda_ok):
    x, w, labels = xent_case(300, 64, 900, BF16, 506)
    dloss = torch.full((300,), 0.01, device="cuda")

    def step():
        loss, lse = kg.softmax_xent(x, w, labels, 4.0)
        return (loss, *kg.softmax_xent_backward(dloss, x, w, labels, lse, 4.0))

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_refusals_on_the_gpu(cuda_ok):
    x = torch.zeros((4, 8), device="cuda", dtype=BF16)
    w = torch.zeros((6, 8), device="cuda", dtype=BF16)
    y = torch.zeros(4, device="cuda", dtype=torch.int64)
    f = torch.zeros(4, device="cuda")
    bad = [
        lambda: kg.linear(x, w.float()),
        lambda: kg.linear(x, w[:, :7]),
        lambda: kg.linear(x.double(), w.double()),
        lambda: kg.linear(x[0], w),
        lambda: kg.linear(x.t(), w[:, :4]),
        lambda: kg.linear(x[:1].expand(4, 8), w),
        lambda: kg.linear(x, w, bias=torch.zeros(5, device="cuda", dtype=BF16)),
        lambda: kg.linear(x, w, residual=torch.zeros((4, 5), device="cuda", dtype=BF16)),
        lambda: kg.linear(x, w, activation="tanh"),
        lambda: kg.linear(x, w, out_dtype=F16),
        lambda: kg.linear(x, w, out=torch.zeros((4, 6), dtype=BF16)),
        lambda: kg.linear(x[:, :0], w[:, :0]),
        lambda: kg.linear(x, w[:0]),
        lambda: kg.linear_backward(x[:, :6], x, w, activation="gelu"),
        lambda: kg.linear_backward(x, x, w),
        lambda: kg.softmax_xent(x, w, y.float()),
        lambda: kg.softmax_xent(x, w, y[:3]),
        lambda: kg.softmax_xent(x, w, y, scale=0.0),
        lambda: kg.softmax_xent(x, w, y, scale=float("nan")),
        lambda: kg.softmax_xent(x, w[:0], y),
        lambda: kg.softmax_xent_backward(f.half(), x, w, y, f),
        lambda: kg.softmax_xent_backward(f, x, w, y, f[:2]),
        lambda: kg.softmax_xent_backward(f, x, w, y, f, scale=-1.0),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(kg.InvalidArgument):
            call()
            pytest.fail(f"call {i} was not refused")


def test_withheld_arrival_times_out_and_results_stay_right(cuda_ok):
    # A wait of ~10 ms runs out, every role unwinds, the status says so once, and the context goes on.
    from knng_gpu_b200 import _native

    lib = _native.gpu_lib()
    assert lib.knng_gpu_selftest_product_wait(20_000_000) == 3
    assert b"bounded device wait" in lib.knng_gpu_last_error()
    g = make_gen(60)
    for m in (100, 3000):
        x, w = rows(g, m, 256, BF16), rows(g, 512, 256, BF16)
        check(kg.linear(x, w), *linear64(x, w, None, None, "none", BF16)[0], "out")


@pytest.mark.parametrize("m", [3, 300])  # the kernel for few rows, and the product
def test_nan_scores_reach_loss_and_lse_of_their_row_only(cuda_ok, m):
    x, w, labels = xent_case(m, 64, 700, BF16, 507)
    labels[1] = -1
    clean = kg.softmax_xent(x, w, labels, 6.0)
    x[:2] = float("nan")
    loss, lse = kg.softmax_xent(x, w, labels, 6.0)
    assert loss[0].isnan() and lse[:2].isnan().all() and loss[1] == 0
    assert torch.equal(loss[2:], clean[0][2:]) and torch.equal(lse[2:], clean[1][2:])


def test_inputs_may_be_dropped_after_a_call_on_another_stream(cuda_ok):
    side = torch.cuda.Stream()
    g = make_gen(508)
    w = rows(g, 512, 512, BF16)
    want, got = [], []
    for i in range(20):
        x = rows(g, 4096, 512, BF16)
        want.append(kg.linear(x, w))
        side.wait_stream(torch.cuda.current_stream())
        got.append(kg.linear(x, w, stream=side))
        del x
        torch.zeros((4096, 512), device="cuda", dtype=BF16)  # would take x's memory at once
    side.synchronize()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_merged_products_with_outputs_of_two_widths(cuda_ok):
    # Short gradients run dx (fp32 pieces) and dw (16-bit rows) in one launch, through the same store boxes.
    for seed in range(8):
        x, w, labels = xent_case(700 + 17 * seed, 128, 9000, BF16, 520 + seed)
        dloss = torch.full((x.shape[0],), 1e-3, device="cuda")
        lse = xent64(x, w, labels, 9.0)[1][0].float()
        got = kg.softmax_xent_backward(dloss, x, w, labels, lse, 9.0)
        for a, (v, b), name in zip(got, xent_backward64(dloss, x, w, labels, lse, 9.0), ("dx", "dw")):
            check(a, v, b, (name, seed))


def test_offsets_beyond_32_bits(cuda_ok):
    # Matrices of more than 2^31 elements: the last rows have to be right.
    g = make_gen(700)
    m, k, n = 2_200_000, 1000, 40
    x = torch.empty((m, k), device="cuda", dtype=BF16)
    x.normal_(generator=g)
    w = rows(g, n, k, BF16, 0, k ** -0.5)
    tail = slice(m - 300, m)
    out = kg.linear(x, w, activation="relu")
    check(out[tail], *linear64(x[tail], w, None, None, "relu", BF16)[0], "linear")
    dy = rows(g, m, n, BF16, 0, 0.1)
    dx, _, _ = kg.linear_backward(dy, x, w, need_dw=False)
    check(dx[tail], *linear_backward64(dy[tail], x[tail], w, None, "none")[0], "dx")
    del out, dy, dx
    # The same matrix as the base rows of the loss.
    labels = torch.tensor([0, m - 1, m - 2, -1], device="cuda")
    few = rows(g, 4, k, BF16, 0, 0.05)
    loss, lse = kg.softmax_xent(few, x, labels, 0.5)
    z = 0.5 * torch.cat([few.double() @ part.double().t() for part in x.split(200_000)], 1)
    want = torch.logsumexp(z, 1)
    assert torch.allclose(lse.double(), want, atol=2e-5, rtol=0)
    at = labels.clamp_min(0)[:, None]
    assert torch.allclose(loss.double(), (want - z.gather(1, at)[:, 0]) * (labels >= 0), atol=4e-5, rtol=0)
    dloss = torch.ones(4, device="cuda")
    _, dw = kg.softmax_xent_backward(dloss, few, x, labels, lse, 0.5, need_dx=False)
    p = torch.exp(z - lse.double()[:, None])
    p[torch.arange(3), labels[:3]] -= 1.0
    p[3] = 0
    want = 0.5 * p[:, tail].t() @ few.double()
    # Rounding of g (bf16, 2^-8) and of the result, and the scores' own error.
    bound = 2.0 ** -7 * (0.5 * p[:, tail].abs().t() @ few.double().abs()) + 2.0 ** -8 * want.abs()
    check(dw[tail], want, bound + 1e-12, "dw")
