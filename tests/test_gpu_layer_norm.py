"""clpk_layer_norm and clpk_layer_norm_backward against 64 bits, element by element."""
import ctypes as C

import pytest
import torch

from clpeak_b200 import native as N
from tests import block_util as B
from tests import ff_util as F

pytestmark = pytest.mark.gpu

TYPES = [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"), ("f32", "f32")]
# one element, inside a vector, around the widths that a warp and CTAs of each size take, and longer than registers hold
WIDTHS = [1, 2, 7, 8, 33, 255, 256, 257, 512, 513, 1000, 1024, 1025, 2048, 2049, 4096, 4099, 8192, 8193, 16384, 16391, 32768, 32771]


def values(rows, cols, seed, mean=0.0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    x = torch.randn(rows, cols, generator=gen, device="cuda") * torch.exp(torch.randn(rows, 1, generator=gen, device="cuda"))
    x[:, ::61] *= 20
    return x + mean


def weights(d, dtype, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    w = torch.randn(2, d, generator=gen, device="cuda").to(F.TORCH[dtype])
    return w[0].clone(), w[1].clone()


def forward(K, x, dtype, wdtype, weight, bias, eps=1e-5, pad=0, y=None):
    m, d = x.shape
    y = F.matrix(m, d, dtype, pad) if y is None else y
    mean, rstd = (torch.full((m + 1,), 77.0, device="cuda") for _ in range(2))
    K.clpk_layer_norm(C.byref(B.norm_args(x, y, weight, bias, mean, rstd, eps, dtype, wdtype)), F.stream())
    assert mean[m] == 77 and rstd[m] == 77
    return y, mean[:m], rstd[:m]


def backward(K, x, dy, mean, rstd, weight, dtype, wdtype, pad=0, want=("dx", "dweight", "dbias"), workspace=None):
    m, d = x.shape
    dx = F.matrix(m, d, dtype, pad) if "dx" in want else None
    wide = {name: torch.full((d + 8,), 77, dtype=F.TORCH[wdtype], device="cuda") if name in want else None for name in ("dweight", "dbias")}
    workspace = B.norm_workspace(K, m, d) if workspace is None else workspace
    K.clpk_layer_norm_backward(C.byref(B.norm_backward_args(x, dy, mean, rstd, weight, dx, wide["dweight"], wide["dbias"], workspace, dtype, wdtype)), F.stream())
    assert dx is None or F.untouched(dx)
    assert all(t is None or bool((t[d:] == 77).all()) for t in wide.values())
    return [dx] + [None if t is None else t[:d] for t in wide.values()]


def check_all(K, x, dy, weight, bias, dtype, wdtype, pad=0, eps=1e-5):
    y, mean, rstd = forward(K, x, dtype, wdtype, weight, bias, eps, pad)
    assert F.untouched(y)
    for got, (want, allowed), name in zip((y, mean, rstd), B.norm64(x, weight, bias, eps, dtype), ("y", "mean", "rstd")):
        F.check(got, want, allowed, name)
    got = backward(K, x, dy, mean, rstd, weight, dtype, wdtype, pad)
    for t, (want, allowed), name in zip(got, B.norm_backward64(x, dy, mean, rstd, weight, dtype, wdtype), ("dx", "dweight", "dbias")):
        F.check(t, want, allowed, name)


@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("d", WIDTHS)
def test_every_width(K, cuda, dtype, wdtype, d):
    for m in (1, 5, 37):
        x, dy = F.filled(values(m, d, d), dtype, pad=m % 3), F.filled(values(m, d, d + 1), dtype, pad=m % 2)
        weight, bias = weights(d, wdtype, d)
        check_all(K, x, dy, weight, bias, dtype, wdtype, pad=m // 5)


@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("m,d", [(4800, 200), (1001, 1000), (700, 1500), (301, 4096), (1500, 72), (200, 9000)])
def test_many_rows(K, cuda, dtype, wdtype, m, d):
    """More rows than CTAs take at a time."""
    weight, bias = weights(d, wdtype, 2)
    check_all(K, F.filled(values(m, d, 3), dtype), F.filled(values(m, d, 4), dtype), weight, bias, dtype, wdtype)


@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("offset,pitch,d", [(1, 67, 64), (0, 1003, 1001), (3, 4111, 4100), (5, 20011, 20001)])
def test_any_address_and_pitch(K, cuda, dtype, wdtype, offset, pitch, d):
    m, t = 19, F.TORCH[dtype]
    rows = lambda seed: torch.as_strided(values(1, offset + m * pitch, seed).flatten().to(t), (m, d), (pitch, 1), offset)     # noqa: E731
    weight, bias = weights(d + 1, wdtype, 5)
    weight, bias = weight[1:], bias[1:]
    x, dy = rows(6), rows(7)
    flat = torch.full((offset + m * pitch + 9,), 77, dtype=t, device="cuda")
    y = torch.as_strided(flat, (m, d), (pitch, 1), offset)
    got = forward(K, x, dtype, wdtype, weight, bias, y=y)
    for v, (want, allowed) in zip(got, B.norm64(x, weight, bias, 1e-5, dtype)):
        F.check(v, want, allowed)
    left = torch.ones_like(flat, dtype=torch.bool)
    torch.as_strided(left, (m, d), (pitch, 1), offset).fill_(False)
    assert bool((flat[left] == 77).all())
    for v, (want, allowed) in zip(backward(K, x, dy, got[1], got[2], weight, dtype, wdtype), B.norm_backward64(x, dy, got[1], got[2], weight, dtype, wdtype)):
        F.check(v, want, allowed)


@pytest.mark.parametrize("d", [40, 700, 5000, 40000])
def test_without_weights_and_one_result_at_a_time(K, cuda, d):
    m = 23
    x, dy = F.filled(values(m, d, 8), "bf16"), F.filled(values(m, d, 9), "bf16")
    check_all(K, x, dy, None, None, "bf16", "bf16")
    weight, bias = weights(d, "bf16", 9)
    _, mean, rstd = forward(K, x, "bf16", "bf16", weight, None)
    whole = backward(K, x, dy, mean, rstd, weight, "bf16", "bf16")
    for i, name in enumerate(("dx", "dweight", "dbias")):
        one = backward(K, x, dy, mean, rstd, weight, "bf16", "bf16", want=(name,))
        assert torch.equal(one[i], whole[i]) and sum(t is not None for t in one) == 1


def test_statistics_may_be_left_out(K, cuda):
    x = F.filled(values(9, 300, 10), "f16")
    weight, bias = weights(300, "f16", 11)
    y, z = F.matrix(9, 300, "f16"), F.matrix(9, 300, "f16")
    K.clpk_layer_norm(C.byref(B.norm_args(x, y, weight, bias, None, None, 1e-5, "f16", "f16")), F.stream())
    z, _, _ = forward(K, x, "f16", "f16", weight, bias)
    assert torch.equal(y, z)


@pytest.mark.parametrize("d", [64, 1500, 9000])
def test_a_mean_far_from_zero(K, cuda, d):
    """A thousand deviations: squares about the mean, not of it."""
    x = F.filled(values(12, d, 12, mean=1000.0), "f32")
    weight, bias = weights(d, "f32", 13)
    check_all(K, x, F.filled(values(12, d, 14), "f32"), weight, bias, "f32", "f32")


@pytest.mark.parametrize("d", [8, 100, 3001, 40000])
def test_rows_of_equal_elements_and_of_none_that_are_finite(K, cuda, d):
    x = F.filled(values(6, d, 15), "bf16")
    x[1], x[2] = 0, 3
    x[3, d // 2], x[4, 0] = float("nan"), float("inf")
    weight, bias = weights(d, "f32", 16)
    y, mean, rstd = forward(K, x, "bf16", "f32", weight, bias)
    for row in (1, 2):
        assert torch.equal(y[row], bias.to(torch.bfloat16)) and abs(float(rstd[row]) - 1e-5 ** -0.5) < 1e-3
    assert bool(torch.isnan(y[3:5]).all()) and bool(torch.isfinite(y[[0, 1, 2, 5]]).all())
    dy = F.filled(values(6, d, 17), "bf16")
    dx, dweight, dbias = backward(K, x, dy, mean, rstd, weight, "bf16", "f32")
    assert bool(torch.isnan(dx[3:5]).all()) and bool(torch.isfinite(dx[[0, 1, 2, 5]]).all())
    assert bool(torch.isnan(dweight).all()) and bool(torch.isfinite(dbias).all())
    y, _, _ = forward(K, x, "bf16", "f32", weight, bias, eps=0.0)
    assert bool(torch.isnan(y[1:3]).all())


def test_gradients_are_those_of_differences(K, cuda):
    m, d = 4, 96
    x, dy = values(m, d, 18).double(), values(m, d, 19).double()
    weight, bias = (t.double() for t in weights(d, "f32", 20))
    loss = lambda x, w, b: float((B.norm64(x, w, b, 1e-5, "f32")[0][0] * dy).sum())      # noqa: E731
    _, mean, rstd = forward(K, F.filled(x, "f32"), "f32", "f32", weight.float(), bias.float())
    dx, dweight, dbias = backward(K, F.filled(x, "f32"), F.filled(dy, "f32"), mean, rstd, weight.float(), "f32", "f32")
    h = 1e-5
    gen = torch.Generator(device="cuda")
    gen.manual_seed(21)
    for _ in range(4):
        vx, vw, vb = (torch.randn(*t.shape, generator=gen, device="cuda", dtype=torch.float64) for t in (x, weight, bias))
        want = (loss(x + h * vx, weight + h * vw, bias + h * vb) - loss(x - h * vx, weight - h * vw, bias - h * vb)) / (2 * h)
        got = float((dx.double() * vx).sum() + (dweight.double() * vw).sum() + (dbias.double() * vb).sum())
        scale = float((dx.double() * vx).abs().sum() + (dweight.double() * vw).abs().sum() + (dbias.double() * vb).abs().sum())
        # differences are off by h^2 and by 2^-53 / h of the sums, the kernel by some 2^-24
        assert abs(got - want) <= 1e-5 * scale


def test_the_same_sums_in_every_call_and_in_a_graph(K, cuda):
    m, d = 3000, 1200
    x, dy = F.filled(values(m, d, 22), "bf16"), F.filled(values(m, d, 23), "bf16")
    weight, bias = weights(d, "f32", 24)
    _, mean, rstd = forward(K, x, "bf16", "f32", weight, bias)
    first = backward(K, x, dy, mean, rstd, weight, "bf16", "f32")
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, backward(K, x, dy, mean, rstd, weight, "bf16", "f32")))
    y, dx, dw, db = F.matrix(m, d, "bf16"), F.matrix(m, d, "bf16"), torch.zeros(d, device="cuda"), torch.zeros(d, device="cuda")
    mean2, rstd2, workspace = torch.zeros_like(mean), torch.zeros_like(rstd), B.norm_workspace(K, m, d)
    one = B.norm_args(x, y, weight, bias, mean2, rstd2, 1e-5, "bf16", "f32")
    two = B.norm_backward_args(x, dy, mean2, rstd2, weight, dx, dw, db, workspace, "bf16", "f32")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.clpk_layer_norm(C.byref(one), F.stream())
        K.clpk_layer_norm_backward(C.byref(two), F.stream())
    for seed in (25, 26):
        x.copy_(values(m, d, seed))
        graph.replay()
        _, mean, rstd = forward(K, x, "bf16", "f32", weight, bias)
        want = backward(K, x, dy, mean, rstd, weight, "bf16", "f32")
        assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), want))


def test_no_rows(K, cuda):
    d = 24
    x = torch.empty(0, d, dtype=torch.float16, device="cuda")
    dw, db = (torch.full((d,), 77.0, device="cuda") for _ in range(2))
    K.clpk_layer_norm(C.byref(N.LayerNormArgs(dtype=N.DT_F16, weight_dtype=N.DT_F32, m=0, d=d, eps=1e-5)), F.stream())
    K.clpk_layer_norm_backward(C.byref(N.LayerNormBackwardArgs(dtype=N.DT_F16, weight_dtype=N.DT_F32, m=0, d=d, d_dweight=dw.data_ptr(), d_dbias=db.data_ptr())), F.stream())
    assert x.numel() == 0 and bool((dw == 0).all()) and bool((db == 0).all())


def test_refusals(K, cuda):
    x, y = F.matrix(3, 64, "bf16", fill=1), F.matrix(3, 64, "bf16")
    weight = torch.ones(64, device="cuda")
    mean, rstd, workspace = torch.zeros(3, device="cuda"), torch.ones(3, device="cuda"), B.norm_workspace(K, 3, 64)
    forward_args = lambda **k: B.norm_args(x, y, weight, weight, mean, rstd, 1e-5, "bf16", "f32")       # noqa: E731
    back_args = lambda: B.norm_backward_args(x, x, mean, rstd, weight, y, weight.clone(), weight.clone(), workspace, "bf16", "f32")     # noqa: E731

    def refused(call, args, match, **change):
        for name, v in change.items():
            setattr(args, name, v)
        with pytest.raises(N.ClpkError, match=match) as e:
            call(C.byref(args), F.stream())
        assert e.value.code == N.ERR_BAD_ARG
    f, b = K.clpk_layer_norm, K.clpk_layer_norm_backward
    for call, args in ((f, forward_args), (b, back_args)):
        refused(call, args(), "dtype 5 is not", dtype=N.DT_I8)
        refused(call, args(), "weight_dtype", weight_dtype=N.DT_F16)
        refused(call, args(), "no elements", d=0)
        refused(call, args(), "too large", m=2 ** 31)
        refused(call, args(), "too large", d=2 ** 30 + 1)
        refused(call, args(), "d_x is NULL", d_x=None)
        refused(call, args(), "pitch of d_x", ldx=63)
        refused(call, args(), "d_x is not aligned", d_x=x.data_ptr() + 1)
        refused(call, args(), "d_weight is not aligned", d_weight=weight.data_ptr() + 2)
        refused(call, args(), "d_mean is not aligned", d_mean=mean.data_ptr() + 1)
        with pytest.raises(N.ClpkError, match="args is NULL"):
            call(None, F.stream())
    refused(f, forward_args(), "d_y is NULL", d_y=None)
    refused(f, forward_args(), "pitch of d_y", ldy=5)
    for eps in (-1e-5, float("nan"), float("inf")):
        refused(f, forward_args(), "eps", eps=eps)
    refused(b, back_args(), "d_dy is NULL", d_dy=None)
    refused(b, back_args(), "pitch of d_dy", lddy=1)
    refused(b, back_args(), "pitch of d_dx", lddx=1)
    refused(b, back_args(), "d_mean or d_rstd", d_rstd=None)
    refused(b, back_args(), "d_dbias is not aligned", d_dbias=weight.data_ptr() + 1)
    for change in ({"d_workspace": None}, {"workspace_bytes": B.norm_workspace(K, 3, 64).numel() - 1}, {"d_workspace": workspace.data_ptr() + 4}):
        refused(b, back_args(), "workspace of", **change)
    K.clpk_layer_norm_backward(C.byref(back_args()), F.stream())
    torch.cuda.synchronize()


@pytest.mark.parametrize("m,d", [(11, 2056), (9, 2560), (7, 2561), (5, 4104), (9, 5120), (7, 5121), (6, 6144), (5, 6145), (149, 8192), (300, 6152), (1777, 600), (1776, 1000), (2000, 1024)])
def test_shapes_of_a_row(K, cuda, m, d):
    """Widths and numbers of rows where the threads that share a row change, the last threads with nothing, a piece of a vector, or all of it."""
    for dtype, wdtype in (("bf16", "f32"), ("f32", "f32"), ("f16", "f16")):
        x, dy = F.filled(values(m, d, d), dtype, pad=8), F.filled(values(m, d, d + 1), dtype, pad=16)
        weight, bias = weights(d, wdtype, d)
        check_all(K, x, dy, weight, bias, dtype, wdtype, pad=8)


def slices(x, dtype, fill=77):
    """The values as rows that do not start on 16 bytes."""
    wide = torch.full((x.shape[0], x.shape[1] + 3), fill, dtype=F.TORCH[dtype], device="cuda")
    wide[:, 1:x.shape[1] + 1] = x.to(F.TORCH[dtype])
    return wide[:, 1:x.shape[1] + 1]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,aligned", [(4, True), (96, True), (300, True), (1000, True), (4096, True), (8200, True), (16391, True), (40000, True), (4, False), (1000, False)])
def test_rows_whose_squares_leave_fp32(K, cuda, dtype, d, aligned):
    """Finite elements with a finite sum, whose squares or the sum of them are beyond fp32: the row is NaN with its rstd and its gradients, and
    no other row is."""
    place = F.filled if aligned else slices
    x = values(7, d, 40)
    sign = 1 - 2 * (torch.arange(d, device="cuda") % 2).float()
    bad = [1, 3, 4]
    x[1], x[3] = 1e20 * sign, 1e25 * sign
    x[4] = (3e38 / d) ** 0.5 * 1.25 * sign                      # each square fits, their sum does not
    x = place(x, dtype)
    weight, bias = weights(d, "f32", 41)
    y, mean, rstd = forward(K, x, dtype, "f32", weight, bias)
    good = [0, 2, 5, 6]
    assert bool(torch.isfinite(mean).all()) and bool(torch.isnan(rstd[bad]).all()) and bool(torch.isnan(y[bad]).all())
    for got, (want, allowed) in zip((y, mean, rstd), B.norm64(x[good], weight, bias, 1e-5, dtype)):
        F.check(got[good], want, allowed)
    dy = place(values(7, d, 42), dtype)
    dx, dweight, dbias = backward(K, x, dy, mean, rstd, weight, dtype, "f32")
    assert bool(torch.isnan(dx[bad]).all()) and bool(torch.isnan(dweight).all()) and bool(torch.isfinite(dbias).all())
    (want, allowed), _, _ = B.norm_backward64(x[good], dy[good], mean[good], rstd[good], weight, dtype, "f32")
    F.check(dx[good], want, allowed, "dx")
    # the largest squares that fit
    x = place(0.5 * (3e38 / d) ** 0.5 * sign.expand(2, d), dtype)
    y, mean, rstd = forward(K, x, dtype, "f32", weight, bias)
    for got, (want, allowed) in zip((y, mean, rstd), B.norm64(x, weight, bias, 1e-5, dtype)):
        F.check(got, want, allowed)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [7, 56, 100, 1000, 1001, 2056, 5000, 9000, 16376, 20000])
def test_the_mean_of_equal_elements_is_one_of_them(K, cuda, dtype, d):
    """Sums of equal elements with few bits are exact, and a sum over the number of its terms is the element again: nothing is left of the
    row but the bias, and nothing at all without eps."""
    equal = (3.0, 1000.0, -0.375, 56.0)
    x = F.filled(torch.tensor(equal, device="cuda")[:, None].expand(4, d), dtype)
    weight, bias = weights(d, "f32", 43)
    y, mean, rstd = forward(K, x, dtype, "f32", weight, bias)
    assert mean.tolist() == list(equal) and bool((abs(rstd - 1e-5 ** -0.5) < 1e-3).all())
    assert torch.equal(y, bias.to(F.TORCH[dtype]).expand(4, d))
    y, _, _ = forward(K, x, dtype, "f32", weight, bias, eps=0.0)
    assert bool(torch.isnan(y).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [40, 250, 1000, 1001, 4096, 6150, 9001, 16391])
def test_gradients_of_very_small_and_very_large_rows(K, cuda, dtype, d):
    """dy times what is left of x without its mean may be no number of fp32 where dy times xhat is one."""
    weight, bias = weights(d, "f32", 44)
    for size, gradient in ((1e-17, 1e-26), (1e-14, 1e-30), (1e15, 1e25), (1e13, 1e30)):
        x, dy = F.filled(values(9, d, 45) * size, dtype), F.filled(values(9, d, 46) * gradient, dtype)
        _, mean, rstd = forward(K, x, dtype, "f32", weight, bias, eps=0.0)
        for t, (want, allowed), name in zip(backward(K, x, dy, mean, rstd, weight, dtype, "f32"), B.norm_backward64(x, dy, mean, rstd, weight, dtype, "f32"),
                                            ("dx", "dweight", "dbias")):
            F.check(t, want, allowed, f"{name}, {size} and {gradient}")


@pytest.mark.parametrize("d", [37, 1001, 4094, 16381])
def test_gradients_of_equal_elements_far_from_zero(K, cuda, d):
    """What lies behind a row in its last vector is no part of it, however large the mean and rstd are."""
    x, dy = F.filled(torch.full((3, d), 2.0 ** 83, device="cuda"), "f32"), F.filled(values(3, d, 47) * 1e-3, "f32")
    weight, bias = weights(d, "f32", 48)
    _, mean, rstd = forward(K, x, "f32", "f32", weight, bias, eps=2e-38)
    assert mean.tolist() == [2.0 ** 83] * 3
    for t, (want, allowed), name in zip(backward(K, x, dy, mean, rstd, weight, "f32", "f32"), B.norm_backward64(x, dy, mean, rstd, weight, "f32", "f32"),
                                        ("dx", "dweight", "dbias")):
        F.check(t, want, allowed, name)


def test_gradients_side_by_side(K, cuda):
    """Two streams with workspaces of their own: as one behind the other."""
    cases = []
    for m, d, seed in ((3000, 1200, 50), (901, 4096, 60)):
        x, dy = F.filled(values(m, d, seed), "bf16"), F.filled(values(m, d, seed + 1), "bf16")
        weight, bias = weights(d, "f32", seed + 2)
        _, mean, rstd = forward(K, x, "bf16", "f32", weight, bias)
        cases.append(((K, x, dy, mean, rstd, weight, "bf16", "f32"), B.norm_workspace(K, m, d)))
    want = [backward(*args, workspace=space) for args, space in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for (args, space), s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(backward(*args, workspace=space))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
