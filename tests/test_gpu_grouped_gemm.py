"""clpk_grouped_gemm and clpk_grouped_gemm_backward against 64 bits, element by element."""
import ctypes as C

import pytest
import torch

from clpeak_b200 import native as N
from tests import block_util as B
from tests import ff_util as F

pytestmark = pytest.mark.gpu

NAN = float("nan")
# rows of the groups, n, k
SMALL = [
    ([1], 8, 8), ([1], 300, 64), ([3, 0, 2], 256, 128), ([0, 0, 5, 0], 130, 72), ([0, 0], 64, 64),
    ([31, 32, 33], 264, 200), ([64, 128, 192], 512, 64), ([255, 256, 257], 100, 130), ([300, 1, 700], 257, 1000),
    ([1] * 40, 128, 256), ([7, 0, 19] * 9, 72, 520), ([513], 1, 1), ([20, 13], 1, 333), ([20, 13], 333, 1),
]
# sums that are cut: few tiles and long sums, of either product; and tiles by the round
LARGE = [([3, 0, 1, 2], 1408, 8192), ([100, 411], 700, 9000), ([9000, 40], 200, 136), ([2500, 0, 3001, 17], 1000, 520), ([1000] * 8, 512, 1024),
         ([70, 1900, 333, 0, 12, 800, 41], 2000, 1111)]


def values(*shape, seed, std=1.0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return torch.randn(*shape, generator=gen, device="cuda") * std


class Case:
    """Operands with NaN behind their rows, between the weights, and in rows that no group has."""

    def __init__(self, rows, n, k, dtype, first=0, spare=0, pad=0, between=0, seed=1):
        self.rows, self.n, self.k, self.dtype, self.first, self.pad, self.between = rows, n, k, dtype, first, pad, between
        self.used, self.m = sum(rows), first + sum(rows) + spare
        self.a, self.dc = (F.matrix(self.m, c, dtype, pad, NAN) for c in (k, n))
        inside = slice(first, first + self.used)
        self.a[inside] = values(self.used, k, seed=seed).to(F.TORCH[dtype])
        self.dc[inside] = values(self.used, n, seed=seed + 1, std=0.5).to(F.TORCH[dtype])
        self.w = B.weights3(len(rows), n, k, dtype, pad, between, values(len(rows), n, k, seed=seed + 2, std=k ** -0.5), NAN)
        self.offsets = B.offsets_of(rows, first)
        self.inside = inside

    def forward(self, K, out, workspace=None, offsets=None, c=None):
        c = F.matrix(self.m, self.n, out, self.pad) if c is None else c
        status = F.word()
        workspace = B.grouped_workspace(K) if workspace is None else workspace
        K.clpk_grouped_gemm(C.byref(B.grouped_args(self.a, self.w, c, self.offsets if offsets is None else offsets, workspace, status, self.dtype, out, self.n)), F.stream())
        return c, status

    def backward(self, K, out, want=("da", "dw"), workspace=None, offsets=None):
        da = F.matrix(self.m, self.k, self.dtype, self.pad) if "da" in want else None
        dw = B.weights3(len(self.rows), self.n, self.k, out, self.pad, self.between) if "dw" in want else None
        status = F.word()
        workspace = B.grouped_workspace(K) if workspace is None else workspace
        args = B.grouped_backward_args(self.a, self.w, self.dc, da, dw, self.offsets if offsets is None else offsets, workspace, status, self.dtype, out, self.n)
        K.clpk_grouped_gemm_backward(C.byref(args), F.stream())
        return da, dw, status

    def only_rows(self, t):
        """Nothing but the groups' rows was written."""
        left = torch.ones(self.m, dtype=torch.bool, device="cuda")
        left[self.inside] = False
        return F.untouched(t) and bool((t[left] == F.SENTINEL).all())

    def check_forward(self, K, out):
        c, status = self.forward(K, out)
        assert int(status) == 0
        if self.used:
            F.check(c[self.inside], *B.grouped64(self.a, self.w, self.rows, self.first, out), "c")
        assert self.only_rows(c)

    def check_backward(self, K, out):
        da, dw, status = self.backward(K, out)
        assert int(status) == 0
        (want_a, off_a), (want_w, off_w) = B.grouped_backward64(self.a, self.w, self.dc, self.rows, self.first, self.dtype, out)
        F.check(da[self.inside], want_a, off_a, "da")
        F.check(dw, want_w, off_w, "dw")
        assert self.only_rows(da) and bool((B.around(dw) == F.SENTINEL).all())


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("rows,n,k", SMALL)
def test_forward(K, cuda, rows, n, k, dtype, out):
    Case(rows, n, k, dtype).check_forward(K, out)
    Case(rows, n, k, dtype, first=5, spare=9, pad=1, between=3, seed=7).check_forward(K, out)


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("rows,n,k", SMALL)
def test_backward(K, cuda, rows, n, k, dtype, out):
    Case(rows, n, k, dtype).check_backward(K, out)
    Case(rows, n, k, dtype, first=5, spare=9, pad=1, between=3, seed=7).check_backward(K, out)


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("rows,n,k", LARGE)
def test_large(K, cuda, rows, n, k, dtype, out):
    case = Case(rows, n, k, dtype, spare=3)
    case.check_forward(K, out)
    case.check_backward(K, out)


def test_as_many_groups_as_there_may_be(K, cuda):
    rows = [(7 * i) % 5 for i in range(1024)]
    case = Case(rows, 64, 96, "bf16")
    case.check_forward(K, "bf16")
    case.check_backward(K, "f32")


def test_groups_far_apart(K, cuda):
    """Hundreds of groups without rows between a pair's tiles, and hundreds of tiles of a group each."""
    rows = [0] * 1024
    for at, n in ((0, 40), (31, 1), (32, 3), (64, 2), (399, 300), (400, 5), (1000, 33), (1023, 2)):
        rows[at] = n
    for case in (Case(rows, 264, 136, "bf16"), Case([2] * 777 + [0] * 64 + [1] * 96, 72, 264, "f16")):
        case.check_forward(K, "f32")
        case.check_backward(K, "f32")


def test_one_gradient_at_a_time(K, cuda):
    case = Case([70, 0, 333], 520, 264, "f16", spare=2)
    da, dw, _ = case.backward(K, "f16")
    assert torch.equal(case.backward(K, "f16", want=("da",))[0], da)
    assert torch.equal(case.backward(K, "f16", want=("dw",))[1], dw)
    status = case.backward(K, "f16", want=())[2]
    assert int(status) == 0


def test_infinities_stay_in_their_group(K, cuda):
    case = Case([40, 50, 60], 200, 136, "bf16")
    case.a[10], case.dc[10, 3] = float("inf"), NAN
    case.w[2, 5, 7] = NAN
    c, _ = case.forward(K, "bf16")
    assert bool(torch.isfinite(c[40:90]).all()) and bool(torch.isfinite(c[:10]).all()) and not bool(torch.isfinite(c[10]).any())
    assert bool(torch.isnan(c[90:, 5]).all()) and bool(torch.isfinite(c[90:, 6:]).all())
    da, dw, _ = case.backward(K, "f32")
    assert bool(torch.isfinite(dw[1:]).all()) and bool(torch.isfinite(da[40:90]).all()) and bool(torch.isnan(da[10]).all())


def test_the_same_sums_in_every_call(K, cuda):
    """Sums that several pairs share, whichever of them comes last."""
    for rows, n, k in LARGE[:4]:
        case = Case(rows, n, k, "bf16")
        workspace = B.grouped_workspace(K)
        c, _ = case.forward(K, "f32", workspace)
        da, dw, _ = case.backward(K, "f32", workspace=workspace)
        for _ in range(10):
            assert torch.equal(case.forward(K, "f32", workspace)[0], c)
            again = case.backward(K, "f32", workspace=workspace)
            assert torch.equal(again[0], da) and torch.equal(again[1], dw)


def test_sizes_change_under_a_graph(K, cuda):
    """Groups' sizes are read where they lie, by every replay; two graphs take turns with one workspace."""
    case = Case([100, 200, 300], 520, 1000, "bf16")
    workspace, status = B.grouped_workspace(K), F.word()
    c, da = F.matrix(case.m, case.n, "bf16"), F.matrix(case.m, case.k, "bf16")
    dw = B.weights3(3, case.n, case.k, "f32")
    offsets = case.offsets.clone()
    one = B.grouped_args(case.a, case.w, c, offsets, workspace, status, "bf16", "bf16", case.n)
    two = B.grouped_backward_args(case.a, case.w, case.dc, da, dw, offsets, workspace, status, "bf16", "f32", case.n)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    with torch.cuda.graph(graphs[0]):
        K.clpk_grouped_gemm(C.byref(one), F.stream())
    with torch.cuda.graph(graphs[1]):
        K.clpk_grouped_gemm_backward(C.byref(two), F.stream())
    for rows in ([100, 200, 300], [0, 600, 0], [599, 0, 1], [17, 18, 19]):
        offsets.copy_(B.offsets_of(rows))
        for g in graphs:
            g.replay()
        used = sum(rows)
        F.check(c[:used], *B.grouped64(case.a, case.w, rows, 0, "bf16"), "c")
        (want_a, off_a), (want_w, off_w) = B.grouped_backward64(case.a, case.w, case.dc, rows, 0, "bf16", "f32")
        F.check(da[:used], want_a, off_a, "da")
        F.check(dw, want_w, off_w, "dw")
        assert int(status) == 0


def test_on_two_streams_with_workspaces_of_their_own(K, cuda):
    cases = [Case([300, 5, 600], 520, 2000, "bf16", seed=20), Case([1, 2, 3, 800], 264, 4000, "bf16", seed=30)]
    want = [case.forward(K, "f32")[0] for case in cases]
    spaces, streams = [B.grouped_workspace(K) for _ in cases], [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for case, space, s in zip(cases, spaces, streams):
            with torch.cuda.stream(s):
                got.append(case.forward(K, "f32", space)[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("offsets", [[0, 20, 10, 60], [0, 20, 40, 61], [-1, 20, 40, 60], [5, 4, 4, 4], [0, 20, 2 ** 31 - 1, 60]])
def test_offsets_that_are_none(K, cuda, offsets):
    """A word that tells it, and no result."""
    case = Case([20, 20, 20], 72, 64, "bf16")
    bad = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    c, status = case.forward(K, "bf16", offsets=bad)
    assert int(status) == 0x401 and bool((c == F.SENTINEL).all())
    da, dw, status = case.backward(K, "bf16", offsets=bad)
    assert int(status) == 0x401 and bool((da == F.SENTINEL).all()) and bool((dw == F.SENTINEL).all())
    assert int(case.forward(K, "bf16")[1]) == 0


def test_no_rows(K, cuda):
    case = Case([0, 0], 72, 40, "bf16", pad=1, between=2)
    dw, status, workspace = B.weights3(2, 72, 40, "bf16", 1, 2), F.word(), B.grouped_workspace(K)
    empty = torch.empty(0, 72, dtype=torch.bfloat16, device="cuda")
    K.clpk_grouped_gemm(C.byref(B.grouped_args(case.a[:0], case.w, empty, case.offsets, workspace, status, "bf16", "bf16", 72)), F.stream())
    assert int(status) == 0
    args = B.grouped_backward_args(case.a[:0], case.w, empty, None, dw, case.offsets, workspace, status, "bf16", "bf16", 72)
    assert args.m == 0
    K.clpk_grouped_gemm_backward(C.byref(args), F.stream())
    assert int(status) == 0 and bool((dw == 0).all()) and bool((B.around(dw) == F.SENTINEL).all())


def test_gradients_are_those_of_differences(K, cuda):
    case = Case([30, 0, 21], 64, 48, "f16")
    da, dw, _ = case.backward(K, "f32")
    h = 1e-3
    va, vw = values(case.m, case.k, seed=40).double(), values(3, case.n, case.k, seed=41).double()
    loss = lambda a, w: float((B.grouped64(a, w, case.rows, 0, "f32")[0] * case.dc.double()).sum())      # noqa: E731
    a, w = case.a.double(), case.w.double()
    want = (loss(a + h * va, w + h * vw) - loss(a - h * va, w - h * vw)) / (2 * h)
    terms = torch.cat(((da.double() * va).flatten(), (dw.double() * vw).flatten()))
    # bilinear: differences are exact but for 2^-53 / h of their sums; da is rounded to 2^-11, dw summed in fp32
    assert abs(float(terms.sum()) - want) <= 2 ** -11 * float(terms.abs().sum()) + 1e-6


def test_refusals(K, cuda):
    case = Case([20, 30], 72, 64, "bf16")
    c, da, dw = F.matrix(50, 72, "bf16"), F.matrix(50, 64, "bf16"), B.weights3(2, 72, 64, "bf16")
    workspace, status = B.grouped_workspace(K), F.word()
    forward = lambda: B.grouped_args(case.a, case.w, c, case.offsets, workspace, status, "bf16", "bf16", 72)              # noqa: E731
    backward = lambda: B.grouped_backward_args(case.a, case.w, case.dc, da, dw, case.offsets, workspace, status, "bf16", "bf16", 72)     # noqa: E731

    def refused(call, args, match, **change):
        for name, v in change.items():
            setattr(args, name, v)
        with pytest.raises(N.ClpkError, match=match) as e:
            call(C.byref(args), F.stream())
        assert e.value.code == N.ERR_BAD_ARG
    for call, args, result in ((K.clpk_grouped_gemm, forward, "out_dtype"), (K.clpk_grouped_gemm_backward, backward, "dw_dtype")):
        refused(call, args(), "is not BF16 or F16", dtype=N.DT_F32)
        refused(call, args(), "neither dtype nor F32", **{result: N.DT_F16})
        for name in ("n", "k"):
            refused(call, args(), "only the number of rows", **{name: 0})
            refused(call, args(), "too large", **{name: 2 ** 29})
        refused(call, args(), "too large", m=2 ** 31 - 256)
        refused(call, args(), "0 groups", groups=0)
        refused(call, args(), "1025 groups", groups=1025)
        refused(call, args(), "d_offsets", d_offsets=None)
        refused(call, args(), "d_offsets", d_offsets=case.offsets.data_ptr() + 2)
        refused(call, args(), "workspace of", d_workspace=None)
        refused(call, args(), "workspace of", workspace_bytes=workspace.numel() - 1)
        refused(call, args(), "workspace of", d_workspace=workspace.data_ptr() + 8)
        refused(call, args(), "d_status", d_status=None)
        for name in ("d_a", "d_w"):
            refused(call, args(), f"{name} is NULL", **{name: None})
            refused(call, args(), f"{name} must start on 16 bytes", **{name: case.a.data_ptr() + 2})
        refused(call, args(), "pitch of d_a", lda=56)
        refused(call, args(), "pitch of d_w", ldw=63)
        refused(call, args(), "stride_w", stride_w=72 * 64 - 8)
        refused(call, args(), "stride_w", stride_w=72 * 64 + 4)
        with pytest.raises(N.ClpkError, match="args is NULL"):
            call(None, F.stream())
    refused(K.clpk_grouped_gemm, forward(), "d_c is NULL", d_c=None)
    refused(K.clpk_grouped_gemm, forward(), "pitch of d_c", ldc=64)
    refused(K.clpk_grouped_gemm_backward, backward(), "d_dc is NULL", d_dc=None)
    refused(K.clpk_grouped_gemm_backward, backward(), "pitch of d_da", ldda=60)
    refused(K.clpk_grouped_gemm_backward, backward(), "pitch of d_dw", lddw=62)
    refused(K.clpk_grouped_gemm_backward, backward(), "stride_dw", stride_dw=8)
    assert bool((c == F.SENTINEL).all()) and bool((da == F.SENTINEL).all()) and bool((dw == F.SENTINEL).all())


def test_sizes_drawn_over_the_whole_range(K, cuda):
    """Sums that are cut and that are not, groups of any size, odd sizes: each element of both passes."""
    import random
    rng = random.Random(11)
    spread = lambda lo, hi: round(lo * (hi / lo) ** rng.random())       # noqa: E731
    for i in range(30):
        groups = spread(1, 60)
        rows = [rng.choice((0, 1, 2, spread(1, 4000 // groups + 1), spread(1, 8000 // groups + 1))) for _ in range(groups)]
        if not sum(rows):
            rows[0] = 3
        n, k = spread(1, 3000), spread(1, 3000)
        if sum(rows) * n * k > 2e10 or groups * n * k > 2e8:
            n, k = n // 8 + 1, k // 8 + 1
        case = Case(rows, n, k, rng.choice(("bf16", "f16")), first=rng.choice((0, 3)), spare=rng.choice((0, 70)), pad=i % 2, seed=i)
        case.check_forward(K, rng.choice((case.dtype, "f32")))
        case.check_backward(K, rng.choice((case.dtype, "f32")))
