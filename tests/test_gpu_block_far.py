"""The operators that train a block on rows, weights and tensors that reach past 2^32 bytes: the same bits as where they lie together."""
import ctypes as C

import pytest
import torch

from tests import block_util as B
from tests import ff_util as F

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def need(gigabytes):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gigabytes << 30:
        pytest.skip(f"needs {gigabytes} GB")


def far(values, pitch, offset=0, fill=False):
    """The values with `pitch` elements from one row (or matrix) to the next."""
    first, rest = values.shape[0], values[0].numel()
    whole = torch.empty(offset + (first - 1) * pitch + rest, dtype=values.dtype, device="cuda")
    assert whole.numel() * whole.element_size() > 2 ** 32
    out = torch.as_strided(whole, tuple(values.shape), (pitch, *values[0].contiguous().stride()), offset)
    return out.fill_(F.SENTINEL) if fill else out.copy_(values)


@pytest.mark.parametrize("dtype,d,offset", [("bf16", 1000, 0), ("f32", 4096, 0), ("bf16", 1000, 1), ("f32", 20000, 0)])
def test_rows_of_a_norm(K, cuda, dtype, d, offset):
    need(44)
    m, pitch = 3, (2 ** 30 if dtype == "f32" else 2 ** 31) + 64
    x, dy = (torch.randn(m, d, generator=gen(s), device="cuda").to(F.TORCH[dtype]) for s in (1, 2))
    weight, bias = torch.randn(2, d, generator=gen(3), device="cuda")
    results = []
    for apart in (False, True):
        place = (lambda v, **k: far(v, pitch, offset, **k)) if apart else (lambda v, **k: v.clone())
        here, y, mean, rstd = place(x), place(x, fill=True) if apart else x.clone(), torch.zeros(m, device="cuda"), torch.zeros(m, device="cuda")
        K.clpk_layer_norm(C.byref(B.norm_args(here, y, weight, bias, mean, rstd, 1e-5, dtype, "f32")), F.stream())
        got = [y.clone(), mean, rstd]
        del y
        there, dx = place(dy), place(x, fill=True) if apart else x.clone()
        dw, db = torch.zeros(d, device="cuda"), torch.zeros(d, device="cuda")
        K.clpk_layer_norm_backward(C.byref(B.norm_backward_args(here, there, mean, rstd, weight, dx, dw, db, B.norm_workspace(K, m, d), dtype, "f32")), F.stream())
        results.append(got + [dx.clone(), dw, db])
        del here, there, dx
    # rows that do not start on 16 bytes are summed by other threads
    if offset:
        for (want, allowed), got in zip(B.norm64(x, weight, bias, 1e-5, dtype), results[1]):
            F.check(got, want, allowed)
        for (want, allowed), got in zip(B.norm_backward64(x, dy, *results[1][1:3], weight, dtype, "f32"), results[1][3:]):
            F.check(got, want, allowed)
    else:
        assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("state,n", [("f32", 2 ** 30 + 300), ("i8", 2 ** 32 + 300)])
def test_tensors_of_a_step(K, cuda, state, n):
    """Blocks at the begin, at the end and beside the powers of two, against a tensor that has them alone; zeros elsewhere stay zeros."""
    dtype, small = ("f32", False) if state == "f32" else ("bf16", True)
    need(40)
    blocks = sorted({0, 1, n // 256 - 1, n // 256, *(2 ** p // 256 + i for p in (29, 30, 31, 32) for i in (-1, 0) if 2 ** p <= n)})
    sizes = [min(256, n - 256 * b) for b in blocks]
    t = B.Tensor(gen(4), sum(sizes), dtype, dtype, state, False)
    whole = lambda a: torch.zeros(n, dtype=a.dtype, device="cuda")               # noqa: E731
    big = B.Tensor.__new__(B.Tensor)
    big.n, big.state, big.master = n, state, None
    big.param, big.grad, big.m, big.v = (whole(a) for a in (t.param, t.grad, t.m, t.v))
    big.m_scale, big.v_scale = (torch.zeros(-(-n // 256), device="cuda") if small else None for _ in range(2))
    at = 0
    for i, (b, size) in enumerate(zip(blocks, sizes)):
        for name in ("param", "grad", "m", "v"):
            getattr(big, name)[256 * b:256 * b + size] = getattr(t, name)[at:at + size]
        if small:
            big.m_scale[b], big.v_scale[b] = t.m_scale[i], t.v_scale[i]
        at += size
    for tensor in (t, big):
        K.clpk_adamw(C.byref(B.adamw_args([tensor], dtype, dtype, state)), F.stream())
    at = 0
    for i, (b, size) in enumerate(zip(blocks, sizes)):
        for name in ("param", "m", "v"):
            assert torch.equal(getattr(big, name)[256 * b:256 * b + size], getattr(t, name)[at:at + size]), (name, b)
            getattr(big, name)[256 * b:256 * b + size] = 0
        if small:
            assert big.m_scale[b] == t.m_scale[i] and big.v_scale[b] == t.v_scale[i]
        at += size
    assert all(not bool(part.any()) for name in ("param", "m", "v") for part in getattr(big, name).split(2 ** 30))


def test_groups_and_their_rows(K, cuda):
    need(40)
    rows, n, k = [7, 30], 72, 136
    m = sum(rows)
    a, dc = (torch.randn(m, c, generator=gen(5 + c), device="cuda").bfloat16() for c in (k, n))
    w = (torch.randn(2, n, k, generator=gen(7), device="cuda") * k ** -0.5).bfloat16()
    offsets, workspace, status = B.offsets_of(rows), B.grouped_workspace(K), F.word()
    results = []
    for apart in (False, True):
        place = (lambda v, fill=False: far(v, 2 ** 31 + 64 if v.dim() == 3 else 2 ** 26 + 64, fill=fill)) if apart else (lambda v, fill=False: v.clone())
        here, weights, c = place(a), place(w), place(torch.zeros(m, n, device="cuda"), True)
        K.clpk_grouped_gemm(C.byref(B.grouped_args(here, weights, c, offsets, workspace, status, "bf16", "f32", n)), F.stream())
        assert int(status) == 0
        got = [c.clone()]
        del c
        there, da, dw = place(dc), place(a, True), place(torch.zeros_like(w), True)
        K.clpk_grouped_gemm_backward(C.byref(B.grouped_backward_args(here, weights, there, da, dw, offsets, workspace, status, "bf16", "bf16", n)), F.stream())
        assert int(status) == 0
        results.append(got + [da.clone(), dw.clone()])
        del here, weights, there, da, dw
    assert all(torch.equal(x, y) for x, y in zip(*results))
    F.check(results[0][0], *B.grouped64(a, w, rows, 0, "f32"))
