"""clpk_quantize_rows_i8 against the same arithmetic in torch: equal, element for element."""
import numpy as np
import pytest
import torch

from clpeak_b200 import native as N
from tests import ff_util as F

pytestmark = pytest.mark.gpu

# one element, below and beyond a vector, a warp's row, a block's, the longest that registers hold, and longer ones
COLS = [1, 3, 7, 8, 31, 64, 255, 1024, 1025, 2049, 4096, 11007, 16385, 32768, 65537]


def run(K, x, q, scales, dtype):
    K.clpk_quantize_rows_i8(q.data_ptr(), scales.data_ptr(), x.data_ptr(), x.shape[0], x.shape[1], q.stride(0), x.stride(0), F.DT[dtype], F.stream())


def values(rows, cols, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    return x * torch.exp(4 * torch.randn(rows, 1, generator=gen, device="cuda"))


def same(q, scales, x):
    want_q, want_s = F.quantize64(x)
    assert torch.equal(torch.nan_to_num(scales, -1), torch.nan_to_num(want_s, -1)) and torch.equal(q, want_q)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("cols", COLS)
def test_every_length(K, cuda, dtype, cols):
    for rows in (1, 5):
        x = F.filled(values(rows, cols, cols).clamp(-6e4, 6e4), dtype, pad=rows // 4)
        q, scales = F.matrix(rows, cols, "i8", pad=1), torch.full((rows,), -1.0, device="cuda")
        run(K, x, q, scales, dtype)
        same(q, scales, x)
        assert F.untouched(q)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("offset,cols", [(1, 64), (3, 1000), (5, 4099)])
def test_any_address_and_pitch(K, cuda, dtype, offset, cols):
    rows = 6
    flat = values(1, offset + rows * (cols + 3), 5).flatten().clamp(-6e4, 6e4).to(F.TORCH[dtype])
    x = torch.as_strided(flat, (rows, cols), (cols + 3, 1), offset)
    q8 = torch.full((rows * (cols + 1) + 9,), 77, dtype=torch.int8, device="cuda")
    q, scales = torch.as_strided(q8, (rows, cols), (cols + 1, 1), offset), torch.full((rows,), -1.0, device="cuda")
    run(K, x, q, scales, dtype)
    same(q, scales, x)
    left = torch.ones_like(q8, dtype=torch.bool)
    torch.as_strided(left, (rows, cols), (cols + 1, 1), offset).fill_(False)
    assert bool((q8[left] == 77).all())


def test_pitch_of_zero_is_the_row(K, cuda):
    x = values(9, 48, 2).to(torch.bfloat16)
    q, scales = torch.empty(9, 48, dtype=torch.int8, device="cuda"), torch.empty(9, device="cuda")
    K.clpk_quantize_rows_i8(q.data_ptr(), scales.data_ptr(), x.data_ptr(), 9, 48, 0, 0, N.DT_BF16, F.stream())
    same(q, scales, x)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cols,pad", [(40, 0), (4000, 0), (40, None)])
def test_rows_without_a_scale(K, cuda, dtype, cols, pad):
    """Zeros, the smallest numbers, infinities and NaNs; every row by itself."""
    x = torch.randn(9, cols, device="cuda")
    x[1] = 0
    x[2] = 0
    x[2, 7] = 127 * 2.0 ** -127                                # half of what has a scale
    x[3] = 0
    x[3, 7] = 127 * 2.0 ** -126                                # the smallest that has one
    x[4, 3] = float("inf")
    x[5, cols - 1] = float("nan")
    x[6, 0] = -float("inf")
    x[7] = -0.0
    x[8] = torch.finfo(F.TORCH[dtype]).max
    if pad is None:                                            # not aligned: element by element
        flat = torch.empty(9 * (cols + 1) + 1, dtype=F.TORCH[dtype], device="cuda")
        xs = torch.as_strided(flat, (9, cols), (cols + 1, 1), 1)
        xs.copy_(x)
    else:
        xs = F.filled(x, dtype)
    q, scales = F.matrix(9, cols, "i8"), torch.full((9,), -1.0, device="cuda")
    run(K, xs, q, scales, dtype)
    same(q, scales, xs)
    assert scales[1] == 0 and scales[2] == 0 and scales[3] == 2.0 ** -126 and scales[7] == 0 and bool(torch.isnan(scales[4:7]).all())
    assert not q[1:3].any() and not q[4:8].any() and q[3, 7] == 127 and bool((q[8] == 127).all())


def test_ties_go_to_the_even_number(K, cuda):
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, -127.0]], device="cuda")
    q, scales = F.matrix(1, 9, "i8"), torch.empty(1, device="cuda")
    x = F.filled(x, "f32")
    run(K, x, q, scales, "f32")
    assert q.tolist() == [[127, 0, 2, 2, 0, -2, -2, 126, -127]] and scales.item() == 1.0


def test_no_rows_and_no_columns(K, cuda):
    K.clpk_quantize_rows_i8(None, None, None, 0, 64, 0, 0, N.DT_F32, F.stream())
    scales = torch.full((3,), -1.0, device="cuda")
    K.clpk_quantize_rows_i8(None, scales.data_ptr(), None, 3, 0, 0, 0, N.DT_F32, F.stream())
    assert scales.tolist() == [0, 0, 0]


def test_beyond_32_bits(K, cuda):
    """Rows whose first element lies more than 2^32 bytes into the array."""
    rows, cols, step = 3, 64, 1 << 30
    flat = torch.empty(2 * step + cols, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(flat, (rows, cols), (step, 1))
    x.copy_(values(rows, cols, 3))
    q, scales = torch.empty(rows, cols, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    run(K, x, q, scales, "bf16")
    same(q, scales, x)


def test_refusals(K, cuda):
    x, q, s = (torch.zeros(64, device="cuda") for _ in range(3))
    for args, text in [((q.data_ptr(), s.data_ptr(), x.data_ptr(), 1, 8, 0, 0, N.DT_E4M3, None), "not F32, F16 or BF16"),
                       ((None, s.data_ptr(), x.data_ptr(), 1, 8, 0, 0, N.DT_F32, None), "NULL buffer"),
                       ((q.data_ptr(), None, x.data_ptr(), 1, 8, 0, 0, N.DT_F32, None), "NULL buffer"),
                       ((q.data_ptr(), s.data_ptr(), None, 1, 8, 0, 0, N.DT_F32, None), "NULL buffer"),
                       ((q.data_ptr(), s.data_ptr(), x.data_ptr(), 1, 8, 7, 0, N.DT_F32, None), "shorter than a row"),
                       ((q.data_ptr(), s.data_ptr(), x.data_ptr(), 1, 8, 0, 7, N.DT_F32, None), "shorter than a row"),
                       ((q.data_ptr(), s.data_ptr(), x.data_ptr(), 1 << 31, 8, 0, 0, N.DT_F32, None), "too large"),
                       ((q.data_ptr(), s.data_ptr(), x.data_ptr() + 1, 1, 8, 0, 0, N.DT_BF16, None), "not aligned")]:
        with pytest.raises(N.ClpkError, match=text) as e:
            K.clpk_quantize_rows_i8(*args)
        assert e.value.code == N.ERR_BAD_ARG


def test_repeats_bit_for_bit(K, cuda):
    x = F.filled(values(513, 3000, 9), "bf16")
    got = []
    for _ in range(3):
        q, scales = F.matrix(513, 3000, "i8"), torch.empty(513, device="cuda")
        run(K, x, q, scales, "bf16")
        got.append((q.clone(), scales))
    assert all(torch.equal(got[0][0], g[0]) and np.array_equal(got[0][1].cpu(), g[1].cpu()) for g in got[1:])
