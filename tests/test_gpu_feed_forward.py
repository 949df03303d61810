"""Gated feed-forward products, their gradients and scaled 8-bit products against 64 bits, within what ff_util counts.

Sizes: single tokens, tokens just below and above a tile's, odd widths, one column, sums of one element."""
import ctypes as C
import threading

import pytest
import torch

from clpeak_b200 import native as N
from tests import ff_util as F

pytestmark = pytest.mark.gpu

# (tokens, model width, hidden width)
SIZES = [(1, 1, 1), (1, 4096, 1000), (2, 65, 33), (3, 1024, 4097), (16, 200, 128), (17, 2048, 136), (37, 1000, 2712), (64, 640, 520),
         (65, 96, 1016), (128, 72, 264), (129, 520, 64), (200, 64, 8), (257, 333, 257), (513, 128, 1400), (1000, 1, 40), (2500, 264, 700)]
# one for every way to split the work: tile widths of 64 to 256, K in one, two or four ranges on CTA pairs, and one to eight ranges
# of the few-token kernel, whose partial sums lie behind its ring or in it (16-bit operands; in 8 bits K is twice as long for that)
SPLIT_PAIRS = [(130, 1000, 8), (130, 2000, 520), (300, 4096, 700), (130, 4096, 520), (130, 4096, 2712), (300, 4096, 520), (130, 8200, 4096), (300, 8200, 700)]
SPLIT_FEW = [(1, 520, 8), (2, 1000, 8), (1, 520, 2712), (1, 8200, 1400), (97, 2000, 8), (112, 2000, 1000), (5, 1000, 16000), (33, 1000, 16000),
             (96, 1000, 16000), (1, 64, 30000)]
SPLIT_SCALED = [(130, 2000, 8), (130, 4096, 1000), (300, 8200, 1400), (130, 8200, 1000), (130, 8200, 6000), (130, 8200, 2712), (300, 16000, 4096),
                (300, 16000, 1400), (520, 64, 6000), (1, 1000, 8), (1, 2000, 8), (97, 4096, 8), (112, 4096, 2712), (33, 2000, 30000), (96, 2000, 30000), (1, 8200, 20000)]
SPLIT_BACKWARD = [(64, 64, 64), (200, 64, 64), (8000, 264, 2816), (4000, 520, 1000), (1000, 2048, 520), (520, 2048, 520), (2000, 64, 64), (100, 64, 1000),
                  (2000, 64, 100), (200, 64, 520), (520, 2048, 200), (2000, 2048, 520), (4000, 2048, 520), (520, 2048, 264), (2000, 2048, 1000),
                  (4000, 520, 4096), (8000, 136, 2816), (4000, 136, 2816),
                  # sums in parts: of dx, of dW
                  (362, 96, 11829), (147, 654, 7749), (100, 4096, 8192), (9, 1436, 6644), (689, 1, 904), (8000, 96, 200), (16000, 40, 100), (1860, 1, 284),
                  (4653, 1818, 8), (1702, 1, 582), (1235, 3, 781), (3585, 132, 1088)]
LARGE = [(1, 8192, 14336), (48, 4096, 11008), (2049, 2056, 1032), (4096, 1024, 2816)]


def normal(seed, rows, cols, std=1.0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return torch.randn(rows, cols, generator=gen, device="cuda") * std


def integers(seed, rows, cols, most=127):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return torch.randint(-most, most + 1, (rows, cols), generator=gen, device="cuda")


def scales(seed, n, size):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return (torch.rand(n, generator=gen, device="cuda") + 0.5) * size


# ---- 16 bits, forward ----------------------------------------------------------------------------------

def forward(K, dtype, act, m, d, f, pad, keep, spread=1.0):
    x = F.filled(normal(1, m, d, spread), dtype, pad)
    wg, wu = (F.filled(normal(s, f, d, d ** -0.5), dtype, pad) for s in (2, 3))
    h, g, u = (F.matrix(m, f, dtype, pad) for _ in range(3))
    status = F.word()
    K.clpk_gated_ffn(C.byref(F.ffn_args(dtype, act, x, wg, wu, h, status, *((g, u) if keep else ()))), F.stream())
    want = F.gated64(act, x, wg, wu, dtype, dtype)
    F.check(h, *want[0], "h")
    if keep:
        F.check(g, *want[1], "g")
        F.check(u, *want[2], "u")
    assert status.item() == 0 and all(F.untouched(t) for t in (h, g, u))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,d,f", SIZES)
def test_gated_sizes(K, cuda, dtype, m, d, f):
    forward(K, dtype, "silu", m, d, f, pad=m % 3, keep=False)
    forward(K, dtype, "gelu_tanh", m, d, f, pad=f % 2, keep=True)


@pytest.mark.parametrize("m,d,f", SPLIT_PAIRS + SPLIT_FEW)
def test_gated_splits(K, cuda, m, d, f):
    forward(K, "bf16", "silu", m, d, f, pad=m % 2, keep=True)


@pytest.mark.parametrize("act", sorted(F.ACTS))
@pytest.mark.parametrize("m", [5, 300])
def test_gated_activations(K, cuda, act, m):
    forward(K, "bf16", act, m, 256, 320, 0, True, spread=3.0)
    forward(K, "f16", act, m, 264, 136, 1, False, spread=0.1)


@pytest.mark.parametrize("m,d,f", LARGE)
def test_gated_large(K, cuda, m, d, f):
    forward(K, "bf16", "silu", m, d, f, 0, m > 1000)


def test_gated_infinities_and_nans_stay_in_their_rows(K, cuda):
    """A token that is not finite spoils its own row of h, a channel its own column, and nothing else."""
    for m in (9, 300):
        x, wg, wu = normal(1, m, 200), normal(2, 136, 200), normal(3, 136, 200)
        x[3, 5], wu[7, 11] = float("nan"), float("inf")
        x, wg, wu = (F.filled(t, "bf16") for t in (x, wg, wu))
        h, status = F.matrix(m, 136, "bf16"), F.word()
        K.clpk_gated_ffn(C.byref(F.ffn_args("bf16", "silu", x, wg, wu, h, status)), F.stream())
        bad = ~torch.isfinite(h)
        want = torch.zeros_like(bad)
        want[3], want[:, 7] = True, True
        assert torch.equal(bad, want)


# ---- 8 bits --------------------------------------------------------------------------------------------

def scaled(K, out, m, k, n):
    pad = (m + n) % 3
    a, b = F.filled(integers(1, m, k), "i8", pad), F.filled(integers(2, n, k), "i8", pad)
    sa, sb = scales(3, m, 0.02), scales(4, n, 1e-3)
    for bias in (None, normal(5, 1, n)[0].to(F.TORCH[out])):
        c, status = F.matrix(m, n, out, pad), F.word()
        K.clpk_gemm_i8_scaled(C.byref(F.linear_args(a, b, c, sa, sb, status, out, bias)), F.stream())
        F.check(c, *F.linear64(a, b, sa, sb, out, bias), "c")
        assert status.item() == 0 and F.untouched(c)


@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,k,n", SIZES + LARGE[1:])
def test_scaled_product(K, cuda, out, m, k, n):
    scaled(K, out, m, k, n)


@pytest.mark.parametrize("m,k,n", SPLIT_SCALED)
def test_scaled_product_splits(K, cuda, m, k, n):
    scaled(K, "f32", m, k, n)


@pytest.mark.parametrize("m", [1, 130])
def test_scaled_product_of_the_longest_sums(K, cuda, m):
    """131071 products of -128 and -128 just fit 32 bits, and -128 is an element like any other."""
    k = 131071
    a, b = (F.filled(torch.full((rows, k), -128, device="cuda"), "i8") for rows in (m, 24))
    a[0, ::2] = 127
    sa, sb = torch.ones(m, device="cuda"), torch.ones(24, device="cuda")
    c, status = F.matrix(m, 24, "f32"), F.word()
    K.clpk_gemm_i8_scaled(C.byref(F.linear_args(a, b, c, sa, sb, status, "f32")), F.stream())
    want = a.double() @ b.double().T
    assert torch.equal(c, want.float()) and (m == 1 or want.max() == 131071 * 16384)


def test_a_row_without_a_scale_is_nan_or_zero(K, cuda):
    a, b = F.filled(integers(1, 4, 64), "i8"), F.filled(integers(2, 40, 64), "i8")
    a[2] = 0
    sa, sb = torch.tensor([1.0, float("nan"), 0.0, 2.0], device="cuda"), torch.ones(40, device="cuda")
    c, status = F.matrix(4, 40, "bf16"), F.word()
    K.clpk_gemm_i8_scaled(C.byref(F.linear_args(a, b, c, sa, sb, status, "bf16")), F.stream())
    assert bool(torch.isnan(c[1]).all()) and not c[2].any() and bool(torch.isfinite(c[[0, 3]]).all())


def gated_i8(K, out, m, d, f):
    pad = (m + f) % 2
    x, wg, wu = (F.filled(integers(s, rows, d), "i8", pad) for s, rows in ((1, m), (2, f), (3, f)))
    ss = scales(4, m, 0.02), scales(5, f, 0.02 / d ** 0.5), scales(6, f, 0.02 / d ** 0.5)
    h, status = F.matrix(m, f, out, pad), F.word()
    act = sorted(F.ACTS)[(m + d) % 5]
    K.clpk_gated_ffn(C.byref(F.ffn_args("i8", act, x, wg, wu, h, status, scales=ss, out=out)), F.stream())
    F.check(h, *F.gated64(act, x, wg, wu, "i8", out, ss)[0], "h")
    assert status.item() == 0 and F.untouched(h)


@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,d,f", SIZES + LARGE[1:])
def test_gated_8_bits(K, cuda, out, m, d, f):
    gated_i8(K, out, m, d, f)


@pytest.mark.parametrize("m,d,f", SPLIT_PAIRS + SPLIT_FEW)
def test_gated_8_bits_splits(K, cuda, m, d, f):
    gated_i8(K, "f32", m, 2 * d, f)


# ---- backward ------------------------------------------------------------------------------------------

def backward(K, dtype, act, m, d, f, pad=0, dx=True, dw=True, spread=1.0):
    x = F.filled(normal(1, m, d), dtype, pad)
    wg, wu = (F.filled(normal(s, f, d, d ** -0.5), dtype, pad) for s in (2, 3))
    dh, g, u = (F.filled(normal(s, m, f, std), dtype, pad) for s, std in ((4, 0.1), (5, spread), (6, 1.0)))
    out = [F.matrix(rows, d, dtype, pad) for rows in (m, f, f)]
    ws, status = F.workspace(K, dtype, m, d, f), F.word()
    args = F.backward_args(dtype, act, x, wg, wu, dh, g, u, out[0] if dx else None, out[1] if dw else None, out[2] if dw else None, ws, status)
    K.clpk_gated_ffn_backward(C.byref(args), F.stream())
    want = F.backward64(act, x, wg, wu, dh, g, u, dtype)
    for t, w, name, asked in zip(out, want, ("dx", "dwg", "dwu"), (dx, dw, dw)):
        if asked:
            F.check(t, *w, name)
        else:
            assert bool((t == F.SENTINEL).all())
        assert F.untouched(t)
    assert status.item() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,d,f", SIZES)
def test_backward_sizes(K, cuda, dtype, m, d, f):
    backward(K, dtype, "silu", m, d, f, pad=m % 2)


@pytest.mark.parametrize("m,d,f", SPLIT_BACKWARD)
def test_backward_splits(K, cuda, m, d, f):
    backward(K, "bf16", "silu", m, d, f, pad=f % 3 % 2)


@pytest.mark.parametrize("act", sorted(F.ACTS))
def test_backward_activations(K, cuda, act):
    backward(K, "bf16", act, 96, 200, 136, spread=4.0)
    backward(K, "f16", act, 40, 64, 333, pad=1, spread=2.0)


@pytest.mark.parametrize("m,d,f", [(2049, 2056, 1032), (4096, 1024, 2816), (9000, 128, 256)])
def test_backward_large(K, cuda, m, d, f):
    backward(K, "bf16", "gelu_tanh", m, d, f)


@pytest.mark.parametrize("dx,dw", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("m,d,f", [(70, 136, 264), (1702, 1, 582), (2049, 520, 1032)])
def test_backward_of_what_is_asked_for(K, cuda, dx, dw, m, d, f):
    backward(K, "bf16", "silu", m, d, f, dx=dx, dw=dw)


@pytest.mark.parametrize("act", sorted(F.ACTS))
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_gradients_against_differences(K, cuda, dtype, act):
    """Forward, then backward, then the slope of sum(dh * h) along a direction of each input, from the formula in 64 bits at two
    points.  The inputs are chosen so that g and u are exact in 16 bits: quarters up to 12.  A difference over 2 t is off by
    t^2 / 6 of the third derivative along the direction; t = 2^-12 leaves 1e-5 of the slope's scale."""
    m, d, f = 40, 24, 56
    x = F.filled(integers(1, m, d, 1), dtype)
    wg, wu = (F.filled(integers(s, f, d, 2) / 4, dtype) for s in (2, 3))
    dh = F.filled(normal(4, m, f, 0.1), dtype)
    h, g, u = (F.matrix(m, f, dtype) for _ in range(3))
    status = F.word()
    K.clpk_gated_ffn(C.byref(F.ffn_args(dtype, act, x, wg, wu, h, status, g, u)), F.stream())
    assert torch.equal(g.double(), x.double() @ wg.double().T) and torch.equal(u.double(), x.double() @ wu.double().T)
    grads = [F.matrix(rows, d, dtype) for rows in (m, f, f)]
    ws = F.workspace(K, dtype, m, d, f)
    K.clpk_gated_ffn_backward(C.byref(F.backward_args(dtype, act, x, wg, wu, dh, g, u, *grads, ws, status)), F.stream())
    allowed = [w[1] for w in F.backward64(act, x, wg, wu, dh, g, u, dtype)]
    point = [t.double() for t in (x, wg, wu)]

    def loss(p):
        return (dh.double() * F.act64(act, p[0] @ p[1].T) * (p[0] @ p[2].T)).sum()
    t = 2.0 ** -12
    for i in range(3):
        v = normal(7 + i, *point[i].shape).double()
        if act == "relu" and i < 2:
            # no g may cross 0 on the way: keep to gates that stay on their side
            gate = point[0] @ point[1].T
            change = (v @ point[1].T) if i == 0 else (point[0] @ v.T)
            crossing = (gate.abs() <= t * change.abs() * 1.01)
            dh_kept = dh.double() * ~crossing
            a, da = F.both64(act, gate)
            dg, du = dh_kept * (point[0] @ point[2].T) * da, dh_kept * a
            missing = (dh.double() * crossing * (point[0] @ point[2].T) * da, dh.double() * crossing * a)
            both = [missing[0] @ point[1] + missing[1] @ point[2], missing[0].T @ point[0]][i]
            ends = [point[:i] + [point[i] + s * v] + point[i + 1:] for s in (t, -t)]
            slope = sum(s * (dh_kept * F.act64(act, p[0] @ p[1].T) * (p[0] @ p[2].T)).sum() for s, p in zip((1, -1), ends)) / (2 * t)
            slope = slope + (both * v).sum()
        else:
            ends = [point[:i] + [point[i] + s * v] + point[i + 1:] for s in (t, -t)]
            slope = (loss(ends[0]) - loss(ends[1])) / (2 * t)
        got = (grads[i].double() * v).sum()
        size = (dh.double().abs() * 12 * 12).sum()
        assert abs(got - slope) <= (allowed[i] * v.abs()).sum() + 1e-5 * size


# ---- no tokens, the same call again, other streams -------------------------------------------------------------

def test_no_tokens(K, cuda):
    d, f = 72, 136
    wg, wu = (F.filled(normal(s, f, d), "bf16") for s in (2, 3))
    none = torch.empty(0, d, dtype=torch.bfloat16, device="cuda")
    status = F.word()
    args = N.GatedFfnArgs(dtype=N.DT_BF16, m=0, d=d, f=f, d_wg=wg.data_ptr(), d_wu=wu.data_ptr(), d_status=status.data_ptr())
    K.clpk_gated_ffn(C.byref(args), F.stream())
    assert status.item() == 0
    dwg, dwu = (F.matrix(f, d, "bf16", 1) for _ in range(2))
    status = F.word()
    args = N.GatedFfnBackwardArgs(dtype=N.DT_BF16, m=0, d=d, f=f, d_x=none.data_ptr(), d_dwg=dwg.data_ptr(), d_dwu=dwu.data_ptr(),
                                  ldw=dwg.stride(0), d_status=status.data_ptr())
    K.clpk_gated_ffn_backward(C.byref(args), F.stream())
    assert status.item() == 0 and not dwg.any() and not dwu.any() and F.untouched(dwg) and F.untouched(dwu)
    status = F.word()
    K.clpk_gemm_i8_scaled(C.byref(N.GemmI8ScaledArgs(m=0, n=8, k=16, out_dtype=N.DT_F32, d_status=status.data_ptr())), F.stream())
    assert status.item() == 0


@pytest.mark.parametrize("m,d,f", [(3, 4096, 520), (700, 520, 1032)])
def test_repeats_bit_for_bit(K, cuda, m, d, f):
    x, wg, wu = F.filled(normal(1, m, d), "bf16"), *(F.filled(normal(s, f, d, d ** -0.5), "bf16") for s in (2, 3))
    dh, first = F.filled(normal(4, m, f), "bf16"), None
    for _ in range(4):
        h, g, u = (F.matrix(m, f, "bf16") for _ in range(3))
        grads = [F.matrix(rows, d, "bf16") for rows in (m, f, f)]
        ws, status = F.workspace(K, "bf16", m, d, f), F.word()
        K.clpk_gated_ffn(C.byref(F.ffn_args("bf16", "silu", x, wg, wu, h, status, g, u)), F.stream())
        K.clpk_gated_ffn_backward(C.byref(F.backward_args("bf16", "silu", x, wg, wu, dh, g, u, *grads, ws, status)), F.stream())
        got = [h, g, u, *grads]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


@pytest.mark.parametrize("m", [2, 400])
def test_a_chain_of_calls_on_a_stream_of_its_own(K, cuda, m):
    """Each call reads what the one before it has just written: quantise, gated half, quantise, down projection."""
    d, f = 520, 1032
    x = F.filled(normal(1, m, d), "bf16")
    weights = [F.filled(normal(s, r, c, c ** -0.5), "bf16") for s, r, c in ((2, f, d), (3, f, d), (4, d, f))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s = side.cuda_stream
        for _ in range(3):
            q = [(F.matrix(*t.shape, "i8"), torch.empty(t.shape[0], device="cuda")) for t in [x, *weights]]
            for t, (qt, st) in zip([x, *weights], q):
                K.clpk_quantize_rows_i8(qt.data_ptr(), st.data_ptr(), t.data_ptr(), *t.shape, qt.stride(0), t.stride(0), N.DT_BF16, s)
            h, hq, hs = F.matrix(m, f, "bf16"), F.matrix(m, f, "i8"), torch.empty(m, device="cuda")
            y, status = F.matrix(m, d, "f32"), F.word()
            K.clpk_gated_ffn(C.byref(F.ffn_args("i8", "silu", q[0][0], q[1][0], q[2][0], h, status, scales=[q[i][1] for i in range(3)], out="bf16")), s)
            K.clpk_quantize_rows_i8(hq.data_ptr(), hs.data_ptr(), h.data_ptr(), m, f, hq.stride(0), h.stride(0), N.DT_BF16, s)
            K.clpk_gemm_i8_scaled(C.byref(F.linear_args(hq, q[3][0], y, hs, q[3][1], status, "f32")), s)
    side.synchronize()
    for t, (qt, st) in zip([x, *weights], q):
        want = F.quantize64(t)
        assert torch.equal(qt, want[0]) and torch.equal(st, want[1])
    F.check(h, *F.gated64("silu", q[0][0], q[1][0], q[2][0], "i8", "bf16", [q[i][1] for i in range(3)])[0], "h")
    want = F.quantize64(h)
    assert torch.equal(hq, want[0]) and torch.equal(hs, want[1])
    F.check(y, *F.linear64(hq, q[3][0], hs, q[3][1], "f32"), "y")


@pytest.mark.parametrize("m,log_pitch", [(3, 30), (130, 25)])
def test_rows_beyond_32_bits(K, cuda, m, log_pitch):
    """Tokens that lie more than 2^32 bytes into x, g, u, h and the gradients, for few of them and for many."""
    d, f, step = 72, 136, 1 << log_pitch

    def far(cols, fill):
        # columns of one allocation: a matrix of its own for each would not fit the card many times over
        far.at += 256
        return torch.as_strided(far.all, (m, cols), (step, 1), far.at - 256).copy_(fill) if fill is not None else torch.as_strided(far.all, (m, cols), (step, 1), far.at - 256)
    far.at, far.all = 0, torch.empty((m - 1) * step + 4096, dtype=torch.bfloat16, device="cuda")
    x, dh = far(d, normal(1, m, d)), far(f, normal(4, m, f))
    h, g, u, dx = far(f, None), far(f, None), far(f, None), far(d, None)
    wg, wu = (F.filled(normal(s, f, d, d ** -0.5), "bf16") for s in (2, 3))
    status = F.word()
    K.clpk_gated_ffn(C.byref(F.ffn_args("bf16", "silu", x, wg, wu, h, status, g, u)), F.stream())
    for got, want, name in zip((h, g, u), F.gated64("silu", x, wg, wu, "bf16", "bf16"), "hgu"):
        F.check(got, *want, name)
    dwg, dwu = (F.matrix(f, d, "bf16") for _ in range(2))
    ws = F.workspace(K, "bf16", m, d, f)
    K.clpk_gated_ffn_backward(C.byref(F.backward_args("bf16", "silu", x, wg, wu, dh, g, u, dx, dwg, dwu, ws, status)), F.stream())
    for got, want, name in zip((dx, dwg, dwu), F.backward64("silu", x, wg, wu, dh, g, u, "bf16"), ("dx", "dwg", "dwu")):
        F.check(got, *want, name)
    assert status.item() == 0


@pytest.mark.parametrize("m", [3, 300])
def test_scales_and_bias_at_any_word(K, cuda, m):
    """They are aligned to their elements and no further."""
    n, k = 200, 130
    a, b = F.filled(integers(1, m, k), "i8"), F.filled(integers(2, n, k), "i8")
    sa, sb, su = scales(3, m + 1, 0.02)[1:], scales(4, n + 3, 1e-3)[3:], scales(5, n + 2, 1e-3)[2:]
    bias = normal(5, 1, n + 1)[0].to(torch.bfloat16)[1:]
    c, status = F.matrix(m, n, "bf16"), F.word()
    K.clpk_gemm_i8_scaled(C.byref(F.linear_args(a, b, c, sa, sb, status, "bf16", bias)), F.stream())
    F.check(c, *F.linear64(a, b, sa, sb, "bf16", bias), "c")
    K.clpk_gated_ffn(C.byref(F.ffn_args("i8", "relu", a, b, b, c, status, scales=(sa, sb, su), out="bf16")), F.stream())
    F.check(c, *F.gated64("relu", a, b, b, "i8", "bf16", (sa, sb, su))[0], "h")


@pytest.mark.parametrize("m,d,f", [(2, 520, 1032), (300, 520, 1032), (1702, 8, 584)])
def test_calls_captured_in_a_graph(K, cuda, m, d, f):
    """Forward and backward captured once and replayed on inputs that have changed since."""
    x, wg, wu, dh = (F.matrix(r, c, "bf16") for r, c in ((m, d), (f, d), (f, d), (m, f)))
    h, g, u = (F.matrix(m, f, "bf16") for _ in range(3))
    grads = [F.matrix(rows, d, "bf16") for rows in (m, f, f)]
    ws, status = F.workspace(K, "bf16", m, d, f), F.word()
    xq, xs = F.matrix(m, d, "i8"), torch.empty(m, device="cuda")
    forward_args = F.ffn_args("bf16", "silu", x, wg, wu, h, status, g, u)
    backward_args = F.backward_args("bf16", "silu", x, wg, wu, dh, g, u, *grads, ws, status)

    def calls(s):
        K.clpk_quantize_rows_i8(xq.data_ptr(), xs.data_ptr(), x.data_ptr(), m, d, xq.stride(0), x.stride(0), N.DT_BF16, s)
        K.clpk_gated_ffn(C.byref(forward_args), s)
        K.clpk_gated_ffn_backward(C.byref(backward_args), s)
    for t in (x, wg, wu, dh):
        t.fill_(1)
    calls(F.stream())                                                   # what a first call sets up is not for a capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(F.stream())
    for seed in (1, 11):
        x.copy_(normal(seed, m, d))
        wg.copy_(normal(seed + 1, f, d, d ** -0.5))
        wu.copy_(normal(seed + 2, f, d, d ** -0.5))
        dh.copy_(normal(seed + 3, m, f, 0.1))
        graph.replay()
        torch.cuda.synchronize()
        want = F.quantize64(x)
        assert torch.equal(xq, want[0]) and torch.equal(xs, want[1])
        for got, w, name in zip((h, g, u), F.gated64("silu", x, wg, wu, "bf16", "bf16"), "hgu"):
            F.check(got, *w, name)
        for got, w, name in zip(grads, F.backward64("silu", x, wg, wu, dh, g, u, "bf16"), ("dx", "dwg", "dwu")):
            F.check(got, *w, name)
    assert status.item() == 0


def test_threads_with_streams_of_their_own(K, cuda):
    """Two host threads, each with its buffers: few tokens on one stream, many on the other, results as of one alone."""
    sizes, alone, failed = ((3, 1032, 2056), (400, 264, 1400)), [], []

    def buffers(i):
        m, d, f = sizes[i]
        x, wg, wu, dh = (F.filled(normal(10 * i + s, r, c, 0.1), "bf16") for s, r, c in ((1, m, d), (2, f, d), (3, f, d), (4, m, f)))
        return x, wg, wu, dh, [F.matrix(r, c, "bf16") for r, c in ((m, f), (m, f), (m, f), (m, d), (f, d), (f, d))], F.workspace(K, "bf16", m, d, f), F.word()

    def calls(b, s):
        x, wg, wu, dh, out, ws, status = b
        K.clpk_gated_ffn(C.byref(F.ffn_args("bf16", "silu", x, wg, wu, out[0], status, out[1], out[2])), s)
        K.clpk_gated_ffn_backward(C.byref(F.backward_args("bf16", "silu", x, wg, wu, dh, out[1], out[2], *out[3:], ws, status)), s)
    both = [buffers(0), buffers(1)]
    for b in both:
        calls(b, F.stream())
        torch.cuda.synchronize()
        alone.append([t.clone() for t in b[4]])

    def work(i):
        stream = torch.cuda.Stream()
        for _ in range(40):
            for t in both[i][4]:
                with torch.cuda.stream(stream):
                    t.zero_()
            calls(both[i], stream.cuda_stream)
            stream.synchronize()
            if both[i][6].item() != 0 or not all(torch.equal(a, t) for a, t in zip(alone[i], both[i][4])):
                failed.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


# ---- refusals ------------------------------------------------------------------------------------------------

def refused(call, args, text):
    with pytest.raises(N.ClpkError, match=text) as e:
        call(C.byref(args) if args is not None else None, None)
    assert e.value.code == N.ERR_BAD_ARG


def changed(args, **kw):
    new = type(args).from_buffer_copy(args)
    for name, v in kw.items():
        setattr(new, name, v)
    return new


def test_refusals_of_the_scaled_product(K, cuda):
    a, b, c = F.matrix(4, 64, "i8"), F.matrix(40, 64, "i8"), F.matrix(4, 40, "f32")
    s = torch.ones(64, device="cuda")
    good = F.linear_args(a, b, c, s, s, F.word(), "f32")
    at = a.data_ptr()
    for kw, text in [({"out_dtype": N.DT_I8}, "out_dtype"), ({"n": 0}, "only the number of tokens"), ({"k": 0}, "only the number of tokens"),
                     ({"k": 131072, "lda": 131072, "ldb": 131072}, "32-bit sum"), ({"d_a": None}, "d_a is NULL"), ({"d_b": None}, "d_b is NULL"),
                     ({"d_c": None}, "d_c is NULL"), ({"d_a": at + 1}, "d_a must start on 16"), ({"d_c": c.data_ptr() + 4}, "d_c must start on 16"),
                     ({"lda": 63}, "pitch of d_a"), ({"lda": 65}, "d_a must start"), ({"ldb": 72}, "d_b must start"), ({"ldc": 42}, "d_c must start"),
                     ({"lda": 1 << 36}, "too large"), ({"d_a_scale": None}, "d_a_scale"), ({"d_b_scale": s.data_ptr() + 2}, "d_b_scale"),
                     ({"d_bias": s.data_ptr() + 2}, "d_bias"), ({"d_status": None}, "d_status"), ({"m": 0xFFFFFFFF}, "too large"),
                     ({"m": 1 << 30, "n": 1 << 28, "ldc": 1 << 28}, "too large")]:
        refused(K.clpk_gemm_i8_scaled, changed(good, **kw), text)
    refused(K.clpk_gemm_i8_scaled, None, "args is NULL")


def test_refusals_of_the_gated_products(K, cuda):
    x, w, h = F.matrix(4, 64, "bf16"), F.matrix(40, 64, "bf16"), F.matrix(4, 40, "bf16")
    s = torch.ones(64, device="cuda")
    good = F.ffn_args("bf16", "silu", x, w, w, h, F.word())
    at = h.data_ptr()
    for kw, text in [({"dtype": N.DT_E4M3}, "dtype"), ({"activation": 5}, "activation"), ({"activation": -1}, "activation"), ({"f": 0}, "only the number"),
                     ({"d": 0}, "only the number"), ({"d_x": None}, "d_x is NULL"), ({"d_wg": None}, "d_wg is NULL"), ({"d_wu": None}, "d_wu is NULL"),
                     ({"d_h": None}, "d_h is NULL"), ({"d_wu": w.data_ptr() + 8}, "d_wu must start"), ({"ldx": 60}, "pitch of d_x"),
                     ({"ldw": 66}, "d_wg must start"), ({"ldh": 44}, "d_h must start"), ({"d_g": at}, "both, or neither"), ({"d_u": at}, "both, or neither"),
                     ({"d_g": at, "d_u": at + 2}, "d_u must start"), ({"d_status": None}, "d_status"),
                     ({"dtype": N.DT_I8, "out_dtype": N.DT_I8}, "out_dtype"), ({"dtype": N.DT_I8, "out_dtype": N.DT_BF16}, "d_x_scale"),
                     ({"dtype": N.DT_I8, "out_dtype": N.DT_BF16, "d_x_scale": s.data_ptr()}, "d_wg_scale"),
                     ({"dtype": N.DT_I8, "out_dtype": N.DT_BF16, "d_x_scale": s.data_ptr(), "d_wg_scale": s.data_ptr()}, "d_wu_scale"),
                     ({"dtype": N.DT_I8, "out_dtype": N.DT_BF16, "d_g": at, "d_u": at}, "not kept in 8 bits"),
                     ({"dtype": N.DT_I8, "out_dtype": N.DT_BF16, "d": 131072}, "32-bit sum")]:
        refused(K.clpk_gated_ffn, changed(good, **kw), text)
    refused(K.clpk_gated_ffn, None, "args is NULL")


def test_refusals_of_the_gradients(K, cuda):
    x, w, h = F.matrix(4, 64, "bf16"), F.matrix(40, 64, "bf16"), F.matrix(4, 40, "bf16")
    ws = F.workspace(K, "bf16", 4, 64, 40)
    good = F.backward_args("bf16", "silu", x, w, w, h, h, h, x, w, w, ws, F.word())
    for kw, text in [({"dtype": N.DT_I8}, "dtype"), ({"activation": 9}, "activation"), ({"f": 0}, "only the number"), ({"d_dh": None}, "d_dh is NULL"),
                     ({"d_g": None}, "d_g is NULL"), ({"d_u": None}, "d_u is NULL"), ({"d_wg": None}, "d_wg is NULL"), ({"d_wu": None}, "d_wu is NULL"),
                     ({"d_x": None}, "d_x is NULL"), ({"d_dwg": None}, "both, or neither"), ({"d_dwu": None}, "both, or neither"),
                     ({"workspace_bytes": ws.numel() // 2}, "workspace of"), ({"d_workspace": None}, "workspace of"),
                     ({"d_workspace": ws.data_ptr() + 8}, "workspace of"), ({"ldh": 41}, "d_dh must start"), ({"ldx": 8}, "pitch of d_dx"),
                     ({"d_status": None}, "d_status")]:
        refused(K.clpk_gated_ffn_backward, changed(good, **kw), text)
    refused(K.clpk_gated_ffn_backward, None, "args is NULL")
    with pytest.raises(N.ClpkError, match="dtype"):
        K.clpk_gated_ffn_backward_workspace_bytes(N.DT_F32, 1, 1, 1, C.byref(C.c_size_t(0)))


# ---- choices and row ends that the sizes above do not reach -------------------------------------------------

# a width of 64 columns with K in two and four ranges, 128 and 192 in two, and several tiles a cluster at 192
@pytest.mark.parametrize("m,d,f", [(4100, 4090, 7), (129, 2559, 7), (4100, 6397, 39), (257, 6397, 1399), (257, 63, 5999)])
def test_gated_in_every_width(K, cuda, m, d, f):
    forward(K, "bf16", "silu", m, d, f, pad=m % 2, keep=f < 1000)
    gated_i8(K, "bf16", m, 2 * d, f)


@pytest.mark.parametrize("m,k,n", [(4100, 8190, 7), (129, 5119, 7), (2049, 12799, 263), (257, 12799, 2711), (257, 127, 13999)])
def test_scaled_product_in_every_width(K, cuda, m, k, n):
    scaled(K, "f16", m, k, n)


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("n", [*range(1, 18), 23, 31, 33, 34, 47, 63, 65, 100, 129, 250])
def test_rows_that_end_anywhere(K, cuda, out, n):
    """The last 16 bytes of a row, whole or in part, in each place of a box, with rows that end a tile early."""
    scaled(K, out, 150, 200, n)
    if out == "bf16":
        forward(K, out, "sigmoid", 150, 72, n, pad=n % 2, keep=True)
        backward(K, out, "relu", 150, n, 40)


# ---- gradients that are not finite --------------------------------------------------------------------------------

@pytest.mark.parametrize("act", sorted(F.ACTS))
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,d,f", [(9, 33, 40), (300, 520, 1032), (100, 64, 1000)])
def test_a_nan_stays_one_through_the_backward_pass(K, cuda, act, dtype, m, d, f):
    """A NaN in g, u or dh of one token and feature: dg and du of it are NaN as far as they depend on it, and with them the token's row
    of dx and the feature's row of dWg or dWu; everything else is finite."""
    for bad, to_dg, to_du in (("g", True, True), ("u", True, False), ("dh", True, True)):
        x = F.filled(normal(1, m, d), dtype)
        wg, wu = (F.filled(normal(s, f, d, d ** -0.5), dtype) for s in (2, 3))
        kept = {"dh": normal(4, m, f, 0.1), "g": normal(5, m, f), "u": normal(6, m, f)}
        kept[bad][3, 7] = float("nan")
        kept = {n: F.filled(t, dtype) for n, t in kept.items()}
        dx, dwg, dwu = (F.matrix(rows, d, dtype) for rows in (m, f, f))
        ws, status = F.workspace(K, dtype, m, d, f), F.word()
        K.clpk_gated_ffn_backward(C.byref(F.backward_args(dtype, act, x, wg, wu, kept["dh"], kept["g"], kept["u"], dx, dwg, dwu, ws, status)), F.stream())
        for got, row, nan in ((dx, 3, True), (dwg, 7, to_dg), (dwu, 7, to_du)):
            want = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
            want[row] = nan
            assert torch.equal(torch.isnan(got), want) and torch.equal(~torch.isfinite(got), want), (bad, row)
        assert status.item() == 0


@pytest.mark.parametrize("act", sorted(F.ACTS))
def test_gates_far_from_zero(K, cuda, act):
    """Where an activation is its argument, or nothing, so is its derivative 1 or 0, up to the largest numbers of the type."""
    m, d, f = 8, 16, 24
    x, w = F.filled(normal(1, m, d), "bf16"), F.filled(normal(2, f, d, 0.25), "bf16")
    size = torch.tensor([40.0, 100.0, 1e4, 1e10, 1e19, 1e25, 1e30, 3e38], device="cuda")[:, None]
    sign = torch.where(torch.arange(f, device="cuda") % 2 == 0, 1.0, -1.0)
    g, u, dh = F.filled(size * sign, "bf16"), F.filled(torch.full((m, f), 0.5, device="cuda"), "bf16"), F.filled(torch.full((m, f), 2.0 ** -130, device="cuda"), "bf16")
    dx, dwg, dwu = F.matrix(m, d, "bf16"), F.matrix(f, d, "bf16"), F.matrix(f, d, "bf16")
    ws, status = F.workspace(K, "bf16", m, d, f), F.word()
    K.clpk_gated_ffn_backward(C.byref(F.backward_args("bf16", act, x, w, w, dh, g, u, dx, dwg, dwu, ws, status)), F.stream())
    for t in (dx, dwg, dwu):
        assert bool(torch.isfinite(t).all())
    if act != "sigmoid":                                        # there a is 1 or 0 and its derivative 0
        assert not dwg[1::2].any() and not dwu[1::2].any()
    assert status.item() == 0


# ---- the choices that the lists above leave out (tests/test_cpu_feed_forward_plans.py says which there are) ---------------

PAIRS_GATED, PAIRS_GATED_8 = [(9804, 2, 138), (99, 3, 4743)], [(9616, 3, 130), (100, 3, 4761)]
PAIRS_SCALED = [(9675, 2, 266)]
# every number of parts of dx and of dW in tiles of 128 and of 256 columns, with the longer sum in either
PARTS_BACKWARD = [(6083, 2, 196), (8137, 2, 196), (1345, 2, 1), (12939, 2, 258), (1475, 2, 1), (16341, 2, 1), (1998, 3, 193), (3017, 2, 1), (3091, 2, 197),
                  (4045, 2, 1), (4167, 2, 193), (519, 2, 3059), (2, 2, 3015), (1076, 2, 5637), (792, 2, 722), (2, 2, 642), (590, 3, 6430), (2, 2, 6249),
                  (2, 2, 12806), (516, 2, 982), (517, 2, 1491), (2, 2, 1489), (516, 3, 1988), (2, 2, 1986), (6663, 129, 1), (6608, 134, 207), (8660, 133, 1),
                  (8965, 142, 193), (4657, 1289, 1), (5477, 132, 1360), (2635, 777, 1), (3900, 279, 604), (2765, 522, 1), (4952, 145, 593), (3437, 398, 1),
                  (3356, 385, 220), (4807, 270, 1), (5453, 145, 261), (523, 139, 3369), (2, 129, 3746), (2, 130, 4117), (2, 132, 6140), (1230, 302, 1819),
                  (2, 1211, 1124), (1325, 133, 2577), (592, 257, 1824), (769, 146, 3223)]


@pytest.mark.parametrize("m,d,f", PARTS_BACKWARD)
def test_backward_in_every_number_of_parts(K, cuda, m, d, f):
    backward(K, "bf16", "silu", m, d, f, pad=m % 2)


@pytest.mark.parametrize("i", range(2))
def test_gated_pairs_of_every_width(K, cuda, i):
    forward(K, "bf16", "silu", *PAIRS_GATED[i], 0, True)
    gated_i8(K, "f32", *PAIRS_GATED_8[i])
    scaled(K, "bf16", *PAIRS_SCALED[0])


def test_gradients_beyond_the_range_of_fp16(K, cuda):
    """dg = dh * u is rounded to fp16 on the way: beyond 65504 it is an infinity and below 2^-25 nothing, though dWg = dg^T x has room
    for what it would be; dh times a power of two (and the gradients divided by it) is the caller's way out."""
    m, d, f = 4, 16, 8

    def dwg(dh, u, x):
        g = F.filled(torch.full((m, f), 2.0, device="cuda"), "f16")
        x, dh, u = (F.filled(torch.full(s, v, device="cuda"), "f16") for s, v in (((m, d), x), ((m, f), dh), ((m, f), u)))
        w = F.filled(torch.ones(f, d, device="cuda"), "f16")
        out, ws, status = [F.matrix(r, d, "f16") for r in (m, f, f)], F.workspace(K, "f16", m, d, f), F.word()
        K.clpk_gated_ffn_backward(C.byref(F.backward_args("f16", "relu", x, w, w, dh, g, u, *out, ws, status)), F.stream())
        assert status.item() == 0 and bool((out[2] == 4 * 2 * dh[0, 0] * x[0, 0]).all())
        return out[1]
    assert bool((dwg(300.0, 256.0, 2.0 ** -10) == float("inf")).all())                       # 4 * 76800 / 1024 = 300
    assert bool((dwg(75.0, 256.0, 2.0 ** -10) == 75).all())
    assert not dwg(2.0 ** -14, 2.0 ** -12, 1024.0).any()                                     # 2^-14
    assert bool((dwg(2.0 ** -8, 2.0 ** -12, 1024.0) == 2.0 ** -8).all())
