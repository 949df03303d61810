"""Plain 64-bit forms of the feed-forward operators, and how far a kernel may be from them.

What a kernel may be off is counted from what it does, element by element:

* a sum of K products in fp32, added in steps of 16 by the tensor cores with truncation: (K / 16 + 8) roundings of 2^-22 of the
  sum of magnitudes;
* an activation in fp32: 4e-6 of its argument (fast exp, division and their arguments' rounding);
* a rounding to 16 bits: half a place, 2^-8 (bf16) or 2^-11 (fp16, 2^-25 below its normal numbers) of the value.
"""
import ctypes as C
import math

import torch

from clpeak_b200 import native as N

DT = {"bf16": N.DT_BF16, "f16": N.DT_F16, "f32": N.DT_F32, "i8": N.DT_I8}
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "i8": torch.int8}
ROUND = {"bf16": (2.0 ** -8, 2.0 ** -134), "f16": (2.0 ** -11, 2.0 ** -25), "f32": (2.0 ** -24, 2.0 ** -150)}
ACTS = {"silu": N.ACT_SILU, "gelu_tanh": N.ACT_GELU_TANH, "gelu": N.ACT_GELU, "relu": N.ACT_RELU, "sigmoid": N.ACT_SIGMOID}
SENTINEL = 77                                   # what lies behind the rows of an output


def matrix(rows, cols, dtype, pad=0, fill=SENTINEL):
    """[rows][cols] whose rows lie at multiples of 16 bytes, `pad` of them further apart than they must; `fill` between them."""
    t = TORCH[dtype]
    unit = 16 // t.itemsize
    step = -(-cols // unit) * unit + pad * unit
    return torch.full((max(rows, 1), step), fill, dtype=t, device="cuda")[:rows, :cols]


def filled(values, dtype, pad=0):
    """The values as an operand; NaN (127 in 8 bits) behind its rows, which no result may see."""
    out = matrix(values.shape[0], values.shape[1], dtype, pad, 127 if dtype == "i8" else float("nan"))
    out.copy_(values)
    return out


def behind(t):
    """What lies behind the rows of a matrix made here."""
    return torch.as_strided(t, (t.shape[0], t.stride(0) - t.shape[1]), (t.stride(0), 1), t.shape[1]) if t.shape[0] else t


def untouched(t):
    return bool((behind(t) == SENTINEL).all())


def act64(act, g):
    if act == "silu":
        return g * torch.sigmoid(g)
    if act == "sigmoid":
        return torch.sigmoid(g)
    if act == "relu":
        return torch.relu(g)
    if act == "gelu":
        return 0.5 * g * (1 + torch.erf(g / math.sqrt(2)))
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))


def both64(act, g):
    g = g.detach().clone().requires_grad_()
    a = act64(act, g)
    return a.detach(), torch.autograd.grad(a.sum(), g)[0]


def rounded(value, dtype):
    """Half a place of `value` in a type."""
    rel, least = ROUND[dtype]
    return value.abs() * rel + least


def sums(k):
    return (k / 16 + 8) * 2.0 ** -22


def check(got, want, allowed, what=""):
    got = got.double()
    assert got.shape == want.shape
    off = (got - want).abs()
    bad = ~(off <= allowed)
    if bad.any():
        at = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} beyond what is allowed, first at {at}: got {float(got[at])!r}, "
                             f"want {float(want[at])!r}, allowed {float(allowed[at]):.3g}")


def stream():
    return torch.cuda.current_stream().cuda_stream


def word():
    return torch.full((1,), -1, dtype=torch.int32, device="cuda")


# ---- forward -------------------------------------------------------------------------------------------

def ffn_args(dtype, act, x, wg, wu, h, status, g=None, u=None, scales=None, out=None):
    m, d = x.shape
    args = N.GatedFfnArgs(dtype=DT[dtype], out_dtype=DT[out or dtype], activation=ACTS[act], m=m, d=d, f=wg.shape[0],
                          d_x=x.data_ptr(), d_wg=wg.data_ptr(), d_wu=wu.data_ptr(), d_h=h.data_ptr(),
                          ldx=x.stride(0), ldw=wg.stride(0), ldh=h.stride(0), d_status=status.data_ptr())
    if g is not None:
        args.d_g, args.d_u = g.data_ptr(), u.data_ptr()
    if scales is not None:
        args.d_x_scale, args.d_wg_scale, args.d_wu_scale = (t.data_ptr() for t in scales)
    return args


def gated64(act, x, wg, wu, dtype, out, scales=None):
    """h, g, u in 64 bits and what each may be off."""
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.T, x @ wu.T
    if scales is None:
        eg, eu = (sums(x.shape[1]) * (x.abs() @ w.abs().T) for w in (wg, wu))
    else:                                       # the sum is exact; its conversion and two products are rounded
        sx, sg, su = (t.double() for t in scales)
        g, u = g * sx[:, None] * sg, u * sx[:, None] * su
        eg, eu = 3 * 2.0 ** -24 * g.abs(), 3 * 2.0 ** -24 * u.abs()
    a = act64(act, g)
    eh = 1.13 * eg * u.abs() + (a.abs() + 1.13 * eg) * eu + 4e-6 * (g.abs() + (act == "sigmoid")) * u.abs()
    h = a * u
    return (h, eh + rounded(h, out)), (g, eg + rounded(g, out)), (u, eu + rounded(u, out))


# ---- backward ------------------------------------------------------------------------------------------

def backward_args(dtype, act, x, wg, wu, dh, g, u, dx, dwg, dwu, workspace, status):
    m, d = x.shape
    ptr = lambda t: None if t is None else t.data_ptr()                  # noqa: E731
    return N.GatedFfnBackwardArgs(dtype=DT[dtype], activation=ACTS[act], m=m, d=d, f=wg.shape[0], d_x=ptr(x), d_wg=ptr(wg),
                                  d_wu=ptr(wu), d_dh=ptr(dh), d_g=ptr(g), d_u=ptr(u), d_dx=ptr(dx), d_dwg=ptr(dwg), d_dwu=ptr(dwu),
                                  ldx=x.stride(0), ldw=wg.stride(0), ldh=dh.stride(0), d_workspace=workspace.data_ptr(),
                                  workspace_bytes=workspace.numel(), d_status=status.data_ptr())


def workspace(K, dtype, m, d, f):
    need = C.c_size_t(0)
    K.clpk_gated_ffn_backward_workspace_bytes(DT[dtype], m, d, f, C.byref(need))
    return torch.empty(max(need.value, 16), dtype=torch.uint8, device="cuda")


def backward64(act, x, wg, wu, dh, g, u, dtype):
    """dx, dWg, dWu in 64 bits and what each may be off."""
    x, wg, wu, dh, g, u = (t.double() for t in (x, wg, wu, dh, g, u))
    a, da = both64(act, g)
    dg, du = dh * u * da, dh * a
    # in fp32, then rounded to the operands' type; a derivative has a few places more than its activation
    eg = 1e-5 * (dh * u).abs() * (1 + g.abs() * da.abs()) + rounded(dg, dtype)
    eu = 4e-6 * dh.abs() * (g.abs() + 1) + rounded(du, dtype)
    m, f, d = x.shape[0], g.shape[1], x.shape[1]

    def product(pairs, k):
        want = sum(p @ q for p, _, q in pairs)
        off = sum(e @ q.abs() + sums(k) * ((p.abs() + e) @ q.abs()) for p, e, q in pairs)
        return want, off + rounded(want, dtype)
    return (product([(dg, eg, wg), (du, eu, wu)], 2 * f), product([(dg.T, eg.T, x)], m), product([(du.T, eu.T, x)], m))


# ---- 8 bits --------------------------------------------------------------------------------------------

def linear_args(a, b, c, sa, sb, status, out, bias=None):
    return N.GemmI8ScaledArgs(m=a.shape[0], n=b.shape[0], k=a.shape[1], out_dtype=DT[out], d_a=a.data_ptr(), d_b=b.data_ptr(),
                              d_c=c.data_ptr(), lda=a.stride(0), ldb=b.stride(0), ldc=c.stride(0), d_a_scale=sa.data_ptr(),
                              d_b_scale=sb.data_ptr(), d_bias=None if bias is None else bias.data_ptr(), d_status=status.data_ptr())


def linear64(a, b, sa, sb, out, bias=None):
    c = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()
    off = 3 * 2.0 ** -24 * c.abs()
    if bias is not None:
        c = c + bias.double()
        off = off + 2.0 ** -24 * (c.abs() + off)
    return c, off + rounded(c, out)


def quantize64(x):
    """The quantiser's own arithmetic, element by element in fp32: its results have one value."""
    x = x.float()
    top = x.abs().amax(1) if x.shape[1] else torch.zeros(x.shape[0], device=x.device)
    finite = torch.isfinite(x).all(1)
    scale = top / torch.tensor(127.0, device=x.device)
    scale = torch.where(scale < 2.0 ** -126, torch.zeros_like(scale), scale)
    r = torch.where(scale > 0, 1 / scale, torch.zeros_like(scale))
    r = torch.where(finite, r, torch.zeros_like(r))
    q = torch.where(finite[:, None], torch.round(torch.nan_to_num(x, 0, 0, 0) * r[:, None]), torch.zeros_like(x))
    return q.to(torch.int8), torch.where(finite, scale, torch.full_like(scale, float("nan")))
