"""Plain forms of the operators that train a block, and how far a kernel may be from them.

Layer norm: 64 bits, and what fp32 may be off, element by element.  u = 2^-24 is half a place.  A sum whose longest chain of
additions is `depth` is off by depth * u times the sum of magnitudes; the rest is counted where it is computed.
AdamW: the same operations in torch, each rounded to fp32: results have one value."""
import ctypes as C
import math

import torch

from clpeak_b200 import native as N
from tests import ff_util as F

U = 2.0 ** -24


# ---- layer norm ----------------------------------------------------------------------------------------------

def norm_args(x, y, weight=None, bias=None, mean=None, rstd=None, eps=1e-5, dtype="bf16", wdtype="f32"):
    ptr = lambda t: None if t is None else t.data_ptr()                  # noqa: E731
    return N.LayerNormArgs(dtype=F.DT[dtype], weight_dtype=F.DT[wdtype], m=x.shape[0], d=x.shape[1], d_x=ptr(x), d_weight=ptr(weight), d_bias=ptr(bias),
                           d_y=ptr(y), d_mean=ptr(mean), d_rstd=ptr(rstd), ldx=x.stride(0), ldy=y.stride(0), eps=eps)


def norm_backward_args(x, dy, mean, rstd, weight, dx, dweight, dbias, workspace, dtype, wdtype):
    ptr = lambda t: None if t is None else t.data_ptr()                  # noqa: E731
    return N.LayerNormBackwardArgs(dtype=F.DT[dtype], weight_dtype=F.DT[wdtype], m=x.shape[0], d=x.shape[1], d_x=ptr(x), d_weight=ptr(weight), d_dy=ptr(dy),
                                   d_mean=ptr(mean), d_rstd=ptr(rstd), d_dx=ptr(dx), d_dweight=ptr(dweight), d_dbias=ptr(dbias), ldx=x.stride(0),
                                   lddy=dy.stride(0), lddx=dx.stride(0) if dx is not None else 0, d_workspace=ptr(workspace),
                                   workspace_bytes=workspace.numel() if workspace is not None else 0)


def norm_workspace(K, m, d):
    need = C.c_size_t(0)
    K.clpk_layer_norm_backward_workspace_bytes(m, d, C.byref(need))
    return torch.full((max(need.value, 16),), 255, dtype=torch.uint8, device="cuda")


def row_depth(d):
    """Additions in a row's longest chain: a thread's share, 32 elements or all it comes to in a CTA of 256 threads, and ten halvings."""
    return max(32, -(-d // 256)) + 12


def norm64(x, weight, bias, eps, dtype):
    """(y, mean, rstd) in 64 bits, each with what it may be off."""
    x = x.double()
    d = x.shape[1]
    w = torch.ones(d, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    b = torch.zeros_like(w) if bias is None else bias.double()
    mean = x.mean(1, keepdim=True)
    off = x - mean
    var = (off * off).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    depth = row_depth(d)
    e_mean = (depth * x.abs().mean(1, keepdim=True) + mean.abs()) * U
    # about a mean that is off the squares' sum is larger by its square; each difference and the root, quotient and sums are rounded
    e_rstd = rstd * (0.5 * ((depth + 6) * U + (e_mean * e_mean + 2 * U * e_mean * off.abs().mean(1, keepdim=True)) / (var + eps)) + 4 * U)
    y = off * rstd * w + b
    e_y = w.abs() * (rstd * e_mean + off.abs() * (e_rstd + 3 * U * rstd)) + 2 * U * (y.abs() + b.abs())
    e_y = 1.01 * e_y
    return (y, e_y + F.rounded(y.abs() + e_y, dtype)), (mean[:, 0], 1.01 * e_mean[:, 0]), (rstd[:, 0], 1.01 * e_rstd[:, 0])


def norm_backward64(x, dy, mean, rstd, weight, dtype, wdtype):
    """(dx, dweight, dbias) in 64 bits from the mean and rstd as they are, each with what it may be off."""
    x, dy, mean, rstd = x.double(), dy.double(), mean.double()[:, None], rstd.double()[:, None]
    m, d = x.shape
    w = torch.ones(d, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    hat = (x - mean) * rstd
    g = dy * w
    c1, c2 = g.mean(1, keepdim=True), (g * hat).mean(1, keepdim=True)
    dx = rstd * (g - c1 - hat * c2)
    depth = row_depth(d)
    e1, e2 = (depth + 3) * U * g.abs().mean(1, keepdim=True), (depth + 5) * U * (g * hat).abs().mean(1, keepdim=True)
    e_dx = 1.01 * rstd * (e1 + hat.abs() * e2 + 5 * U * (g.abs() + c1.abs() + (hat * c2).abs()))
    # down the columns: a chain of at most all rows, and what joins the parts
    rows = (m + 80) * U
    dw, db = (dy * hat).sum(0), dy.sum(0)
    e_dw, e_db = 1.01 * (rows + 3 * U) * (dy * hat).abs().sum(0), 1.01 * rows * dy.abs().sum(0)
    return (dx, e_dx + F.rounded(dx.abs() + e_dx, dtype)), (dw, e_dw + F.rounded(dw.abs() + e_dw, wdtype)), (db, e_db + F.rounded(db.abs() + e_db, wdtype))


# ---- AdamW ---------------------------------------------------------------------------------------------------

STATE = {"f32": (torch.float32, torch.float32), "i8": (torch.int8, torch.uint8)}


class Tensor:
    """One tensor of a step with its gradient and moments; `shift`: elements that every array begins behind a multiple of 16 bytes."""

    def __init__(self, gen, n, dtype, grad, state, master, shift=0):
        self.n, self.state, self.blocks = n, state, -(-n // N.ADAMW_BLOCK)
        self.whole = {}

        def array(name, values, t):
            whole = torch.full((n + shift + 24,), 77, dtype=t, device="cuda")
            whole[shift:shift + n] = values.to(t)
            self.whole[name] = whole
            return whole[shift:shift + n]
        normal = lambda std: torch.randn(n, generator=gen, device="cuda") * std     # noqa: E731
        spread = torch.exp(2 * torch.randn(n, generator=gen, device="cuda"))
        value = normal(0.05)
        self.param = array("param", value, F.TORCH[dtype])
        self.master = array("master", value, torch.float32) if master else None
        self.grad = array("grad", normal(1e-2) * spread, F.TORCH[grad])
        if state == "f32":
            self.m, self.v = array("m", normal(1e-3), torch.float32), array("v", normal(1e-3) ** 2, torch.float32)
            self.m_scale = self.v_scale = None
        else:
            whole = lambda lo, hi: torch.randint(lo, hi, (n,), generator=gen, device="cuda")  # noqa: E731
            self.m, self.v = array("m", whole(-127, 128), torch.int8), array("v", whole(0, 256), torch.uint8)
            scales = lambda top: (torch.rand(self.blocks, generator=gen, device="cuda") + 0.5) * 1e-3 / top     # noqa: E731
            self.m_scale, self.v_scale = scales(127 ** 2), scales(255 ** 2)
            self.whole["m_scale"] = torch.cat((self.m_scale, torch.full((3,), 77.0, device="cuda")))
            self.whole["v_scale"] = torch.cat((self.v_scale, torch.full((3,), 77.0, device="cuda")))
            self.m_scale, self.v_scale = self.whole["m_scale"][:self.blocks], self.whole["v_scale"][:self.blocks]
        self.shift = shift

    def entry(self):
        ptr = lambda t: None if t is None else t.data_ptr()                  # noqa: E731
        return N.AdamwTensor(n=self.n, d_param=ptr(self.param), d_grad=ptr(self.grad), d_master=ptr(self.master), d_m=ptr(self.m), d_v=ptr(self.v),
                             d_m_scale=ptr(self.m_scale), d_v_scale=ptr(self.v_scale))

    def values(self):
        return {name: getattr(self, name).clone() for name in ("param", "master", "m", "v", "m_scale", "v_scale") if getattr(self, name) is not None}

    def untouched(self):
        """Nothing around the arrays was written."""
        for name, whole in self.whole.items():
            if name.endswith("scale"):
                ok = bool((whole[self.blocks:] == 77).all())
            else:
                ok = bool((whole[:self.shift] == 77).all()) and bool((whole[self.shift + self.n:] == 77).all())
            if not ok:
                return False
        return True


def adamw_args(tensors, dtype, grad, state, lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, step=3, **more):
    table = (N.AdamwTensor * max(1, len(tensors)))(*[t.entry() for t in tensors])
    args = N.AdamwArgs(dtype=F.DT[dtype], grad_dtype=F.DT[grad], state_dtype=F.DT[state], count=len(tensors), h_tensors=C.addressof(table), lr=lr, beta1=beta1,
                       beta2=beta2, eps=eps, weight_decay=weight_decay, step=step, **more)
    args.table = table                              # lives as long as what points to it
    return args


def in_blocks(v):
    n = v.numel()
    blocks = -(-n // N.ADAMW_BLOCK)
    out = torch.zeros(blocks * N.ADAMW_BLOCK, device=v.device)
    out[:n] = v
    return out.view(blocks, N.ADAMW_BLOCK)


def codes(size, steps):
    """Scales and codes of sizes >= 0, by blocks; codes as a flat array with whole blocks."""
    size = in_blocks(size)
    finite = torch.isfinite(size).all(1)
    scale = torch.nan_to_num(size, 0, 0, 0).amax(1) / torch.full((), float(steps) ** 2, device=size.device)
    scale = torch.where(scale < 2.0 ** -126, torch.zeros_like(scale), scale)
    scale = torch.where(finite, scale, torch.full_like(scale, math.nan))
    inverse = torch.where(scale > 0, 1 / scale, torch.zeros_like(scale))
    q = torch.round(torch.sqrt(torch.nan_to_num(size, 0, 0, 0) * inverse[:, None]))
    return scale, torch.where(finite[:, None], q, torch.zeros_like(q)).flatten()


def step_off(p, update):
    """What a parameter may be off in fp32 with moments in 8 bits.  A root that is 2^-23 off, a product and a sum (2^-24 each) make the
    quotient's lower side 2^-22 off, its reciprocal 2^-23 more, the two products behind it 2^-24 each; the plain form has five
    roundings of 2^-24 there: less than 2^-20 of the update in all.  The last sum is rounded on either side."""
    return 2.0 ** -20 * update.double().abs() + 2 * U * p.double().abs() + 2.0 ** -149


def same_step(got, want):
    """Equal, bit for bit, and parameters with moments in 8 bits as near as step_off says; one of 16 bits besides by a place, where its
    rounding falls to the other side."""
    want = dict(want)
    off = want.pop("off", None)
    if off is not None:
        for name in ("param", "master"):
            if name not in want:
                continue
            a, b = got[name], want.pop(name)
            assert a.dtype == b.dtype and a.shape == b.shape
            assert torch.equal(torch.isfinite(a), torch.isfinite(b)) and torch.equal(torch.isnan(a), torch.isnan(b))
            fine = torch.isfinite(b)
            place = 0 if b.dtype == torch.float32 else 2 * F.rounded(b.double(), "bf16" if b.dtype == torch.bfloat16 else "f16")
            F.check(torch.where(fine, a, torch.zeros_like(a)), torch.where(fine, b, torch.zeros_like(b)).double(), torch.nan_to_num(off + place, 0, 0, 0), name)
    same(got, want)


def adamw_plain(t, lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, step=3, grad_scale=None):
    """What one step makes of a Tensor: its values by name."""
    p = t.master.clone() if t.master is not None else t.param.float()
    g, m, v = t.grad.float(), t.m.float(), t.v.float()
    if t.state == "i8":
        each = lambda s: s.repeat_interleave(N.ADAMW_BLOCK)[:t.n]            # noqa: E731
        m = (m * m.abs()) * each(t.m_scale)
        root = (v * v) * each(t.v_scale)
        v = root * root
    if grad_scale is not None:
        g = g * grad_scale
    m = m * beta1 + g * (1 - beta1)
    v = v * beta2 + (g * g) * (1 - beta2)
    root = torch.sqrt(v)
    c1, c2 = -math.expm1(step * math.log(beta1)) if beta1 else 1.0, -math.expm1(step * math.log(beta2)) if beta2 else 1.0
    update = (m / (root * (1 / math.sqrt(c2)) + eps)) * (lr / c1)
    p = p * (1 - lr * weight_decay) - update
    out = {"param": p.to(t.param.dtype)}
    if t.master is not None:
        out["master"] = p
    if t.state == "f32":
        return dict(out, m=m, v=v)
    out["off"] = step_off(p, update)
    out["m_scale"], q = codes(m.abs(), 127)
    out["m"] = (q[:t.n] * torch.sign(torch.nan_to_num(m))).to(torch.int8)
    out["v_scale"], q = codes(root, 255)
    some = (root > 0) & (out["v_scale"].repeat_interleave(N.ADAMW_BLOCK)[:t.n] > 0)
    out["v"] = torch.where(some, q[:t.n].clamp(min=1), q[:t.n]).to(torch.uint8)
    return out


def same(got, want):
    """Bit for bit, any NaN for any other."""
    for name in want:
        a, b = got[name], want[name]
        assert a.shape == b.shape and a.dtype == b.dtype, name
        if a.is_floating_point():
            differ = ~((a == b) | (torch.isnan(a) & torch.isnan(b)))
        else:
            differ = a != b
        if differ.any():
            at = int(differ.nonzero()[0])
            raise AssertionError(f"{name}: {int(differ.sum())} of {a.numel()} differ, first at {at}: {a[at].item()!r}, want {b[at].item()!r}")


# ---- products of groups ----------------------------------------------------------------------------------------

def grouped_workspace(K, groups=1):
    need = C.c_size_t(0)
    K.clpk_grouped_gemm_workspace_bytes(groups, C.byref(need))
    return torch.full((need.value,), 255, dtype=torch.uint8, device="cuda")


def offsets_of(rows, first=0):
    return torch.tensor([first] + list(rows), device="cuda").cumsum(0).to(torch.int32)


def grouped_args(a, w, c, offsets, workspace, status, dtype, out, n):
    groups = offsets.numel() - 1
    return N.GroupedGemmArgs(dtype=F.DT[dtype], out_dtype=F.DT[out], m=a.shape[0], n=n, k=a.shape[1], groups=groups, d_a=a.data_ptr(), d_w=w.data_ptr(),
                             d_offsets=offsets.data_ptr(), d_c=c.data_ptr(), lda=a.stride(0), ldw=w.stride(1), stride_w=w.stride(0), ldc=c.stride(0),
                             d_workspace=workspace.data_ptr(), workspace_bytes=workspace.numel(), d_status=status.data_ptr())


def grouped_backward_args(a, w, dc, da, dw, offsets, workspace, status, dtype, out, n):
    ptr = lambda t: None if t is None else t.data_ptr()                  # noqa: E731
    args = N.GroupedGemmBackwardArgs(dtype=F.DT[dtype], dw_dtype=F.DT[out], m=a.shape[0], n=n, k=a.shape[1], groups=offsets.numel() - 1, d_a=ptr(a), d_w=ptr(w),
                                     d_offsets=ptr(offsets), d_dc=ptr(dc), d_da=ptr(da), d_dw=ptr(dw), lda=a.stride(0), ldw=w.stride(1), stride_w=w.stride(0),
                                     lddc=dc.stride(0), d_workspace=ptr(workspace), workspace_bytes=workspace.numel(), d_status=ptr(status))
    if da is not None:
        args.ldda = da.stride(0)
    if dw is not None:
        args.lddw, args.stride_dw = dw.stride(1), dw.stride(0)
    return args


def weights3(groups, n, k, dtype, pad=0, between=0, values=None, fill=F.SENTINEL):
    """[groups][n][k] whose rows lie at multiples of 16 bytes and whose matrices lie `between` multiples of 16 bytes apart."""
    t = F.TORCH[dtype]
    unit = 16 // t.itemsize
    step = -(-k // unit) * unit + pad * unit
    stride = n * step + between * unit
    whole = torch.full((groups * stride,), fill, dtype=t, device="cuda")
    out = torch.as_strided(whole, (groups, n, k), (stride, step, 1))
    if values is not None:
        out.copy_(values)
    return out


def around(t):
    """What lies around the elements of a matrix of weights3."""
    whole = torch.as_strided(t, (t.shape[0] * t.stride(0),), (1,))
    left = torch.ones_like(whole, dtype=torch.bool)
    torch.as_strided(left, tuple(t.shape), t.stride()).fill_(False)
    return whole[left]


def grouped64(a, w, rows, first, out):
    """C's rows of all groups in 64 bits, and what each element may be off: the tensor cores' sums, parts of which are added in fp32."""
    want, off, at = [], [], first
    for e, r in enumerate(rows):
        x, y = a[at:at + r].double(), w[e].double()
        want.append(x @ y.T)
        off.append((F.sums(a.shape[1]) + 75 * U) * (x.abs() @ y.abs().T))
        at += r
    want, off = torch.cat(want), torch.cat(off)
    return want, off + F.rounded(want.abs() + off, out)


def grouped_backward64(a, w, dc, rows, first, dtype, out):
    """(dA of all groups' rows, dW) in 64 bits, each with what it may be off."""
    da, e_da, dw, e_dw, at = [], [], [], [], first
    for e, r in enumerate(rows):
        x, y, g = a[at:at + r].double(), w[e].double(), dc[at:at + r].double()
        da.append(g @ y)
        e_da.append((F.sums(w.shape[1]) + 75 * U) * (g.abs() @ y.abs()))
        dw.append(g.T @ x)
        e_dw.append((F.sums(r) + 75 * U) * (g.abs().T @ x.abs()))
        at += r
    da, e_da, dw, e_dw = torch.cat(da), torch.cat(e_da), torch.stack(dw), torch.stack(e_dw)
    return (da, e_da + F.rounded(da.abs() + e_da, dtype)), (dw, e_dw + F.rounded(dw.abs() + e_dw, out))
