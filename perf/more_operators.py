"""The operators that train a block of a model, as cases that are timed and compared with their plain forms.

Five paths, next to those of the feed-forward layer:

* ``norm``              clpk_layer_norm: y = (x - mean) * rstd * weight + bias, with the statistics that the backward pass takes;
* ``norm_backward``     clpk_layer_norm_backward: gradients of x, weight and bias;
* ``adamw``             clpk_adamw: one step over many tensors, moments in fp32 or in 8 bits;
* ``grouped``           clpk_grouped_gemm: rows sorted by expert, each multiplied by its expert's weights;
* ``grouped_backward``  clpk_grouped_gemm_backward: gradients of the rows and of every expert's weights.

A case is a dict: ``path``; ``m`` rows / ``d`` / ``dtype`` / ``wdtype`` / ``pad`` (norm, norm_backward); ``dtype`` / ``grad`` / ``state`` / ``master`` and
``layers`` / ``d`` / ``f`` or ``tensors`` / ``largest`` (adamw); ``m`` rows / ``n`` / ``k`` / ``groups`` / ``skew`` / ``spare`` / ``dtype`` / ``out`` / ``pad`` (grouped,
grouped_backward).  ``pad``: rows lie further apart than their length; rows whose length is no multiple of 16 bytes lie at the
next one in any case.
"""
import ctypes as C
import math
import random

import torch

own = False

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "i8": torch.int8}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "i8": 1}
EPS = 1e-5                                                      # of the norm
LR, BETA1, BETA2, ADAM_EPS, DECAY, STEP = 1e-3, 0.9, 0.95, 1e-8, 0.1, 100
BLOCK = 256                                                     # elements that share a scale, 8-bit moments


def norm(name, dtype, m, d, wdtype=None, path="norm", pad=False):
    return {"name": name, "path": path, "dtype": dtype, "wdtype": wdtype or dtype, "m": m, "d": d, "pad": pad}


def adamw(name, dtype, grad, state, master, layers=0, d=0, f=0, tensors=0, largest=0):
    return {"name": name, "path": "adamw", "dtype": dtype, "grad": grad, "state": state, "master": master, "layers": layers, "d": d, "f": f,
            "tensors": tensors, "largest": largest}


def grouped(name, dtype, m, n, k, groups, skew=1.0, spare=0, out=None, path="grouped", pad=False):
    return {"name": name, "path": path, "dtype": dtype, "out": out or dtype, "m": m, "n": n, "k": k, "groups": groups, "skew": skew, "spare": spare, "pad": pad}


def listed():
    return [
        # the smallest call: one token in front of a layer, while text is generated
        norm("norm_bf16_1x4096", "bf16", 1, 4096),
        # a batch of long prompts, weights in single precision
        norm("norm_bf16_16384x8192", "bf16", 16384, 8192, "f32"),
        # backward pass of a small ragged batch, rows that are slices of longer ones
        norm("norm_backward_f16_1001x1000_pad", "f16", 1001, 1000, "f32", "norm_backward", True),
        # backward pass of a training batch
        norm("norm_backward_bf16_8192x4096", "bf16", 8192, 4096, "bf16", "norm_backward"),
        # a step of what is trained besides matrices: the norms' weights and biases of 32 layers
        adamw("adamw_f32_64x4096", "f32", "f32", "f32", False, 32, 4096, 0),
        # a step of two feed-forward layers in mixed precision: 16-bit parameters with their master copies
        adamw("adamw_bf16_2x4096x11008", "bf16", "bf16", "f32", True, 2, 4096, 11008),
        # the same with moments in 8 bits and gradients that were summed in single precision, no master copies
        adamw("adamw_bf16_i8_2x4096x11008", "bf16", "f32", "i8", False, 2, 4096, 11008),
        # fine-tuning: tensors of any size, down to single elements
        adamw("adamw_f16_i8_61_ragged", "f16", "f16", "i8", True, tensors=61, largest=2500000),
        # eight decoding sequences with four experts each: most experts have no row or one
        grouped("grouped_bf16_32x1408x2048_of_64", "bf16", 32, 1408, 2048, 64),
        # a training batch sorted by expert, some experts asked for more than others
        grouped("grouped_bf16_16384x8192x4096_of_8", "bf16", 16384, 8192, 4096, 8),
        # backward pass of a small ragged batch with rows that no expert has
        grouped("grouped_backward_f16_1403x1000x520_of_17", "f16", 1403, 1000, 520, 17, 2.0, 38, path="grouped_backward", pad=True),
        # backward pass of a training batch, the weights' gradients in single precision
        grouped("grouped_backward_bf16_8192x4096x2048_of_16", "bf16", 8192, 4096, 2048, 16, out="f32", path="grouped_backward"),
    ]


def spread(rng, lo, hi, unit=1):
    """A multiple of `unit` in [lo, hi], even over its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // unit, max(-(-lo // unit), round(v / unit))) * unit


def draw(rng):
    path = rng.choices(("norm", "norm_backward", "adamw", "grouped", "grouped_backward"), (2, 2, 3, 3, 2))[0]
    pad, unit = rng.random() < 0.25, rng.choice((1, 8, 64))
    while True:
        if path in ("norm", "norm_backward"):
            dtype = rng.choice(("bf16", "f16", "f32"))
            case = norm("", dtype, spread(rng, 1, 16384), spread(rng, 64, 16384, unit), rng.choice((dtype, "f32")), path, pad)
            cost, most = case["m"] * case["d"] * SIZE[dtype], 16384 * 8192 * 2 if path == "norm" else 8192 * 4096 * 2
        elif path == "adamw":
            dtype = rng.choice(("bf16", "f16", "f32"))
            kind = (dtype, rng.choice((dtype, "f32")), rng.choice(("f32", "i8")), dtype != "f32" and rng.random() < 0.5)
            if rng.random() < 0.5:
                case = adamw("", *kind, rng.randint(1, 4), spread(rng, 256, 4096, unit), spread(rng, 512, 11008, unit))
            else:
                case = adamw("", *kind, tensors=rng.randint(1, 200), largest=spread(rng, 16, 10000000))
            cost, most = sum(sizes(case)), 2 * 3 * 4096 * 11008
        else:
            dtype = rng.choice(("bf16", "f16"))
            case = grouped("", dtype, spread(rng, 1 if path == "grouped" else 64, 16384), spread(rng, 64, 8192, unit), spread(rng, 64, 4096, unit),
                           spread(rng, 1, 64), rng.choice((0.0, 1.0, 2.0)), rng.choice((0, 0, 5)), rng.choice((dtype, "f32")), path, pad)
            cost, most = case["m"] * case["n"] * case["k"], 16384 * 8192 * 4096 if path == "grouped" else 8192 * 4096 * 2048
            cost = max(cost, case["groups"] * case["n"] * case["k"] * 200)
        if cost <= most:
            del case["name"]
            return case


def sizes(case):
    """Elements of the tensors of a step."""
    if case["layers"]:
        d, f = case["d"], case["f"]
        return ([d, d] + [d * f] * (3 if f else 0)) * case["layers"]
    rng = random.Random("%d tensors up to %d" % (case["tensors"], case["largest"]))
    return [spread(rng, 1, case["largest"]) for _ in range(case["tensors"])]


def rows_of(case):
    """Rows of the groups: the busier the lower a group's place in an order of their own, `skew` to `skew` + 1 times; `spare` rows have no group."""
    rng = random.Random("%(m)d rows, %(n)d x %(k)d, %(groups)d groups" % case)
    share = [(1 + case["skew"] * rng.random() ** 2) * (rng.random() < 0.9) for _ in range(case["groups"])]
    total, rows = max(1, case["m"] - case["spare"]), [0] * case["groups"]
    if not any(share):
        share[0] = 1
    if total < 16 * case["groups"]:                             # few: each row asks for itself
        for _ in range(total):
            rows[rng.choices(range(case["groups"]), share)[0]] += 1
    else:
        for e in range(case["groups"]):
            rows[e] = int(total * share[e] / sum(share))
        rows[share.index(max(share))] += total - sum(rows)
    return rows


# ---- inputs -------------------------------------------------------------------------------------------------

def pitch(cols, elem, pad):
    """Elements from one row to the next: a multiple of 16 bytes, and more of them for a slice of longer rows."""
    unit = 16 // elem
    return -(-cols // unit) * unit + (4 * unit if pad else 0)


def matrix(rows, cols, dtype, pad):
    t = TORCH[dtype]
    return torch.zeros(rows, pitch(cols, t.itemsize, pad), dtype=t, device="cuda")[:, :cols]


def normal(gen, rows, cols, dtype, pad, std=1.0):
    out = matrix(rows, cols, dtype, pad)
    out.copy_(torch.randn(rows, cols, generator=gen, device="cuda").mul_(std))
    return out


def moments(gen, n, blocks, state):
    """Moments as some steps leave them, zeros between the tensors: (m, v) or in 8 bits (codes of m, of v, scales of m, of v)."""
    m, v = (torch.randn(n, generator=gen, device="cuda").mul_(1e-3) for _ in range(2))
    v.square_().add_(1e-8)
    if state == "f32":
        return {"m": m.mul_(blocks), "v": v.mul_(blocks)}
    del m, v
    codes = {"m": torch.randint(-127, 128, (n,), generator=gen, device="cuda", dtype=torch.int8), "v": torch.randint(1, 256, (n,), generator=gen, device="cuda", dtype=torch.uint8)}
    codes["m"].mul_(blocks)
    codes["v"].mul_(blocks)
    scale = lambda top: torch.rand(n // BLOCK, generator=gen, device="cuda").add_(0.5).mul_(2e-3 / top)  # noqa: E731
    return dict(codes, m_scale=scale(127 ** 2), v_scale=scale(255 ** 2))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    path = case["path"]
    s = dict(case)
    if path in ("norm", "norm_backward"):
        m, d, dtype, pad = case["m"], case["d"], case["dtype"], case["pad"]
        x = torch.randn(m, d, generator=gen, device="cuda")
        x[:, ::61] *= 20                                        # channels that stand out, as activations have them
        x += torch.randn(m, 1, generator=gen, device="cuda")
        s["x"] = matrix(m, d, dtype, pad)
        s["x"].copy_(x)
        s["weight"] = torch.randn(d, generator=gen, device="cuda").mul_(0.2).add_(1).to(TORCH[case["wdtype"]])
        s["bias"] = torch.randn(d, generator=gen, device="cuda").mul_(0.2).to(TORCH[case["wdtype"]])
        s["mean"], s["rstd"] = (torch.empty(m, device="cuda") for _ in range(2))
        if path == "norm":
            s["y"] = matrix(m, d, dtype, pad)
            return s
        wide = s["x"].double()                                  # what the forward pass kept
        s["mean"].copy_(wide.mean(1))
        s["rstd"].copy_(1 / torch.sqrt(wide.var(1, correction=0) + EPS))
        s["dy"] = normal(gen, m, d, dtype, pad, 0.1)
        s["dx"] = matrix(m, d, dtype, pad)
        s["dweight"], s["dbias"] = (torch.empty(d, dtype=TORCH[case["wdtype"]], device="cuda") for _ in range(2))
        return s
    if path == "adamw":
        # parameters, gradients and moments are slices of one buffer each, every tensor from a multiple of 256 elements on
        s["sizes"], s["starts"], n = sizes(case), [], 0
        for size in s["sizes"]:
            s["starts"].append(n)
            n += -(-size // BLOCK) * BLOCK
        inside = torch.zeros(n + 1, dtype=torch.int8, device="cuda")
        inside[torch.tensor(s["starts"], device="cuda")] += 1
        ends = torch.tensor([a + size for a, size in zip(s["starts"], s["sizes"])], device="cuda")
        inside.scatter_add_(0, ends, torch.full_like(ends, -1, dtype=torch.int8))
        inside = inside[:n].cumsum(0, dtype=torch.int8)
        s.update(moments(gen, n, inside, case["state"]))
        value = torch.randn(n, generator=gen, device="cuda").mul_(0.02).mul_(inside)
        s["param"] = value.to(TORCH[case["dtype"]])
        s["master"] = value if case["master"] else None
        s["grad"] = torch.randn(n, generator=gen, device="cuda").mul_(1e-3).mul_(inside).to(TORCH[case["grad"]])
        return s
    m, n, k, groups, dtype, pad = (case[x] for x in ("m", "n", "k", "groups", "dtype", "pad"))
    s["rows"] = rows_of(case)
    s["most"] = max(1, max(s["rows"]))
    s["offsets"] = torch.tensor([0] + s["rows"], device="cuda").cumsum(0).to(torch.int32)
    s["a"] = normal(gen, m, k, dtype, pad)
    s["w"] = normal(gen, groups * n, k, dtype, pad, 1 / math.sqrt(k))
    if path == "grouped":
        s["c"] = matrix(m, n, case["out"], pad)
        return s
    s["dc"] = normal(gen, m, n, dtype, pad, 0.1)
    s["da"] = matrix(m, k, dtype, pad)
    s["dw"] = matrix(groups * n, k, case["out"], pad)
    return s


# ---- the framework's calls ------------------------------------------------------------------------------------

def bind(s):
    """What a program sets up once and keeps with its buffers: the function, its arguments, the workspace and the stream.  Every
    pass then makes the call itself."""
    from clpeak_b200 import native as N
    K, stream = N.kernels(), torch.cuda.current_stream().cuda_stream
    DT = {"bf16": N.DT_BF16, "f16": N.DT_F16, "f32": N.DT_F32, "i8": N.DT_I8}
    path, ptr, step = s["path"], lambda name: s[name].data_ptr(), lambda name: s[name].stride(0)
    need = C.c_size_t(0)
    if path == "norm":
        args = N.LayerNormArgs(dtype=DT[s["dtype"]], weight_dtype=DT[s["wdtype"]], m=s["m"], d=s["d"], d_x=ptr("x"), d_weight=ptr("weight"),
                               d_bias=ptr("bias"), d_y=ptr("y"), d_mean=ptr("mean"), d_rstd=ptr("rstd"), ldx=step("x"), ldy=step("y"), eps=EPS)
        return K.clpk_layer_norm, (C.byref(args), stream)
    if path == "norm_backward":
        K.clpk_layer_norm_backward_workspace_bytes(s["m"], s["d"], C.byref(need))
        s["workspace"] = torch.empty(max(need.value, 16), dtype=torch.uint8, device="cuda")
        args = N.LayerNormBackwardArgs(dtype=DT[s["dtype"]], weight_dtype=DT[s["wdtype"]], m=s["m"], d=s["d"], d_x=ptr("x"), d_weight=ptr("weight"),
                                       d_dy=ptr("dy"), d_mean=ptr("mean"), d_rstd=ptr("rstd"), d_dx=ptr("dx"), d_dweight=ptr("dweight"),
                                       d_dbias=ptr("dbias"), ldx=step("x"), lddy=step("dy"), lddx=step("dx"), d_workspace=ptr("workspace"),
                                       workspace_bytes=need.value)
        return K.clpk_layer_norm_backward, (C.byref(args), stream)
    if path == "adamw":
        at = lambda name, i, unit=1: s[name][i // unit:].data_ptr()  # noqa: E731
        small = s["state"] == "i8"
        table = (N.AdamwTensor * len(s["sizes"]))(*[
            N.AdamwTensor(n=n, d_param=at("param", i), d_grad=at("grad", i), d_master=at("master", i) if s["master"] is not None else None, d_m=at("m", i),
                          d_v=at("v", i), d_m_scale=at("m_scale", i, BLOCK) if small else None, d_v_scale=at("v_scale", i, BLOCK) if small else None)
            for i, n in zip(s["starts"], s["sizes"])])
        args = N.AdamwArgs(dtype=DT[s["dtype"]], grad_dtype=DT[s["grad"].dtype is torch.float32 and "f32" or s["dtype"]], state_dtype=DT[s["state"]],
                           count=len(table), h_tensors=C.addressof(table), lr=LR, beta1=BETA1, beta2=BETA2, eps=ADAM_EPS, weight_decay=DECAY, step=STEP)
        s["table"] = table
        return K.clpk_adamw, (C.byref(args), stream)
    s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.clpk_grouped_gemm_workspace_bytes(s["groups"], C.byref(need))
    s["workspace"] = torch.empty(max(need.value, 16), dtype=torch.uint8, device="cuda")
    common = dict(dtype=DT[s["dtype"]], m=s["m"], n=s["n"], k=s["k"], groups=s["groups"], d_a=ptr("a"), d_w=ptr("w"), d_offsets=ptr("offsets"),
                  lda=step("a"), ldw=step("w"), stride_w=s["n"] * step("w"), d_workspace=ptr("workspace"), workspace_bytes=need.value, d_status=ptr("status"))
    if path == "grouped":
        args = N.GroupedGemmArgs(out_dtype=DT[s["out"]], d_c=ptr("c"), ldc=step("c"), **common)
        return K.clpk_grouped_gemm, (C.byref(args), stream)
    args = N.GroupedGemmBackwardArgs(dw_dtype=DT[s["out"]], d_dc=ptr("dc"), d_da=ptr("da"), d_dw=ptr("dw"), lddc=step("dc"), ldda=step("da"),
                                     lddw=step("dw"), stride_dw=s["n"] * step("dw"), **common)
    return K.clpk_grouped_gemm_backward, (C.byref(args), stream)


def outputs(s):
    if s["path"] == "adamw":
        return [s[name] for name in ("param", "master", "m", "v", "m_scale", "v_scale") if s.get(name) is not None]
    return [s[name] for name in {"norm": ("y", "mean", "rstd"), "norm_backward": ("dx", "dweight", "dbias"), "grouped": ("c",),
                                 "grouped_backward": ("da", "dw")}[s["path"]]]


def run_own(s):
    if "call" not in s:
        s["call"] = bind(s)
    function, args = s["call"]
    function(*args)
    return outputs(s)


# ---- plain forms ------------------------------------------------------------------------------------------------

def plain_norm(s):
    x = s["x"].float()
    mean = x.sum(1) / s["d"]
    off = x - mean[:, None]
    rstd = 1 / torch.sqrt((off * off).sum(1) / s["d"] + EPS)
    y = off * rstd[:, None] * s["weight"].float() + s["bias"].float()
    return [y.to(s["x"].dtype), mean, rstd]


def plain_norm_backward(s):
    dy, t = s["dy"].float(), TORCH[s["wdtype"]]
    xhat = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * s["weight"].float()
    dx = (g - (g.sum(1) / s["d"])[:, None] - xhat * ((g * xhat).sum(1) / s["d"])[:, None]) * s["rstd"][:, None]
    return [dx.to(s["x"].dtype), (dy * xhat).sum(0).to(t), dy.sum(0).to(t)]


def to_codes(size, steps):
    """`size` >= 0, a block of elements a row: scales, and codes whose squares times them it is."""
    scale = size.amax(1) / torch.full((), float(steps * steps), device=size.device)
    whole = torch.isfinite(scale)
    scale = torch.where(whole, torch.where(scale >= 2.0 ** -126, scale, torch.zeros_like(scale)), torch.full_like(scale, math.nan))
    inverse = torch.where(scale > 0, torch.reciprocal(scale), torch.zeros_like(scale))
    codes = torch.round(torch.sqrt(size * inverse[:, None]))
    return scale, torch.where(whole[:, None], codes, torch.zeros_like(codes))


def plain_adamw(s):
    small = s["state"] == "i8"
    p = s["master"] if s["master"] is not None else s["param"].float()
    g, m, v = s["grad"].float(), s["m"].float(), s["v"].float()
    if small:
        m = (m * m.abs()).view(-1, BLOCK) * s["m_scale"][:, None]
        root = (v * v).view(-1, BLOCK) * s["v_scale"][:, None]
        m, v = m.view(-1), (root * root).view(-1)
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    root = torch.sqrt(v)
    # corrections of the two moments' start, and the decay, are numbers of the step
    p = p * (1 - LR * DECAY) - (m / (root * (1 / math.sqrt(1 - BETA2 ** STEP)) + ADAM_EPS)) * (LR / (1 - BETA1 ** STEP))
    s["param"] = p.to(s["param"].dtype)
    if s["master"] is not None:
        s["master"] = p
    if not small:
        s["m"], s["v"] = m, v
        return outputs(s)
    s["m_scale"], codes = to_codes(m.abs().view(-1, BLOCK), 127)
    s["m"] = (codes.view(-1) * torch.sign(m)).to(torch.int8)
    s["v_scale"], codes = to_codes(root.view(-1, BLOCK), 255)
    some = (root.view(-1, BLOCK) > 0) & (s["v_scale"] > 0)[:, None]
    s["v"] = torch.where(some, codes.clamp(min=1), codes).to(torch.uint8).view(-1)
    return outputs(s)


def by_group(s, rows):
    """The rows of every group behind one another, filled up with zeros: [groups][most][cols], and where each row is."""
    r = torch.arange(rows.shape[0], device=rows.device)
    e = (r[:, None] >= s["offsets"][None, 1:]).sum(1)           # `groups` for rows that have none
    out = torch.zeros(s["groups"] + 1, max(s["most"], s["spare"]), rows.shape[1], device=rows.device)
    at = r - s["offsets"][e]
    out[e, at] = rows.float()
    return out[:-1], (e, at)


def back(s, values, where, dtype):
    """Rows out of groups; zeros for those that have none."""
    values = torch.cat((values, torch.zeros_like(values[:1])))
    e, at = where
    return values[e, at.clamp(max=values.shape[1] - 1)].to(dtype)


def plain_grouped(s):
    a, where = by_group(s, s["a"])
    w = s["w"].float().view(s["groups"], s["n"], s["k"])
    return [back(s, torch.bmm(a, w.transpose(1, 2)), where, TORCH[s["out"]])]


def plain_grouped_backward(s):
    a, where = by_group(s, s["a"])
    dc, _ = by_group(s, s["dc"])
    w = s["w"].float().view(s["groups"], s["n"], s["k"])
    dw = torch.bmm(dc.transpose(1, 2), a)
    return [back(s, torch.bmm(dc, w), where, s["a"].dtype), dw.view(-1, s["k"]).to(TORCH[s["out"]])]


def run(state):
    if own:
        return run_own(state)
    return {"norm": plain_norm, "norm_backward": plain_norm_backward, "adamw": plain_adamw, "grouped": plain_grouped,
            "grouped_backward": plain_grouped_backward}[state["path"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def work(case):
    path = case["path"]
    if path in ("norm", "norm_backward"):
        m, d, e, w = case["m"], case["d"], SIZE[case["dtype"]], SIZE[case["wdtype"]]
        if path == "norm":
            return {"bytes": 2 * m * d * e + 2 * d * w + 8 * m, "flops": 8 * m * d}
        return {"bytes": 3 * m * d * e + 3 * d * w + 8 * m, "flops": 14 * m * d}
    if path == "adamw":
        n, e = sum(sizes(case)), SIZE[case["dtype"]]
        blocks = sum(-(-x // BLOCK) for x in sizes(case))
        param = e + (8 if case["master"] else e) + SIZE[case["grad"]]
        return {"bytes": n * (param + (16 if case["state"] == "f32" else 4)) + (16 * blocks if case["state"] == "i8" else 0), "flops": 16 * n}
    m, n, k, e, o = case["m"] - case["spare"], case["n"], case["k"], SIZE[case["dtype"]], SIZE[case["out"]]
    some = sum(r > 0 for r in rows_of(case))
    if path == "grouped":
        return {"bytes": m * k * e + some * n * k * e + m * n * o, "flops": 2 * m * n * k}
    return {"bytes": m * (2 * k + n) * e + some * n * k * e + case["groups"] * n * k * o, "flops": 4 * m * n * k}


# ---- from the definitions, in 64 bits -----------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    wide = lambda name: s[name].to(torch.float64)  # noqa: E731
    path = case["path"]
    if path in ("norm", "norm_backward"):
        x, w = wide("x"), wide("weight").requires_grad_()
        b = wide("bias").requires_grad_()
        if path == "norm":
            var, mean = torch.var_mean(x, 1, correction=0)
            return [((x - mean.unsqueeze(1)) / (var + EPS).sqrt().unsqueeze(1) * w + b).detach(), mean, (var + EPS).rsqrt()]
        # the gradients of sum(dy y), as they follow from the forward pass's definition
        x.requires_grad_()
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        y = (x - mean) / (var + EPS).sqrt() * w + b
        return list(torch.autograd.grad(y, (x, w, b), wide("dy")))
    if path == "adamw":
        m, v, g = wide("m"), wide("v"), wide("grad")
        p = wide("param") if s["master"] is None else wide("master")
        if case["state"] == "i8":
            m = m * m.abs() * wide("m_scale").repeat_interleave(BLOCK)
            v = (v * v * wide("v_scale").repeat_interleave(BLOCK)) ** 2
        m = BETA1 * m + (1 - BETA1) * g
        v = BETA2 * v + (1 - BETA2) * g ** 2
        p = p - LR * DECAY * p - LR * (m / (1 - BETA1 ** STEP)) / ((v / (1 - BETA2 ** STEP)).sqrt() + ADAM_EPS)
        first = [p] if s["master"] is None else [p, p]
        if case["state"] == "f32":
            return first + [m, v]
        return first + [None, None, m.abs().view(-1, BLOCK).amax(1) / 127 ** 2, v.sqrt().view(-1, BLOCK).amax(1) / 255 ** 2]
    ends = [0]
    for rows in s["rows"]:
        ends.append(ends[-1] + rows)
    a, n = wide("a"), case["n"]
    if path == "grouped":
        c = torch.zeros(case["m"], n, dtype=torch.float64, device="cuda")
        for e in range(case["groups"]):
            c[ends[e]:ends[e + 1]] = a[ends[e]:ends[e + 1]] @ s["w"][e * n:(e + 1) * n].double().t()
        return [c]
    dc, da, dw = wide("dc"), torch.zeros_like(a), torch.zeros(case["groups"] * n, case["k"], dtype=torch.float64, device="cuda")
    for e in range(case["groups"]):
        r = slice(ends[e], ends[e + 1])
        da[r] = dc[r] @ s["w"][e * n:(e + 1) * n].double()
        dw[e * n:(e + 1) * n] = dc[r].t() @ a[r]
    return [da, dw]
