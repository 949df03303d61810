"""The operators of a feed-forward layer, as cases that are timed and compared with their plain forms.

Four operators, which a model with gated feed-forward layers needs together:

* ``quantize``  clpk_quantize_rows_i8: one scale for each row (token or output channel) and 8-bit integers;
* ``linear``    clpk_gemm_i8_scaled: product of 8-bit integers, scaled for each token and channel, with a bias;
* ``ffn``       clpk_gated_ffn: h = act(x Wg^T) * (x Wu^T) in 16-bit floats, or in 8-bit integers with scales;
* ``backward``  clpk_gated_ffn_backward: gradients of x, Wg and Wu from that of h and from what the forward pass kept.

A case is a dict: ``path``; ``rows`` / ``cols`` / ``dtype`` (quantize), ``m`` / ``n`` / ``k`` / ``out`` / ``bias`` (linear), or
``m`` tokens / ``d`` model width / ``f`` hidden width / ``dtype`` / ``act`` (ffn, backward); ``pad``: rows lie further apart than
their length.  Rows whose length is no multiple of 16 bytes lie at the next one in any case.
"""
import ctypes as C
import math

import torch

own = False

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "i8": torch.int8}
ACTS = ("silu", "gelu_tanh", "gelu", "relu", "sigmoid")


def quantize(name, dtype, rows, cols, pad=False):
    return {"name": name, "path": "quantize", "dtype": dtype, "rows": rows, "cols": cols, "pad": pad}


def linear(name, m, n, k, out="bf16", bias=False, pad=False):
    return {"name": name, "path": "linear", "m": m, "n": n, "k": k, "out": out, "bias": bias, "pad": pad}


def ffn(name, dtype, m, d, f, act="silu", out="bf16", path="ffn", pad=False):
    return {"name": name, "path": path, "dtype": dtype, "m": m, "d": d, "f": f, "act": act, "out": out, "pad": pad}


def listed():
    return [
        # the smallest call: one token's activations in front of an 8-bit product
        quantize("quantize_bf16_1x4096", "bf16", 1, 4096),
        # the weights of one layer in single precision, odd row length
        quantize("quantize_f32_4097x11007", "f32", 4097, 11007),
        # one token through one projection: all the time is reading the weights
        linear("linear_i8_1x4096x4096", 1, 4096, 4096),
        # a ragged batch of sequences in the decode phase, results in single precision
        linear("linear_i8_37x1016x5000_f32", 37, 1016, 5000, "f32", True),
        # a long prompt through the largest product of the GEMM configuration's sizes that a layer has
        linear("linear_i8_8192x8192x8192", 8192, 8192, 8192, "bf16", True),
        # one token through the gated half of a layer
        ffn("ffn_bf16_1x4096x11008", "bf16", 1, 4096, 11008),
        # the same in 8 bits for a batch of decoding sequences
        ffn("ffn_i8_48x4096x11008", "i8", 48, 4096, 11008),
        # a small ragged prompt, the other 16-bit type, rows that are slices of longer ones
        ffn("ffn_f16_333x1000x2712_pad", "f16", 333, 1000, 2712, "gelu_tanh", "f16", pad=True),
        # a training batch
        ffn("ffn_bf16_8192x4096x8192", "bf16", 8192, 4096, 8192),
        # a long prompt in 8 bits
        ffn("ffn_i8_4096x4096x11008", "i8", 4096, 4096, 11008, "gelu"),
        # backward pass of a small ragged batch
        ffn("backward_f16_1000x520x1400", "f16", 1000, 520, 1400, "gelu_tanh", "f16", "backward"),
        # backward pass of a training batch
        ffn("backward_bf16_8192x2048x8192", "bf16", 8192, 2048, 8192, "silu", "bf16", "backward"),
    ]


def spread(rng, lo, hi, unit=1):
    """A multiple of `unit` in [lo, hi], even over its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    v = min(hi // unit, max(-(-lo // unit), round(v / unit))) * unit
    return v if v != 3 * 1024 else v + unit


def draw(rng):
    path = rng.choices(("quantize", "linear", "ffn", "backward"), (1, 2, 3, 2))[0]
    pad, unit = rng.random() < 0.25, rng.choice((1, 8, 64))
    while True:
        if path == "quantize":
            case = quantize("", rng.choice(("bf16", "f16", "f32")), spread(rng, 1, 16384), spread(rng, 64, 16384, unit), pad)
            cost, most = case["rows"] * case["cols"], 4097 * 11007
        elif path == "linear":
            case = linear("", spread(rng, 1, 8192), spread(rng, 64, 16384, unit), spread(rng, 64, 16384, unit),
                          rng.choice(("bf16", "f16", "f32")), rng.random() < 0.5, pad)
            cost, most = case["m"] * case["n"] * case["k"], 8192 ** 3
        else:
            dtype = rng.choice(("bf16", "f16", "i8") if path == "ffn" else ("bf16", "f16"))
            case = ffn("", dtype, spread(rng, 1 if path == "ffn" else 64, 8192), spread(rng, 64, 8192, unit), spread(rng, 64, 14336, unit),
                       rng.choice(ACTS), rng.choice(("bf16", "f16", "f32")) if dtype == "i8" else dtype, path, pad)
            cost, most = case["m"] * case["d"] * case["f"], 8192 * 4096 * 8192 if path == "ffn" else 8192 * 2048 * 8192
        if cost <= most:
            del case["name"]
            return case


# ---- inputs -------------------------------------------------------------------------------------------------

def pitch(cols, elem, pad):
    """Elements from one row to the next: a multiple of 16 bytes, and more of them for a slice of longer rows."""
    unit = 16 // elem
    return -(-cols // unit) * unit + (4 * unit if pad else 0)


def matrix(rows, cols, dtype, pad):
    t = TORCH[dtype]
    step = pitch(cols, t.itemsize, pad)
    return torch.empty(rows, step, dtype=t, device="cuda")[:, :cols]


def normal(gen, rows, cols, dtype, pad, std=1.0):
    out = matrix(rows, cols, dtype, pad)
    out.copy_(torch.randn(rows, cols, generator=gen, device="cuda").mul_(std))
    return out


def whole(gen, rows, cols, pad):
    """8-bit integers as the quantiser leaves them for normal values (the largest of some thousand is four deviations), and
    their rows' scales."""
    out = matrix(rows, cols, "i8", pad)
    out.copy_(torch.randn(rows, cols, generator=gen, device="cuda").mul_(32).round_().clamp_(-127, 127))
    return out, torch.rand(rows, generator=gen, device="cuda").mul_(0.5).add_(0.75).mul_(1 / (32 * math.sqrt(cols)))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    path, pad = case["path"], case["pad"]
    s = dict(case, status=torch.zeros(1, dtype=torch.int32, device="cuda"))
    if path == "quantize":
        rows, cols = case["rows"], case["cols"]
        x = normal(gen, rows, cols, case["dtype"], pad)
        x[:, :: 61] *= 20                                       # channels that stand out, as activations have them
        if rows > 8:
            x[rows // 3] = 0                                    # a padding token
        s.update(x=x, q=matrix(rows, cols, "i8", pad), scale=torch.empty(rows, device="cuda"))
        return s
    if path == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["a_scale"] = whole(gen, m, k, pad)
        s["b"], s["b_scale"] = whole(gen, n, k, pad)
        s["a_scale"] *= math.sqrt(k)                            # so that results are of the order of one
        s["bias"] = normal(gen, 1, n, case["out"], False)[0] if case["bias"] else None
        s["c"] = matrix(m, n, case["out"], pad)
        return s
    m, d, f, dtype = case["m"], case["d"], case["f"], case["dtype"]
    if dtype == "i8":
        s["x"], s["x_scale"] = whole(gen, m, d, pad)
        s["x_scale"] *= math.sqrt(d)
        s["wg"], s["wg_scale"] = whole(gen, f, d, pad)
        s["wu"], s["wu_scale"] = whole(gen, f, d, pad)
    else:
        s["x"] = normal(gen, m, d, dtype, pad)
        s["wg"], s["wu"] = (normal(gen, f, d, dtype, pad, 1 / math.sqrt(d)) for _ in range(2))
    if path == "ffn":
        s["h"] = matrix(m, f, case["out"], pad)
        return s
    s["dh"] = normal(gen, m, f, dtype, pad, 0.1)
    for name, w in (("g", "wg"), ("u", "wu")):                  # what the forward pass kept
        s[name] = matrix(m, f, dtype, pad)
        s[name].copy_(s["x"].float() @ s[w].float().T)
    s["dx"] = matrix(m, d, dtype, pad)
    s["dwg"], s["dwu"] = (matrix(f, d, dtype, pad) for _ in range(2))
    return s


# ---- the framework's calls ------------------------------------------------------------------------------------

def bind(s):
    """What a program sets up once and keeps with its buffers: the function, its arguments, the workspace and the stream.  Every
    pass then makes the call itself."""
    from clpeak_b200 import native as N
    K, stream = N.kernels(), torch.cuda.current_stream().cuda_stream
    DT = {"bf16": N.DT_BF16, "f16": N.DT_F16, "f32": N.DT_F32, "i8": N.DT_I8}
    path, ptr, step = s["path"], lambda name: s[name].data_ptr(), lambda name: s[name].stride(0)
    if path == "quantize":
        return K.clpk_quantize_rows_i8, (ptr("q"), ptr("scale"), ptr("x"), s["rows"], s["cols"], step("q"), step("x"), DT[s["dtype"]], stream)
    if path == "linear":
        args = N.GemmI8ScaledArgs(m=s["m"], n=s["n"], k=s["k"], out_dtype=DT[s["out"]], d_a=ptr("a"), d_b=ptr("b"), d_c=ptr("c"),
                                  lda=step("a"), ldb=step("b"), ldc=step("c"), d_a_scale=ptr("a_scale"), d_b_scale=ptr("b_scale"),
                                  d_bias=ptr("bias") if s["bias"] is not None else None, d_status=ptr("status"))
        return K.clpk_gemm_i8_scaled, (C.byref(args), stream)
    act = ACTS.index(s["act"])
    if path == "ffn":
        args = N.GatedFfnArgs(dtype=DT[s["dtype"]], out_dtype=DT[s["out"]], activation=act, m=s["m"], d=s["d"], f=s["f"],
                              d_x=ptr("x"), d_wg=ptr("wg"), d_wu=ptr("wu"), d_h=ptr("h"), ldx=step("x"), ldw=step("wg"), ldh=step("h"),
                              d_status=ptr("status"))
        if s["dtype"] == "i8":
            args.d_x_scale, args.d_wg_scale, args.d_wu_scale = ptr("x_scale"), ptr("wg_scale"), ptr("wu_scale")
        return K.clpk_gated_ffn, (C.byref(args), stream)
    need = C.c_size_t(0)
    K.clpk_gated_ffn_backward_workspace_bytes(DT[s["dtype"]], s["m"], s["d"], s["f"], C.byref(need))
    s["workspace"] = torch.empty(max(need.value, 16), dtype=torch.uint8, device="cuda")
    args = N.GatedFfnBackwardArgs(dtype=DT[s["dtype"]], activation=act, m=s["m"], d=s["d"], f=s["f"], d_x=ptr("x"), d_wg=ptr("wg"),
                                  d_wu=ptr("wu"), d_dh=ptr("dh"), d_g=ptr("g"), d_u=ptr("u"), d_dx=ptr("dx"), d_dwg=ptr("dwg"),
                                  d_dwu=ptr("dwu"), ldx=step("x"), ldw=step("wg"), ldh=step("dh"), d_workspace=ptr("workspace"),
                                  workspace_bytes=need.value, d_status=ptr("status"))
    return K.clpk_gated_ffn_backward, (C.byref(args), stream)


OUTPUTS = {"quantize": ("q", "scale"), "linear": ("c",), "ffn": ("h",), "backward": ("dx", "dwg", "dwu")}


def run_own(s):
    if "call" not in s:
        s["call"] = bind(s)
    function, args = s["call"]
    function(*args)
    return [s[name] for name in OUTPUTS[s["path"]]]


# ---- plain forms ------------------------------------------------------------------------------------------------

def activation(act, g):
    """The activation and its derivative."""
    if act == "silu":
        p = 1 / (1 + torch.exp(-g))
        return g * p, p * (1 + g * (1 - p))
    if act == "sigmoid":
        p = 1 / (1 + torch.exp(-g))
        return p, p * (1 - p)
    if act == "relu":
        return torch.where(g > 0, g, torch.zeros_like(g)), (g > 0).to(g.dtype)
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def run_plain(s):
    path = s["path"]
    if path == "quantize":
        x = s["x"].float()
        top = x.abs().amax(1)
        scale = top / torch.full((), 127.0, device=x.device)
        scale = torch.where(scale >= 2.0 ** -126, scale, torch.zeros_like(scale))           # below: taken as zeros
        inverse = torch.where(scale > 0, torch.reciprocal(scale), torch.zeros_like(scale))
        return [torch.round(x * inverse[:, None]).to(torch.int8), scale]
    if path == "linear":
        c = (s["a"].float() @ s["b"].float().T) * s["a_scale"][:, None] * s["b_scale"]
        if s["bias"] is not None:
            c = c + s["bias"].float()
        return [c.to(TORCH[s["out"]])]
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    if path == "ffn":
        g, u = x @ wg.T, x @ wu.T
        if s["dtype"] == "i8":
            g, u = g * s["x_scale"][:, None] * s["wg_scale"], u * s["x_scale"][:, None] * s["wu_scale"]
        return [(activation(s["act"], g)[0] * u).to(TORCH[s["out"]])]
    dh, g, u = s["dh"].float(), s["g"].float(), s["u"].float()
    a, da = activation(s["act"], g)
    dg, du = dh * u * da, dh * a
    out = dg @ wg + du @ wu, dg.T @ x, du.T @ x
    return [t.to(TORCH[s["dtype"]]) for t in out]


def run(state):
    return run_own(state) if own else run_plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def work(case):
    path = case["path"]
    size = {"bf16": 2, "f16": 2, "f32": 4, "i8": 1}
    if path == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (size[case["dtype"]] + 1) + 4 * case["rows"], "flops": 2 * n}
    if path == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * (k + 4) + m * n * size[case["out"]] + (n * size[case["out"]] if case["bias"] else 0), "flops": 2 * m * n * k}
    m, d, f, e = case["m"], case["d"], case["f"], size[case["dtype"]]
    if path == "ffn":
        scales = 4 * (m + 2 * f) if case["dtype"] == "i8" else 0
        return {"bytes": (m + 2 * f) * d * e + m * f * size[case["out"]] + scales, "flops": 4 * m * d * f}
    return {"bytes": (2 * m * d + 4 * f * d + 3 * m * f) * e, "flops": 8 * m * d * f}


# ---- from the definitions, in 64 bits -----------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    w = {n: t.to(torch.float64) for n, t in s.items() if isinstance(t, torch.Tensor) and n not in ("q", "scale", "c", "h", "dx", "dwg", "dwu", "workspace")}
    if case["path"] == "quantize":
        return [None, w["x"].abs().max(dim=1).values / 127]
    if case["path"] == "linear":
        c = torch.matmul(w["a"] * w["a_scale"].unsqueeze(1), (w["b"] * w["b_scale"].unsqueeze(1)).t())
        return [c + w["bias"] if case["bias"] else c]
    act = case["act"]

    def phi(z):                                                 # the activation alone, as its textbook form has it
        if act == "relu":
            return z.clamp(min=0)
        if act == "gelu":
            return z * torch.special.ndtr(z)
        if act == "gelu_tanh":                                  # (1 + tanh y) / 2 = sigmoid(2 y)
            return z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))
        return z * torch.sigmoid(z) if act == "silu" else torch.sigmoid(z)

    if case["path"] == "ffn":
        if case["dtype"] == "i8":
            for n in ("x", "wg", "wu"):
                w[n] = w[n] * w[n + "_scale"].unsqueeze(1)
        gate = phi(torch.matmul(w["x"], w["wg"].t()))
        return [gate * torch.matmul(w["x"], w["wu"].t())]
    g = w["g"].requires_grad_()
    u = w["u"].requires_grad_()
    dg, du = torch.autograd.grad(phi(g) * u, (g, u), w["dh"])   # through the two products by hand, from their definition
    return [torch.matmul(dg, w["wg"]) + torch.matmul(du, w["wu"]), torch.matmul(dg.t(), w["x"]), torch.matmul(du.t(), w["x"])]
