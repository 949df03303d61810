"""What trains a block of a model around its products: a norm in front of it, a layer of experts, and the optimiser's step.

    norm = Norm(d, tokens)                              # fp32 weights, bf16 rows
    y = norm.forward(x)                                 # keeps what the backward pass needs
    dx, dweight, dbias = norm.backward(dy)
    experts = Experts(groups, n, k, rows)               # rows sorted by expert, each multiplied by its expert's weights
    y = experts.forward(x, offsets)
    dx, dw = experts.backward(dy)
    step = AdamW([layer.wg, layer.wu], [layer.dwg, layer.dwu], state="i8", master=True)
    step.step(rate)

Buffers, workspaces and argument structures are set up once and used again by every call; calls run on torch's current stream.  What a
call returns is a view of them: it is good until the object's next call of that kind.  What a forward pass was given is read again
by the backward pass and has to be as it was until then.  An object is for one stream and one host thread at a time.
``train`` fits a norm and a feed-forward layer behind it (clpeak_b200.feed_forward) to another pair of them.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import native as N
from .feed_forward import FeedForward, _bytes, _check_device, _check_status, _stream

BAD_OFFSETS = 0x401                     # status word of a call whose offsets are none
DTYPES = {torch.float32: N.DT_F32, torch.float16: N.DT_F16, torch.bfloat16: N.DT_BF16}


def _check_rows(name: str, x: torch.Tensor, dtype: torch.dtype, most: int, cols: int, device: torch.device) -> torch.Tensor:
    """x with rows that share no elements: a stride of 0 is one row for all to torch, and rows one behind another to the calls."""
    if x.dtype != dtype or x.dim() != 2 or x.shape[1] != cols or x.stride(1) != 1 or x.shape[0] > most:
        raise ValueError(f"{name} must be {dtype} [up to {most}][{cols}] with rows of neighbours")
    _check_device(name, x, device)
    return x.contiguous() if x.shape[0] > 1 and x.stride(0) < cols else x


def _span(x: torch.Tensor) -> tuple[int, int]:
    """The bytes from x's first element to behind its last."""
    last = sum((n - 1) * s for n, s in zip(x.shape, x.stride()))
    return x.data_ptr(), x.data_ptr() + (last + 1) * x.element_size() if x.numel() else x.data_ptr()


def _check_apart(name: str, x: torch.Tensor, other: str, out: torch.Tensor) -> None:
    """What a call reads may not lie where it writes."""
    (a, b), (c, d) = _span(x), _span(out)
    if a < d and c < b:
        raise ValueError(f"{name} lies in the object's own {other}")


def _pitch(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


class Norm:
    """Layer norm of up to `rows` rows of `d` elements; weight and bias in fp32."""

    def __init__(self, d: int, rows: int, dtype: torch.dtype = torch.bfloat16, eps: float = 1e-5):
        if dtype not in DTYPES:
            raise ValueError(f"rows of {dtype}")
        self.d, self.rows, self.dtype, self.eps, self.K = d, rows, dtype, eps, N.kernels()
        self.weight, self.bias = torch.ones(d, device="cuda"), torch.zeros(d, device="cuda")
        self.device = self.weight.device
        self.dweight, self.dbias = torch.zeros_like(self.weight), torch.zeros_like(self.bias)
        self.y, self.dx = (torch.empty(rows, d, dtype=dtype, device="cuda") for _ in range(2))
        self.mean, self.rstd = (torch.empty(rows, device="cuda") for _ in range(2))
        need = C.c_size_t(0)
        self.K.clpk_layer_norm_backward_workspace_bytes(rows, d, C.byref(need))
        self.workspace = _bytes(need.value)
        self.x = None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        x = _check_rows("x", x, self.dtype, self.rows, self.d, self.device)
        for name, out in (("y", self.y), ("dx", self.dx)):
            _check_apart("x", x, name, out)
        m = x.shape[0]
        self.x = None
        args = N.LayerNormArgs(dtype=DTYPES[self.dtype], weight_dtype=N.DT_F32, m=m, d=self.d, d_x=x.data_ptr(), d_weight=self.weight.data_ptr(),
                               d_bias=self.bias.data_ptr(), d_y=self.y.data_ptr(), d_mean=self.mean.data_ptr(), d_rstd=self.rstd.data_ptr(), ldx=_pitch(x),
                               eps=self.eps)
        self.K.clpk_layer_norm(C.byref(args), _stream(self.device))
        self.x = x
        return self.y[:m]

    def backward(self, dy: torch.Tensor):
        """(dx, dweight, dbias) from the gradient of the last forward pass's y."""
        if self.x is None:
            raise RuntimeError("backward() without forward()")
        x, m = self.x, self.x.shape[0]
        dy = _check_rows("dy", dy, self.dtype, self.rows, self.d, self.device)
        if dy.shape[0] != m:
            raise ValueError(f"dy must have {m} rows")
        _check_apart("dy", dy, "dx", self.dx)
        args = N.LayerNormBackwardArgs(dtype=DTYPES[self.dtype], weight_dtype=N.DT_F32, m=m, d=self.d, d_x=x.data_ptr(), d_weight=self.weight.data_ptr(),
                                       d_dy=dy.data_ptr(), d_mean=self.mean.data_ptr(), d_rstd=self.rstd.data_ptr(), d_dx=self.dx.data_ptr(),
                                       d_dweight=self.dweight.data_ptr(), d_dbias=self.dbias.data_ptr(), ldx=_pitch(x), lddy=_pitch(dy),
                                       d_workspace=self.workspace.data_ptr(), workspace_bytes=self.workspace.numel())
        self.K.clpk_layer_norm_backward(C.byref(args), _stream(self.device))
        return self.dx[:m], self.dweight, self.dbias


class Experts:
    """y[r] = x[r] W[e]^T in bf16 for up to `rows` rows that lie sorted by expert; expert e has the rows from offsets[e] to offsets[e + 1]
    (int32 on the GPU).  Rows of no expert are zeros in y and dx.  `n` and `k` are multiples of 8 (rows of 16 bytes)."""

    def __init__(self, groups: int, n: int, k: int, rows: int, seed: int = 0):
        if n % 8 or k % 8:
            raise ValueError(f"n and k must be multiples of 8 (got {n}, {k})")
        self.groups, self.n, self.k, self.rows, self.K = groups, n, k, rows, N.kernels()
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.w = (torch.randn(groups, n, k, generator=gen, device="cuda") * k ** -0.5).to(torch.bfloat16)
        self.device = self.w.device
        self.dw = torch.zeros_like(self.w)
        self.y, self.dx = torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda"), torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
        self.status = torch.zeros(2, dtype=torch.int32, device="cuda")
        need = C.c_size_t(0)
        self.K.clpk_grouped_gemm_workspace_bytes(groups, C.byref(need))
        self.workspace = _bytes(need.value)
        self.x = None

    def _common(self, x: torch.Tensor, i: int) -> dict:
        return dict(dtype=N.DT_BF16, m=x.shape[0], n=self.n, k=self.k, groups=self.groups, d_a=x.data_ptr(), d_w=self.w.data_ptr(),
                    d_offsets=self.offsets.data_ptr(), lda=_pitch(x), d_workspace=self.workspace.data_ptr(), workspace_bytes=self.workspace.numel(),
                    d_status=self.status.data_ptr() + 4 * i)

    def forward(self, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
        x = _check_rows("x", x, torch.bfloat16, self.rows, self.k, self.device)
        for name, out in (("y", self.y), ("dx", self.dx), ("dw", self.dw)):
            _check_apart("x", x, name, out)
        if offsets.dtype != torch.int32 or tuple(offsets.shape) != (self.groups + 1,) or not offsets.is_contiguous():
            raise ValueError(f"offsets must be contiguous int32 [{self.groups + 1}]")
        _check_device("offsets", offsets, self.device)
        self.x, self.offsets = None, offsets
        y = self.y[:x.shape[0]].zero_()                 # the call leaves rows of no expert as they are
        args = N.GroupedGemmArgs(out_dtype=N.DT_BF16, d_c=y.data_ptr(), **self._common(x, 0))
        self.K.clpk_grouped_gemm(C.byref(args), _stream(self.device))
        self.x = x
        return y

    def backward(self, dy: torch.Tensor):
        """(dx, dw) from the gradient of the last forward pass's y."""
        if self.x is None:
            raise RuntimeError("backward() without forward()")
        dy = _check_rows("dy", dy, torch.bfloat16, self.rows, self.n, self.device)
        if dy.shape[0] != self.x.shape[0]:
            raise ValueError(f"dy must have {self.x.shape[0]} rows")
        for name, out in (("dx", self.dx), ("dw", self.dw)):
            _check_apart("dy", dy, name, out)
        dx = self.dx[:self.x.shape[0]].zero_()
        args = N.GroupedGemmBackwardArgs(dw_dtype=N.DT_BF16, d_dc=dy.data_ptr(), lddc=_pitch(dy), d_da=dx.data_ptr(), d_dw=self.dw.data_ptr(), **self._common(self.x, 1))
        self.K.clpk_grouped_gemm_backward(C.byref(args), _stream(self.device))
        return dx, self.dw

    def check(self) -> None:
        """Raises if the last passes' offsets were none, or a device-side wait expired.  Waits for the stream."""
        if BAD_OFFSETS in self.status.tolist():
            raise N.ClpkError(N.ERR_BAD_ARG, "offsets decrease or leave the rows", "experts")
        _check_status(self.status, "experts")


class AdamW:
    """Steps of Adam with decoupled weight decay on tensors of one type, whose gradients lie in tensors of that type or in fp32.  `state`:
    moments in "f32" or "i8"; `master`: 16-bit parameters have a copy in fp32, on which the step is taken.  The tensors are contiguous
    and keep their places, which do not overlap: a parameter that two layers share is given once; parameters that are changed by others
    need load() where there are master copies."""

    def __init__(self, params: list[torch.Tensor], grads: list[torch.Tensor], state: str = "f32", master: bool = False, beta1: float = 0.9, beta2: float = 0.95,
                 eps: float = 1e-8, weight_decay: float = 0.0):
        if not params or len(params) != len(grads):
            raise ValueError(f"{len(params)} parameters and {len(grads)} gradients")
        if state not in ("f32", "i8"):
            raise ValueError(f'state must be "f32" or "i8" (got {state!r})')
        self.device = params[0].device
        for i, (p, g) in enumerate(zip(params, grads)):
            if p.dtype != params[0].dtype or p.dtype not in DTYPES or g.dtype != grads[0].dtype or g.dtype not in (p.dtype, torch.float32):
                raise ValueError(f"tensor {i}: parameter of {p.dtype}, gradient of {g.dtype}")
            if p.numel() != g.numel() or not p.is_contiguous() or not g.is_contiguous():
                raise ValueError(f"tensor {i}: parameter and gradient must be contiguous and as large as one another")
            _check_device(f"parameter {i}", p, self.device)
            _check_device(f"gradient {i}", g, self.device)
        spans = sorted(_span(t) for t in [*params, *grads] if t.numel())
        if any(begin < end for (_, end), (begin, _) in zip(spans, spans[1:])):
            raise ValueError("parameters and gradients overlap")
        if master and params[0].dtype == torch.float32:
            raise ValueError("parameters in fp32 have no master copies")
        self.params, self.grads, self.K, self.count = list(params), list(grads), N.kernels(), 0       # the table points to them
        new = lambda p, t, n: torch.zeros(n, dtype=t, device=p.device)          # noqa: E731
        blocks = lambda p: -(-p.numel() // N.ADAMW_BLOCK)                        # noqa: E731
        small = state == "i8"
        self.m = [new(p, torch.int8 if small else torch.float32, p.numel()) for p in params]
        self.v = [new(p, torch.uint8 if small else torch.float32, p.numel()) for p in params]
        self.m_scale, self.v_scale = ([new(p, torch.float32, blocks(p)) for p in params] if small else None for _ in range(2))
        self.master = [new(p, torch.float32, p.numel()) for p in params] if master else None
        self.load()
        of = lambda tensors, i: tensors[i].data_ptr() if tensors else None       # noqa: E731
        self.table = (N.AdamwTensor * len(params))(*[
            N.AdamwTensor(n=p.numel(), d_param=p.data_ptr(), d_grad=g.data_ptr(), d_master=of(self.master, i), d_m=of(self.m, i), d_v=of(self.v, i),
                          d_m_scale=of(self.m_scale, i), d_v_scale=of(self.v_scale, i)) for i, (p, g) in enumerate(zip(params, grads))])
        self.args = N.AdamwArgs(dtype=DTYPES[params[0].dtype], grad_dtype=DTYPES[grads[0].dtype], state_dtype=N.DT_I8 if small else N.DT_F32, count=len(params),
                                h_tensors=C.addressof(self.table), beta1=beta1, beta2=beta2, eps=eps, weight_decay=weight_decay)

    def load(self) -> None:
        """The master copies from the parameters."""
        for p, c in zip(self.params, self.master or ()):
            c.copy_(p.detach().flatten())

    def step(self, rate: float | torch.Tensor, grad_scale: torch.Tensor | None = None, number: torch.Tensor | None = None) -> None:
        """One step; `grad_scale`: a factor of all gradients, fp32 on the GPU.  A captured step repeats its rate and its number, which are
        part of the launch, unless both are tensors on the GPU: a rate in fp32 and the number of the step, from 1, in int32."""
        told = {}
        for name, t, dtype in (("rate", rate, torch.float32), ("grad_scale", grad_scale, torch.float32), ("number", number, torch.int32)):
            told[name] = None
            if isinstance(t, torch.Tensor):
                if t.dtype != dtype or t.numel() != 1:
                    raise ValueError(f"{name} must be one number in {dtype}")
                _check_device(name, t, self.device)
                told[name] = t.data_ptr()
        self.args.lr, self.args.step = 0.0 if told["rate"] else rate, self.count + 1
        self.args.d_lr, self.args.d_grad_scale, self.args.d_step = told["rate"], told["grad_scale"], told["number"]
        self.K.clpk_adamw(C.byref(self.args), _stream(self.device))
        self.count += 1


def train(norm: Norm, layer: FeedForward, target: tuple[Norm, FeedForward], steps: int, rate: float, state: str = "i8", seed: int = 1) -> list[float]:
    """Steps on a norm and the two trained projections of the layer behind it, towards another norm and layer with the same down projection;
    the mean squared error of every step."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    matrices = AdamW([layer.wg, layer.wu], [layer.dwg, layer.dwu], state, master=True)
    vectors = AdamW([norm.weight, norm.bias], [norm.dweight, norm.dbias])
    losses, waits = [], torch.zeros_like(layer.status)
    for _ in range(steps):
        x = torch.randn(layer.tokens, layer.d, generator=gen, device="cuda").to(torch.bfloat16)
        off = layer.forward(norm.forward(x)).float() - target[1].forward(target[0].forward(x)).float()
        losses.append(off.square().mean())
        dx, _, _ = layer.backward((off * (2 / off.numel() * 1024)).to(torch.bfloat16))      # Adam's step does not see the factor
        norm.backward(dx)
        matrices.step(rate)
        vectors.step(rate)
        waits |= layer.status | target[1].status
    _check_status(waits, "train")
    return [float(v) for v in losses]


def main() -> None:
    d, f, tokens = 512, 1408, 2048
    target = Norm(d, tokens), FeedForward(d, f, tokens, seed=1)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    target[0].weight.copy_(1 + 0.3 * torch.randn(d, generator=gen, device="cuda"))
    for state in ("f32", "i8"):
        norm, layer = Norm(d, tokens), FeedForward(d, f, tokens, seed=2)
        layer.wd.copy_(target[1].wd)
        layer.wd_t.copy_(target[1].wd_t)
        losses = train(norm, layer, target, steps=60, rate=3e-3, state=state)
        print(f"trained a norm and {d} x {f} on {tokens} tokens a step, moments in {state}: mean squared error {losses[0]:.4f} -> {losses[-1]:.4f}")


if __name__ == "__main__":
    main()
