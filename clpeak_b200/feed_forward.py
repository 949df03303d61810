"""A gated feed-forward layer  y = (act(x Wg^T) * (x Wu^T)) Wd^T  on the framework's products, trained in 16 bits and served in 8.

    layer = FeedForward(d=1024, f=2816, tokens=4096)
    y = layer.forward(x)                      # bf16, keeps what the backward pass needs
    dx, dwg, dwu = layer.backward(dy)         # gradients of x and of the two projections that are trained
    served = ServedFeedForward(layer)         # weights quantised once, one scale for each output channel
    y = served.forward(x)                     # tokens quantised on the way, one scale for each

Buffers, workspaces and argument structures are set up once and used again by every call; calls run on torch's current stream.  What a
call returns is a view of them: it is good until the layer's next call of that kind, and a program that needs it longer copies it.  x
is read again by backward() and has to be as it was until then.  A layer is for one stream and one host thread at a time: every
call of another stream or thread needs a layer of its own, or has to come after the calls before it.
``python -m clpeak_b200.feed_forward`` fits the projections of a small layer to those of another one and then serves it.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import native as N


def _stream(device: torch.device) -> int:
    """The current stream, which has to be one of the GPU that the layer's tensors lie on."""
    if torch.cuda.current_device() != device.index:
        raise ValueError(f"the layer is on {device}, the current device is cuda:{torch.cuda.current_device()}")
    return torch.cuda.current_stream().cuda_stream


def _check_device(name: str, t: torch.Tensor, device: torch.device) -> None:
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, as the layer (got {t.device})")


def _bytes(n: int) -> torch.Tensor:
    return torch.empty(max(int(n), 16), dtype=torch.uint8, device="cuda")


def _wide(rows: int, cols: int, dtype: torch.dtype) -> torch.Tensor:
    """A matrix whose rows lie at multiples of 16 bytes."""
    unit = 16 // dtype.itemsize
    return torch.empty(rows, -(-cols // unit) * unit, dtype=dtype, device="cuda")[:, :cols]


def _check_x(x: torch.Tensor, layer) -> None:
    if x.dtype != torch.bfloat16 or x.dim() != 2 or x.shape[1] != layer.d or x.stride(1) != 1 or x.shape[0] > layer.tokens:
        raise ValueError(f"x must be bf16 [up to {layer.tokens}][{layer.d}] with rows of neighbours")
    _check_device("x", x, layer.device)


def _check_status(status: torch.Tensor, what: str) -> None:
    if status.any():
        raise N.ClpkError(N.ERR_TIMEOUT, f"status words {status.tolist()}", what)


def _rows(x: torch.Tensor):
    """x and its pitch as the calls take it.  A stride of 0 is one row for all tokens to torch, and rows one behind another to the
    calls: rows that share elements are copied.  The stride of a single row says nothing."""
    m, d = x.shape
    if m > 1 and x.stride(0) < d:
        x = x.contiguous()
    return x, x.stride(0) if m > 1 else d


class FeedForward:
    """The layer in bf16 for up to `tokens` tokens.  The down projection is frozen: its transpose is kept beside it, for the
    gradient of h is a product with it.  `d` and `f` are multiples of 8 (rows of 16 bytes, which clpk_gemm asks for)."""

    def __init__(self, d: int, f: int, tokens: int, activation: int = N.ACT_SILU, seed: int = 0):
        if d % 8 or f % 8:
            raise ValueError(f"d and f must be multiples of 8 (got {d}, {f})")
        self.d, self.f, self.tokens, self.activation = d, f, tokens, activation
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        weight = lambda rows, cols: (torch.randn(rows, cols, generator=gen, device="cuda") * cols ** -0.5).to(torch.bfloat16)  # noqa: E731
        self.wg, self.wu, self.wd = weight(f, d), weight(f, d), weight(d, f)
        self.wd_t = self.wd.T.contiguous()
        self.device = self.wg.device
        # a matrix of h's shape for each: what the forward pass keeps, and the gradient of h
        self.h, self.g, self.u, self.dh = (torch.empty(tokens, f, dtype=torch.bfloat16, device="cuda") for _ in range(4))
        self.y, self.dx = (torch.empty(tokens, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.dwg, self.dwu = torch.empty_like(self.wg), torch.empty_like(self.wu)
        self.status = torch.zeros(4, dtype=torch.int32, device="cuda")
        self.K = N.kernels()
        # fewer tokens can need more (their sums are cut into more parts); the most is that of a multiple of 64 or of all
        self.workspace = _bytes(max(self._need(m) for m in (*range(64, tokens, 64), tokens)))
        self.x = None

    def _status(self, i: int) -> int:
        return self.status.data_ptr() + 4 * i

    def _need(self, m: int) -> int:
        need = C.c_size_t(0)
        self.K.clpk_gated_ffn_backward_workspace_bytes(N.DT_BF16, m, self.d, self.f, C.byref(need))
        return need.value

    def _gemm(self, a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, i: int) -> None:
        args = N.GemmArgs(dtype=N.DT_BF16, m=a.shape[0], n=b.shape[0], k=a.shape[1], d_a=a.data_ptr(), d_b=b.data_ptr(), d_c=c.data_ptr(),
                          alpha=1.0, d_status=self._status(i))
        self.K.clpk_gemm(C.byref(args), _stream(self.device))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        _check_x(x, self)
        m = x.shape[0]
        if m == 0:
            self.x = x
            return self.y[:0]
        x, ldx = _rows(x)
        self.x = None                                   # until h, g, u and y are of this x
        args = N.GatedFfnArgs(dtype=N.DT_BF16, activation=self.activation, m=m, d=self.d, f=self.f, d_x=x.data_ptr(), d_wg=self.wg.data_ptr(),
                              d_wu=self.wu.data_ptr(), d_h=self.h.data_ptr(), d_g=self.g.data_ptr(), d_u=self.u.data_ptr(), ldx=ldx,
                              d_status=self._status(0))
        self.K.clpk_gated_ffn(C.byref(args), _stream(self.device))
        self._gemm(self.h[:m], self.wd, self.y, 1)
        self.x = x
        return self.y[:m]

    def backward(self, dy: torch.Tensor):
        """(dx, dwg, dwu) from the gradient of the last forward pass's y."""
        if self.x is None:
            raise RuntimeError("backward() without forward()")
        x, m = self.x, self.x.shape[0]
        if dy.dtype != torch.bfloat16 or tuple(dy.shape) != (m, self.d) or not dy.is_contiguous():
            raise ValueError(f"dy must be contiguous bf16 [{m}][{self.d}]")
        _check_device("dy", dy, self.device)
        if m:
            self._gemm(dy, self.wd_t, self.dh, 2)
        # x's pitch is that of dx as well: a pitch of dx's own where x is a slice
        if m > 1 and x.stride(0) != self.d:
            x = x.contiguous()
        args = N.GatedFfnBackwardArgs(dtype=N.DT_BF16, activation=self.activation, m=m, d=self.d, f=self.f, d_x=x.data_ptr(), d_wg=self.wg.data_ptr(),
                                      d_wu=self.wu.data_ptr(), d_dh=self.dh.data_ptr(), d_g=self.g.data_ptr(), d_u=self.u.data_ptr(),
                                      d_dx=self.dx.data_ptr(), d_dwg=self.dwg.data_ptr(), d_dwu=self.dwu.data_ptr(),
                                      d_workspace=self.workspace.data_ptr(), workspace_bytes=self.workspace.numel(), d_status=self._status(3))
        self.K.clpk_gated_ffn_backward(C.byref(args), _stream(self.device))
        return self.dx[:m], self.dwg, self.dwu

    def check(self) -> None:
        """Raises if a device-side wait expired in the last forward or backward pass, whose results are wrong then.  Waits for the
        stream."""
        _check_status(self.status, "feed-forward layer")


class ServedFeedForward:
    """The same layer in 8-bit integers for up to `tokens` tokens a call: four launches."""

    def __init__(self, layer: FeedForward, tokens: int | None = None):
        self.d, self.f, self.tokens, self.activation, self.K = layer.d, layer.f, tokens or layer.tokens, layer.activation, layer.K
        self.device = layer.device
        self.weights = {name: self._quantize(getattr(layer, name)) for name in ("wg", "wu", "wd")}
        self.xq, self.hq = _wide(self.tokens, self.d, torch.int8), _wide(self.tokens, self.f, torch.int8)
        self.xs, self.hs = (torch.empty(self.tokens, device="cuda") for _ in range(2))
        self.h, self.y = _wide(self.tokens, self.f, torch.bfloat16), _wide(self.tokens, self.d, torch.bfloat16)
        self.status = torch.zeros(2, dtype=torch.int32, device="cuda")
        ptr = lambda name, i: self.weights[name][i].data_ptr()  # noqa: E731
        self.gated = N.GatedFfnArgs(dtype=N.DT_I8, out_dtype=N.DT_BF16, activation=self.activation, d=self.d, f=self.f, d_x=self.xq.data_ptr(),
                                    d_wg=ptr("wg", 0), d_wu=ptr("wu", 0), d_x_scale=self.xs.data_ptr(), d_wg_scale=ptr("wg", 1), d_wu_scale=ptr("wu", 1),
                                    d_h=self.h.data_ptr(), ldx=self.xq.stride(0), ldw=self.weights["wg"][0].stride(0), ldh=self.h.stride(0),
                                    d_status=self.status.data_ptr())
        self.down = N.GemmI8ScaledArgs(n=self.d, k=self.f, out_dtype=N.DT_BF16, d_a=self.hq.data_ptr(), d_b=ptr("wd", 0), d_c=self.y.data_ptr(),
                                       lda=self.hq.stride(0), ldb=self.weights["wd"][0].stride(0), ldc=self.y.stride(0), d_a_scale=self.hs.data_ptr(),
                                       d_b_scale=ptr("wd", 1), d_status=self.status.data_ptr() + 4)

    def _quantize(self, w: torch.Tensor):
        q, scale = _wide(*w.shape, torch.int8), torch.empty(w.shape[0], device="cuda")
        self.K.clpk_quantize_rows_i8(q.data_ptr(), scale.data_ptr(), w.data_ptr(), *w.shape, q.stride(0), w.stride(0), N.DT_BF16, _stream(self.device))
        return q, scale

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        _check_x(x, self)
        m = x.shape[0]
        x, ldx = _rows(x)
        s, K = _stream(self.device), self.K
        self.gated.m = self.down.m = m
        K.clpk_quantize_rows_i8(self.xq.data_ptr(), self.xs.data_ptr(), x.data_ptr(), m, self.d, self.xq.stride(0), ldx, N.DT_BF16, s)
        K.clpk_gated_ffn(C.byref(self.gated), s)
        K.clpk_quantize_rows_i8(self.hq.data_ptr(), self.hs.data_ptr(), self.h.data_ptr(), m, self.f, self.hq.stride(0), self.h.stride(0), N.DT_BF16, s)
        K.clpk_gemm_i8_scaled(C.byref(self.down), s)
        return self.y[:m]

    def check(self) -> None:
        """Raises if a device-side wait expired in the last pass, whose results are wrong then.  Waits for the stream."""
        _check_status(self.status, "feed-forward layer in 8 bits")


def fit(layer: FeedForward, target: FeedForward, steps: int, rate: float, seed: int = 1) -> list[float]:
    """Gradient descent on the two projections towards another layer with the same down projection; the mean squared error of every
    step."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    wg, wu = layer.wg.float(), layer.wu.float()
    losses, waits = [], torch.zeros_like(layer.status)
    for _ in range(steps):
        x = torch.randn(layer.tokens, layer.d, generator=gen, device="cuda").to(torch.bfloat16)
        off = layer.forward(x).float() - target.forward(x).float()
        losses.append(off.square().mean())
        _, dwg, dwu = layer.backward((off * (2 / layer.tokens)).to(torch.bfloat16))
        wg -= rate * dwg.float()
        wu -= rate * dwu.float()
        layer.wg.copy_(wg)
        layer.wu.copy_(wu)
        waits |= layer.status | target.status
    _check_status(waits, "fit")
    return [float(v) for v in losses]


def main() -> None:
    d, f, tokens = 512, 1408, 2048
    target, layer = FeedForward(d, f, tokens, seed=1), FeedForward(d, f, tokens, seed=2)
    layer.wd.copy_(target.wd)
    layer.wd_t.copy_(target.wd_t)
    losses = fit(layer, target, steps=60, rate=0.2)
    print(f"fitted {d} x {f} on {tokens} tokens a step: mean squared error {losses[0]:.4f} -> {losses[-1]:.4f}")
    x = torch.randn(tokens, d, device="cuda").to(torch.bfloat16)
    y = layer.forward(x).float()
    served = ServedFeedForward(layer)
    for m in (1, 64, tokens):
        off = (served.forward(x[:m]).float() - y[:m]).norm() / y[:m].norm()
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        for _ in range(50):
            served.forward(x[:m])
        end.record()
        end.synchronize()
        served.check()
        print(f"served in 8 bits, {m} tokens: {float(off):.4f} off the layer in bf16, {begin.elapsed_time(end) / 50 * 1e3:.1f} us a call")


if __name__ == "__main__":
    main()
