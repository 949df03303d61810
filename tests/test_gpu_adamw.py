"""clpk_adamw against the same operations in torch, each rounded to fp32: equal, bit for bit, but for parameters with moments in 8 bits;
and those against 64 bits."""
import ctypes as C
import math

import pytest
import torch

from clpeak_b200 import native as N
from tests import block_util as B
from tests import ff_util as F

pytestmark = pytest.mark.gpu

# parameters, gradients, master copies
TYPES = [("f32", "f32", False), ("bf16", "bf16", False), ("bf16", "bf16", True), ("bf16", "f32", False), ("bf16", "f32", True),
         ("f16", "f16", False), ("f16", "f16", True), ("f16", "f32", False), ("f16", "f32", True)]
# none, one, around a lane's elements, a block of 256 and a CTA's chunk of 2048
SIZES = [0, 1, 7, 8, 9, 255, 256, 257, 300, 2047, 2048, 2049, 4096, 5000, 70001]


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def step(K, tensors, dtype, grad, state, **k):
    args = B.adamw_args(tensors, dtype, grad, state, **k)
    K.clpk_adamw(C.byref(args), F.stream())


def check(K, tensors, dtype, grad, state, plain=None, **k):
    want = [B.adamw_plain(t, **(k if plain is None else plain)) for t in tensors]
    step(K, tensors, dtype, grad, state, **k)
    for t, w in zip(tensors, want):
        B.same_step(t.values(), w)
        assert t.untouched()


@pytest.mark.parametrize("state", ["f32", "i8"])
@pytest.mark.parametrize("dtype,grad,master", TYPES)
def test_every_type_and_size(K, cuda, dtype, grad, master, state):
    g = gen(1)
    tensors = [B.Tensor(g, n, dtype, grad, state, master) for n in SIZES]
    for i in range(3):
        check(K, tensors, dtype, grad, state, step=i + 1)


@pytest.mark.parametrize("state", ["f32", "i8"])
@pytest.mark.parametrize("dtype,grad,master", [("f32", "f32", False), ("bf16", "f32", True), ("f16", "f16", False)])
@pytest.mark.parametrize("shift", [1, 2, 4, 8])
def test_any_alignment(K, cuda, dtype, grad, master, state, shift):
    g = gen(2)
    check(K, [B.Tensor(g, n, dtype, grad, state, master, shift) for n in (1, 256, 2048, 5001)], dtype, grad, state)


@pytest.mark.parametrize("count", [1, 47, 48, 49, 439, 440, 441, 1000])
def test_as_many_tensors_as_there_are(K, cuda, count):
    """Around what a launch takes of each kind, with empty ones between."""
    g = gen(3)
    tensors = [B.Tensor(g, (37 * i) % 700 if i % 5 else 0, "bf16", "bf16", "i8", False) for i in range(count)]
    check(K, tensors, "bf16", "bf16", "i8")


def test_a_step_against_64_bits(K, cuda):
    """The definition: the bound counts the roundings of fp32, for results of the order of their terms."""
    g = gen(4)
    t = B.Tensor(g, 20000, "f32", "f32", "f32", False)
    p, grad, m, v = (x.double().clone() for x in (t.param, t.grad, t.m, t.v))
    lr, b1, b2, eps, wd, n = 1e-3, 0.9, 0.95, 1e-8, 0.1, 7
    step(K, [t], "f32", "f32", "f32", lr=lr, beta1=b1, beta2=b2, eps=eps, weight_decay=wd, step=n)
    m64, v64 = b1 * m + (1 - b1) * grad, b2 * v + (1 - b2) * grad * grad
    p64 = p - lr * wd * p - lr * (m64 / (1 - b1 ** n)) / (torch.sqrt(v64 / (1 - b2 ** n)) + eps)
    u = B.U
    e_m, e_v = 3 * u * ((b1 * m).abs() + (1 - b1) * grad.abs()), 5 * u * v64
    update = lr * (m64.abs() + e_m) / (1 - b1 ** n) / (torch.sqrt(v64 / (1 - b2 ** n)) + eps)
    F.check(t.m, m64, e_m, "m")
    F.check(t.v, v64, e_v, "v")
    F.check(t.param, p64, 3 * u * p.abs() + 12 * u * update + update * e_m / (m64.abs() + e_m + 1e-300), "p")


@pytest.mark.parametrize("state", ["f32", "i8"])
def test_scaled_gradients(K, cuda, state):
    g = gen(5)
    scale = torch.full((1,), 0.3701, device="cuda")
    check(K, [B.Tensor(g, n, "bf16", "bf16", state, False) for n in (100, 4096)], "bf16", "bf16", state, d_grad_scale=scale.data_ptr(),
          plain={"grad_scale": scale})


@pytest.mark.parametrize("k", [{"beta1": 0.0}, {"beta2": 0.0}, {"weight_decay": 0.0}, {"lr": 0.0}, {"eps": 1.0}, {"beta2": 0.999, "step": 1}, {"beta1": 0.99, "beta2": 0.9999, "step": 10 ** 6}])
@pytest.mark.parametrize("state", ["f32", "i8"])
def test_numbers_of_the_step(K, cuda, state, k):
    g = gen(6)
    check(K, [B.Tensor(g, n, "f32", "f32", state, False) for n in (300, 2048)], "f32", "f32", state, **k)


def test_rate_and_step_from_the_device_in_a_graph(K, cuda):
    g = gen(7)
    tensors = [B.Tensor(g, n, "bf16", "f32", "i8", True) for n in (5, 600, 9000)]
    lr, count = torch.zeros(1, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    args = B.adamw_args(tensors, "bf16", "f32", "i8", lr=float("nan"), step=0, d_lr=lr.data_ptr(), d_step=count.data_ptr())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.clpk_adamw(C.byref(args), F.stream())
    del args                                        # the table was read by the call
    for n in (1, 2, 3, 500):
        lr.fill_(1e-3 / n)
        count.fill_(n)
        want = [B.adamw_plain(t, lr=float(lr), step=n) for t in tensors]
        graph.replay()
        for t, w in zip(tensors, want):
            got = t.values()
            # the step's two factors are formed on the device in 64 bits there: they may be the next fp32 number, one place of their
            # product with the step, 0.01 at most, and of the decay's with the parameter
            w["off"] = w["off"] + 2 * B.U * w["master"].double().abs() + 4e-9
            B.same_step(got, w)


def test_a_step_of_none_is_the_first(K, cuda):
    t, u = (B.Tensor(gen(15), 700, "f32", "f32", "f32", False) for _ in range(2))
    count = torch.zeros(1, dtype=torch.int32, device="cuda")
    step(K, [t], "f32", "f32", "f32", d_step=count.data_ptr())
    count.fill_(1)
    step(K, [u], "f32", "f32", "f32", d_step=count.data_ptr())
    B.same(t.values(), u.values())
    assert bool(torch.isfinite(t.param).all())


def test_blocks_of_nothing_and_of_what_is_not_finite(K, cuda):
    g = gen(8)
    t = B.Tensor(g, 256 * 6 + 10, "f32", "f32", "i8", False)
    block = lambda x, i: x[256 * i:256 * (i + 1)]                # noqa: E731
    for x in (t.grad, t.m, t.v):
        block(x, 0).zero_()                                      # nothing ever
    block(t.grad, 1).fill_(1e-38)                                # below the least scale
    for x in (t.m, t.v):
        block(x, 1).zero_()
    block(t.grad, 2)[17] = float("nan")
    block(t.grad, 3)[5] = float("inf")
    block(t.grad, 4).fill_(1e-9)                                 # small ones beside a large one keep a code
    block(t.grad, 4)[100] = 1.0
    block(t.v, 4).zero_()
    check(K, [t], "f32", "f32", "i8")
    assert bool((block(t.m, 0) == 0).all()) and bool((block(t.v, 0) == 0).all()) and t.m_scale[0] == 0 and t.v_scale[0] == 0
    assert bool(torch.isnan(t.m_scale[2:4]).all()) and bool(torch.isfinite(t.m_scale[[0, 1, 4, 5, 6]]).all())
    assert bool((block(t.v, 4) >= 1).all()) and bool(torch.isfinite(block(t.param, 4)).all())
    # of a NaN among the gradients all but its own element take their step, and with it the moments of the block are NaN
    assert int(torch.isnan(block(t.param, 2)).sum()) == 1
    check(K, [t], "f32", "f32", "i8", step=4)
    assert bool(torch.isnan(block(t.param, 2)).all()) and bool(torch.isfinite(block(t.param, 4)).all())


@pytest.mark.parametrize("power", [-40, -60, -80])
def test_moments_near_the_least_numbers(K, cuda, power):
    """Gradients whose squares are below fp32's normal numbers, or beside them."""
    g = gen(13)
    t = B.Tensor(g, 256 * 8, "f32", "f32", "i8", False)
    t.grad.mul_(2.0 ** power)
    t.v.zero_()
    t.m.zero_()
    t.grad[::3] *= 2.0 ** -24
    check(K, [t], "f32", "f32", "i8", eps=1e-30)


def test_codes_between_two(K, cuda):
    """Sizes whose roots lie next to the middle between two codes: the largest of a block is a code's own, the others are spread about
    (c + 1/2)^2 by single places."""
    n = 256 * 250
    t = B.Tensor(gen(14), n, "f32", "f32", "i8", False)
    block, at = torch.arange(n, device="cuda") // 256, torch.arange(n, device="cuda") % 256
    for x in (t.m, t.v):
        x.zero_()
    # beta1 = beta2 = 0: m is the gradient and sqrt(v) its size; block b has those about (b + 1/2)^2 of 255^2, then of 127^2
    for steps in (255, 127):
        middle = ((block % steps).float() + 0.5) ** 2
        t.grad.copy_(torch.where(at == 0, torch.full_like(middle, float(steps) ** 2), middle * (1 + (at - 128).float() * 2.0 ** -23)))
        check(K, [t], "f32", "f32", "i8", beta1=0.0, beta2=0.0)


def test_codes_are_near_what_they_stand_for(K, cuda):
    """m = s q |q|: half a step of sqrt(m / s) is 1/2, so m is off by s (|q| + 1/4) at most; sqrt(v) = s c^2 likewise, and by s where c is
    raised to 1."""
    g = gen(9)
    small, plain = B.Tensor(g, 8000, "f32", "f32", "i8", False), B.Tensor(gen(9), 8000, "f32", "f32", "f32", False)
    each = lambda s: s.double().repeat_interleave(256)[:8000]    # noqa: E731
    plain.grad.copy_(small.grad)
    plain.m.copy_(each(small.m_scale) * small.m.double() * small.m.double().abs())
    plain.v.copy_((each(small.v_scale) * small.v.double() ** 2) ** 2)
    step(K, [small], "f32", "f32", "i8")
    step(K, [plain], "f32", "f32", "f32")
    q, c = small.m.double(), small.v.double()
    F.check(each(small.m_scale) * q * q.abs(), plain.m.double(), each(small.m_scale) * (q.abs() + 0.26) * 1.0001 + 1e-12, "m")
    F.check(each(small.v_scale) * c * c, plain.v.double().sqrt(), each(small.v_scale) * (c + 0.26) * 1.0001 + 1e-12, "root of v")


def test_steps_in_8_bits_follow_those_in_32(K, cuda):
    """Twenty steps towards a minimum from the same start: where 32 bits go, 8 go too."""
    n, out = 4096, {}
    target = torch.randn(n, generator=gen(10), device="cuda")
    for state in ("f32", "i8"):
        t = B.Tensor(gen(11), n, "f32", "f32", state, False)
        for x in (t.m, t.v, t.param):
            x.zero_()
        for i in range(20):
            t.grad.copy_(t.param - target)
            step(K, [t], "f32", "f32", state, lr=0.01, weight_decay=0.0, step=i + 1)
        out[state] = t.param.clone()
    start = torch.zeros_like(target)
    moved = (out["f32"] - start).norm()
    assert bool(torch.isfinite(out["i8"]).all()) and bool(((out["i8"] - start).sign() == target.sign())[target.abs() > 0.3].all())
    # a code of c is within 1/(2c) of the root of m or of sqrt(v); most are above 30 of 127 and 60 of 255: a few hundredths of each step
    assert (out["i8"] - out["f32"]).norm() < 0.1 * moved


def test_an_empty_call(K, cuda):
    K.clpk_adamw(C.byref(N.AdamwArgs(dtype=N.DT_F32, grad_dtype=N.DT_F32, state_dtype=N.DT_F32, count=0, lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, step=1)), F.stream())
    empty = N.AdamwTensor(n=0)
    K.clpk_adamw(C.byref(N.AdamwArgs(dtype=N.DT_F32, grad_dtype=N.DT_F32, state_dtype=N.DT_I8, count=1, h_tensors=C.addressof(empty), lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8,
                                     step=1)), F.stream())


def test_refusals(K, cuda):
    g = gen(12)

    def refused(match, tensor=None, state="i8", dtype="bf16", grad="bf16", **change):
        t = [B.Tensor(g, 300, dtype, grad, state, False), B.Tensor(g, 300, dtype, grad, state, False)]
        before = [x.values() for x in t]
        args = B.adamw_args(t, dtype, grad, state)
        for name, v in change.items():
            setattr(args, name, v)
        for name, v in (tensor or {}).items():
            setattr(args.table[1], name, v)
        with pytest.raises(N.ClpkError, match=match) as e:
            K.clpk_adamw(C.byref(args), F.stream())
        assert e.value.code == N.ERR_BAD_ARG
        for x, y in zip(t, before):
            B.same(x.values(), y)
    word = torch.zeros(4, device="cuda").data_ptr()
    refused("grad_dtype", grad_dtype=N.DT_F16)
    args = B.adamw_args([], "bf16", "bf16", "f32")
    args.dtype = args.grad_dtype = N.DT_I8
    with pytest.raises(N.ClpkError, match="dtype 5 is not"):
        K.clpk_adamw(C.byref(args), F.stream())
    refused("state_dtype", state_dtype=N.DT_BF16)
    for name in ("beta1", "beta2"):
        for v in (-0.1, 1.0, math.nan):
            refused("beta", **{name: v})
    for v in (0.0, -1.0, 1e-39, 1e30, math.inf, math.nan):
        refused("eps", eps=v)
    for v in (-1.0, math.inf, math.nan):
        refused("lr", lr=v)
        refused("weight_decay", weight_decay=v)
    refused("counted from 1", step=0)
    refused("h_tensors", h_tensors=None)
    refused("is not aligned", d_step=word + 1)
    for name in ("d_param", "d_grad", "d_m", "d_v", "d_m_scale", "d_v_scale"):
        refused(f"{name} of tensor 1", tensor={name: None})
    for name in ("d_param", "d_grad"):
        refused(f"{name} of tensor 1", tensor={name: word + 1})
    for name in ("d_m", "d_v"):
        refused(f"{name} of tensor 1", tensor={name: word + 2}, state="f32")
    refused("d_m_scale of tensor 1", tensor={"d_m_scale": word + 2})
    refused("d_master: give it for every", tensor={"d_master": word})
    refused("no master copies", dtype="f32", grad="f32", tensor={"d_master": word})
    refused("has", tensor={"n": 2 ** 41})
    with pytest.raises(N.ClpkError, match="args is NULL"):
        K.clpk_adamw(None, F.stream())


@pytest.mark.parametrize("power", [0, -113, -112, 127])
def test_the_scale_of_every_number(K, cuda, power):
    """Of all 2^23 numbers between two powers of two: the scale is the quotient by a constant, rounded once, and 0 below 2^-126."""
    count = 1 << 19
    t = B.Tensor.__new__(B.Tensor)
    t.n, t.state, t.master = 256 * count, "i8", None
    t.param, t.grad = (torch.zeros(t.n, device="cuda") for _ in range(2))
    t.m, t.v = torch.zeros(t.n, dtype=torch.int8, device="cuda"), torch.zeros(t.n, dtype=torch.uint8, device="cuda")
    t.m_scale, t.v_scale = (torch.zeros(count, device="cuda") for _ in range(2))
    for part in range(16):
        bits = torch.arange(part * count, (part + 1) * count, device="cuda", dtype=torch.int32) + ((power + 127) << 23)
        size = bits.view(torch.float32)
        t.grad.view(-1, 256)[:, 37] = size
        # beta1 = beta2 = 0: m is the gradient, and the root of its square is its size
        step(K, [t], "f32", "f32", "i8", beta1=0.0, beta2=0.0, lr=0.0)
        for scale, steps in ((t.m_scale, 127), (t.v_scale, 255) if power == 0 else (t.m_scale, 127)):
            want = (size.double() / steps ** 2).float()         # 53 bits are enough for one rounding to 24 behind another
            want = torch.where(want < 2.0 ** -126, torch.zeros_like(want), want)
            assert torch.equal(scale, want)
            codes = (t.m if steps == 127 else t.v).view(-1, 256)[:, 37]
            assert torch.equal(codes, torch.where(want > 0, steps, 0).to(codes.dtype))


def test_steps_side_by_side(K, cuda):
    """Two streams with tensors of their own: as one behind the other."""
    make = lambda: [[B.Tensor(gen(20 + i), n, "bf16", "f32", "i8", True) for n in (70000, 5, 300001)] for i in range(2)]      # noqa: E731
    one, two, streams = make(), make(), [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(5):
        for tensors in one:
            step(K, tensors, "bf16", "f32", "i8", step=i + 1)
    torch.cuda.synchronize()
    for i in range(5):
        for tensors, s in zip(two, streams):
            with torch.cuda.stream(s):
                step(K, tensors, "bf16", "f32", "i8", step=i + 1)
    torch.cuda.synchronize()
    for a, b in zip(one, two):
        for x, y in zip(a, b):
            B.same(x.values(), y.values())


@pytest.mark.parametrize("above", [0.9, 1.01, 16.0])
def test_roots_that_eps_hides(K, cuda, above):
    """Moments whose v lies about 2^-126, where a near root is 0, with eps about the least that makes up for it: 2^-41 of the root's factor."""
    root_scale = 1 / math.sqrt(-math.expm1(3 * math.log(0.95)))
    t = B.Tensor(gen(16), 256 * 8, "f32", "f32", "i8", False)
    for x in (t.m, t.v, t.param):
        x.zero_()
    spread = 2 ** torch.linspace(-4, 1, t.n, device="cuda", dtype=torch.float64)
    t.grad.copy_((2.0 ** -126 * spread / 0.05).sqrt())
    check(K, [t], "f32", "f32", "i8", step=3, eps=above * root_scale * 2.0 ** -41)
    assert bool((t.param < 0).all())
