"""The operators that train a block, one behind another as a program calls them (clpeak_b200.block)."""
import pytest
import torch

from clpeak_b200 import block
from clpeak_b200 import native as N
from clpeak_b200.feed_forward import FeedForward
from tests import block_util as B
from tests import ff_util as F

pytestmark = pytest.mark.gpu


def randn(*shape, seed, std=1.0, dtype=torch.bfloat16):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)


def near(got, want, what):
    """Rounded to bf16 on the way a few times, 2^-8 each of what they are then: of the order of 2^-6 of the norm."""
    off = (got.double() - want.double()).norm() / want.double().norm()
    assert off < 2.0 ** -6, (what, float(off))


def test_norm_then_experts_then_a_step(K, cuda):
    """A block of experts behind a norm: forward, gradients of all that is trained against autograd in 64 bits, and two steps."""
    d, n, rows, spare = 264, 136, [70, 0, 33, 129, 1], 6
    m = sum(rows) + spare
    norm, experts = block.Norm(d, m), block.Experts(len(rows), n, d, m, seed=1)
    norm.weight.copy_(randn(d, seed=2, std=0.2, dtype=torch.float32) + 1)
    norm.bias.copy_(randn(d, seed=3, std=0.2, dtype=torch.float32))
    offsets = B.offsets_of(rows)
    vectors = block.AdamW([norm.weight, norm.bias], [norm.dweight, norm.dbias], weight_decay=0.1)
    matrices = block.AdamW([experts.w], [experts.dw], "i8", master=True)
    for turn in range(2):
        x, dy = randn(m, d, seed=10 + turn), randn(m, n, seed=20 + turn, std=0.1)
        # in 64 bits
        x64, w64, b64, e64 = (t.double().clone().requires_grad_() for t in (x, norm.weight, norm.bias, experts.w))
        off = x64 - x64.mean(1, keepdim=True)
        h = off / torch.sqrt((off * off).mean(1, keepdim=True) + norm.eps) * w64 + b64
        parts, at = [], 0
        for e, r in enumerate(rows):
            parts.append(h[at:at + r] @ e64[e].T)
            at += r
        y64 = torch.cat(parts)
        want = torch.autograd.grad((y64 * dy[:sum(rows)].double()).sum(), (x64, w64, b64, e64))
        # here
        y = experts.forward(norm.forward(x), offsets)
        near(y[:sum(rows)], y64, "y")
        assert bool((y[sum(rows):] == 0).all())
        dh, dw = experts.backward(dy)
        dx, dweight, dbias = norm.backward(dh)
        for got, w, what in zip((dx, dweight, dbias, dw), want, ("dx", "dweight", "dbias", "dw")):
            near(got, w, what)
        assert bool((dx[sum(rows):] == 0).all())
        experts.check()
        before = experts.w.clone(), norm.weight.clone()
        matrices.step(1e-3)
        vectors.step(1e-3)
        assert matrices.count == vectors.count == turn + 1
        # a step goes against the gradient, by the rate at most where the moments are new
        moved = (experts.w - before[0]).double()
        assert float((moved * dw.double()).sum()) < 0 and torch.equal(experts.w.flatten(), matrices.master[0].to(torch.bfloat16))
        if turn == 0:
            assert float((norm.weight - before[1]).abs().max()) <= 1e-3 * (1 + 0.1 * 3) * 1.001


def test_the_whole_step_in_a_graph(K, cuda):
    """Norm, feed-forward layer, both backward passes and the step, captured once: as the same calls one by one."""
    d, f, tokens = 128, 256, 300

    def parts():
        norm, layer = block.Norm(d, tokens), FeedForward(d, f, tokens, seed=4)
        return norm, layer, block.AdamW([layer.wg, layer.wu], [layer.dwg, layer.dwu], "i8", master=True), block.AdamW([norm.weight, norm.bias], [norm.dweight, norm.dbias])

    def turn(norm, layer, matrices, vectors, x, dy):
        layer.forward(norm.forward(x))
        dx, _, _ = layer.backward(dy)
        norm.backward(dx)
        matrices.step(1e-3)
        vectors.step(1e-3)
    x, dy = randn(tokens, d, seed=5), randn(tokens, d, seed=6, std=0.1)
    one, two = parts(), parts()
    for _ in range(2):
        turn(*one, x, dy)
    turn(*two, x, dy)
    two[2].count = two[3].count = 1                     # the captured step is the second
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turn(*two, x, dy)
    graph.replay()
    for a, b in zip((one[1].wg, one[1].wu, one[0].weight, one[0].bias), (two[1].wg, two[1].wu, two[0].weight, two[0].bias)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("state", ["f32", "i8"])
def test_training_runs(K, cuda, state):
    d, f, tokens = 64, 128, 256
    target = block.Norm(d, tokens), FeedForward(d, f, tokens, seed=1)
    norm, layer = block.Norm(d, tokens), FeedForward(d, f, tokens, seed=2)
    layer.wd.copy_(target[1].wd)
    layer.wd_t.copy_(target[1].wd_t)
    losses = block.train(norm, layer, target, steps=4, rate=1e-3, state=state)
    assert len(losses) == 4 and all(torch.isfinite(torch.tensor(losses)))
    for t in (layer.wg, layer.wu, norm.weight, norm.bias):
        assert bool(torch.isfinite(t).all())


def test_rows_that_share_elements_and_slices(K, cuda):
    norm = block.Norm(40, 9)
    row = randn(1, 40, seed=7)
    y = norm.forward(row.expand(9, 40)).clone()
    assert torch.equal(y, norm.forward(row.repeat(9, 1)))
    wide = randn(9, 96, seed=8)
    y = norm.forward(wide[:, 8:48]).clone()
    assert torch.equal(y, norm.forward(wide[:, 8:48].contiguous()))


def test_refusals(K, cuda):
    norm, experts = block.Norm(40, 9), block.Experts(3, 16, 24, 9)
    x = randn(9, 40, seed=9)
    with pytest.raises(RuntimeError, match="without forward"):
        norm.backward(x)
    with pytest.raises(RuntimeError, match="without forward"):
        experts.backward(x[:, :16].contiguous())
    for bad in (x.float(), x[:, :39], x[0], x.T, torch.cat((x, x))):
        with pytest.raises(ValueError, match="x must be"):
            norm.forward(bad)
    with pytest.raises(ValueError, match="must be on"):
        norm.forward(x.cpu())
    norm.forward(x)
    with pytest.raises(ValueError, match="9 rows"):
        norm.backward(x[:8])
    with pytest.raises(ValueError, match="multiples of 8"):
        block.Experts(3, 12, 24, 9)
    with pytest.raises(ValueError, match="offsets"):
        experts.forward(randn(9, 24, seed=1), torch.zeros(3, dtype=torch.int32, device="cuda"))
    experts.forward(randn(9, 24, seed=1), torch.tensor([0, 4, 3, 9], dtype=torch.int32, device="cuda"))
    with pytest.raises(N.ClpkError, match="offsets") as e:
        experts.check()
    assert e.value.code == N.ERR_BAD_ARG
    p, g = torch.zeros(8, device="cuda"), torch.zeros(8, device="cuda")
    for params, grads, k in (([], [], {}), ([p], [], {}), ([p], [g.half()], {}), ([p], [torch.zeros(9, device="cuda")], {}), ([p], [g], {"state": "i4"}),
                             ([p], [g], {"master": True}), ([p, p.half()], [g, g], {}), ([p], [g.cpu()], {})):
        with pytest.raises(ValueError):
            block.AdamW(params, grads, **k)
    step = block.AdamW([p], [g])
    with pytest.raises(ValueError, match="grad_scale"):
        step.step(1e-3, torch.zeros(2, device="cuda"))
    with pytest.raises(N.ClpkError, match="lr"):
        step.step(-1.0)
    assert step.count == 0


def test_results_as_arguments(K, cuda):
    """An object's own results lie where its next call writes; a copy, or another object's, will do."""
    norm, other, experts = block.Norm(16, 9), block.Norm(16, 9), block.Experts(3, 16, 16, 9)
    offsets = torch.tensor([0, 4, 4, 9], dtype=torch.int32, device="cuda")
    x = randn(9, 16, seed=10)
    y, z = norm.forward(x), experts.forward(x, offsets)
    for call, name in ((lambda: norm.forward(y), "x lies in .* y"), (lambda: norm.forward(norm.dx[:4]), "x lies in .* dx"), (lambda: norm.backward(norm.dx), "dy lies"),
                       (lambda: experts.forward(z, offsets), "x lies in .* y"), (lambda: experts.forward(experts.dx, offsets), "x lies in .* dx"),
                       (lambda: experts.backward(experts.dx), "dy lies")):
        with pytest.raises(ValueError, match=name):
            call()
    assert torch.equal(other.forward(y), other.forward(y.clone())) and torch.equal(norm.y, y)
    want = other.forward(y).clone()
    assert torch.equal(norm.forward(y.clone()), want)
    want = experts.forward(z.clone(), offsets).clone()
    assert torch.equal(experts.forward(x, offsets), z) and torch.equal(experts.forward(z.clone(), offsets), want)


def test_tensors_that_overlap_and_parameters_with_gradients(K, cuda):
    p, g = torch.randn(40, device="cuda"), torch.randn(40, device="cuda")
    for params, grads in (([p, p], [g, g.clone()]), ([p[:8], p[7:]], [g[:8], g[7:].clone()]), ([p, p.clone()], [g, g]), ([p], [p])):
        with pytest.raises(ValueError, match="overlap"):
            block.AdamW(params, grads)
    halves = block.AdamW([p[:8], p[8:], p[:0]], [g[:8], g[8:], g[:0]])
    whole = torch.nn.Parameter(p.clone())
    all_of = block.AdamW([whole], [g.clone()])
    halves.step(1e-2)
    all_of.step(1e-2)
    assert torch.equal(p, whole.detach())
    weight = torch.nn.Parameter(torch.randn(300, device="cuda").half())
    step = block.AdamW([weight], [torch.randn(300, device="cuda")], master=True)
    step.step(1e-2)
    assert not step.master[0].requires_grad and torch.equal(step.master[0].half(), weight.detach())


@pytest.mark.parametrize("state", ["f32", "i8"])
def test_a_captured_step_that_counts(K, cuda, state):
    """Rate and number in tensors are those of each replay: as steps one by one."""
    p, g = randn(700, seed=11, dtype=torch.float32), randn(700, seed=12, dtype=torch.float32)
    one, two = (block.AdamW([p.clone()], [g.clone()], state) for _ in range(2))
    rate, number = torch.zeros((), device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        two.step(rate, number=number)
        number += 1
    for i in range(4):
        rate.fill_(0.5 ** (i + 4))
        graph.replay()
        one.step(0.5 ** (i + 4))
        assert torch.equal(one.params[0], two.params[0]), i
    for bad in ({"rate": torch.zeros(2, device="cuda")}, {"rate": rate.half()}, {"rate": rate, "number": number.long()}, {"rate": rate, "number": number.cpu()}):
        with pytest.raises(ValueError):
            two.step(**bad)


@pytest.mark.parametrize("state", ["f32", "i8"])
def test_gradients_of_a_training_step(K, cuda, state):
    """One step of train(): its loss and all its gradients against autograd in 64 bits, and each parameter goes against its own."""
    d, f, tokens = 64, 128, 256
    target, norm, layer = (block.Norm(d, tokens), FeedForward(d, f, tokens, seed=1)), block.Norm(d, tokens), FeedForward(d, f, tokens, seed=2)
    layer.wd.copy_(target[1].wd)
    layer.wd_t.copy_(target[1].wd_t)
    for i, t in enumerate((target[0].weight, norm.weight)):
        t.add_(randn(d, seed=30 + i, std=0.3, dtype=torch.float32))
    for i, t in enumerate((target[0].bias, norm.bias)):
        t.add_(randn(d, seed=40 + i, std=0.3, dtype=torch.float32))
    trained = {"weight": norm.weight, "bias": norm.bias, "wg": layer.wg, "wu": layer.wu}
    before = {name: t.clone() for name, t in trained.items()}
    x = randn(tokens, d, seed=1)                            # train()'s own, of the same seed

    def run(norm, layer, weight, bias, wg, wu):
        x64 = x.double()
        off = x64 - x64.mean(1, keepdim=True)
        h = off / torch.sqrt((off * off).mean(1, keepdim=True) + norm.eps) * weight + bias
        return (F.act64("silu", h @ wg.T) * (h @ wu.T)) @ layer.wd.double().T
    leaves = [t.double().clone().requires_grad_() for t in before.values()]
    loss = (run(norm, layer, *leaves) - run(*target, *(t.double() for t in (target[0].weight, target[0].bias, target[1].wg, target[1].wu)))).square().mean()
    want = torch.autograd.grad(loss * 1024, leaves)         # train() scales by it
    losses = block.train(norm, layer, target, steps=1, rate=1e-3, state=state)
    # bf16 rounds the norm's rows, h and y on both sides of the difference: as near() counts
    assert len(losses) == 1 and abs(losses[0] - float(loss.detach())) < 2.0 ** -6 * float(loss.detach())
    for (name, t), got, w in zip(trained.items(), (norm.dweight, norm.dbias, layer.dwg, layer.dwu), want):
        near(got, w, name)
        moved = t.double() - before[name].double()
        assert float((moved * w).sum()) < 0 and float(moved.abs().max()) > 0, name


def test_weights_gradients_as_arguments(K, cuda):
    """Experts' dw has rows as long as x's, and as dy's where n is k; the backward pass writes it while it reads both."""
    experts, other = block.Experts(3, 16, 16, 9), block.Experts(3, 16, 16, 9)
    offsets = torch.tensor([0, 4, 4, 9], dtype=torch.int32, device="cuda")
    x, dy = randn(9, 16, seed=13), randn(9, 16, seed=14)
    experts.forward(x, offsets)
    dw = experts.backward(dy)[1]
    for call, name in ((lambda: experts.forward(dw[1, :9], offsets), "x lies in .* dw"), (lambda: experts.backward(dw[2, 2:11]), "dy lies in .* dw")):
        with pytest.raises(ValueError, match=name):
            call()
    assert torch.equal(other.forward(dw[0, :9], offsets), other.forward(dw[0, :9].clone(), offsets))
