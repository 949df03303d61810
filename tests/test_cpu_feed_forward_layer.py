"""What the feed-forward layer hands to the kernels, and what it refuses, with its tensors in host memory and the calls written down
instead of made."""
import ctypes as C

import pytest
import torch

from clpeak_b200 import feed_forward as ff
from clpeak_b200 import native as N


class HostTorch:
    """torch, whose "cuda" is host memory."""

    def __getattr__(self, name):
        made = getattr(torch, name)
        if name not in ("Generator", "empty", "randn", "zeros"):
            return made
        return lambda *args, **kw: made(*args, **{**kw, "device": "cpu" if kw.get("device") == "cuda" else kw.get("device")})


class Calls(list):
    """Calls in place of the kernels: (name, arguments), structures by their fields; "x" is what the call finds as x in 16 bits, as a
    copy that it reads may be gone after it.  Sizes come from the library itself."""

    def __init__(self, K):
        self.K = K

    def __getattr__(self, name):
        if name.endswith("_workspace_bytes"):
            return getattr(self.K, name)

        def call(*args):
            args = [{f: getattr(a._obj, f) for f, _ in a._obj._fields_} if isinstance(a, type(C.byref(C.c_int()))) else a for a in args]
            if isinstance(args[0], dict) and args[0].get("d_x") and args[0]["dtype"] == N.DT_BF16 and args[0]["m"]:
                args[0]["x"] = rows_at(args[0]["d_x"], args[0]["m"], args[0]["d"], args[0]["ldx"])
            self.append((name, *args))
        return call

    def of(self, name):
        return [args for called, *args in self if called == name]


@pytest.fixture
def calls(K, monkeypatch):
    made = Calls(K)
    monkeypatch.setattr(ff, "torch", HostTorch())
    monkeypatch.setattr(ff, "_stream", lambda *_: 0)
    monkeypatch.setattr(ff.N, "kernels", lambda: made)
    return made


def values(rows, cols, seed=0):
    gen = torch.Generator()
    gen.manual_seed(seed)
    return torch.randn(rows, cols, generator=gen).to(torch.bfloat16)


def rows_at(address, m, d, pitch):
    """The m rows that a call finds behind an address with a pitch; 0: one behind another."""
    pitch = pitch or d
    flat = (C.c_uint16 * ((m - 1) * pitch + d)).from_address(address)
    return torch.tensor([[flat[r * pitch + c] for c in range(d)] for r in range(m)], dtype=torch.int32)


def bits(x):
    return x.contiguous().view(torch.int16).to(torch.int32) & 0xFFFF


# ---- rows that share elements ---------------------------------------------------------------------------------

def shared_rows():
    """A row for all tokens, a window that moves by eight elements, one row whatever its stride, and rows as they should lie."""
    row = values(1, 64)
    return [row.expand(4, 64), torch.as_strided(values(1, 96), (5, 64), (8, 1)), torch.as_strided(values(1, 64), (1, 64), (0, 1)),
            torch.as_strided(values(1, 64), (1, 64), (3, 1)), values(3, 64), values(3, 200)[:, 8:72]]


@pytest.mark.parametrize("i", range(6))
def test_rows_that_share_elements_reach_the_calls_as_rows(calls, i):
    """A stride of 0 says the same row again to torch and rows one behind another to the calls: what they read has to be x."""
    x = shared_rows()[i]
    m = x.shape[0]
    layer = ff.FeedForward(64, 128, 8)
    layer.forward(x)
    args, = [a[0] for a in calls.of("clpk_gated_ffn")]
    assert args["ldx"] >= 64 and torch.equal(args["x"], bits(x))
    layer.backward(values(m, 64))
    args, = [a[0] for a in calls.of("clpk_gated_ffn_backward")]
    assert torch.equal(args["x"], bits(x))


@pytest.mark.parametrize("i", range(6))
def test_rows_that_share_elements_reach_the_quantiser_as_rows(calls, i):
    x, read = shared_rows()[i], []
    m = x.shape[0]

    class Quantiser:                                            # the copy lives as long as the call
        def clpk_quantize_rows_i8(self, q, scales, src, rows, cols, ld_q, ld, dtype, stream):
            assert ld >= cols
            read.append(bits(x) if cols != 64 else rows_at(src, rows, cols, ld))

        def clpk_gated_ffn(self, args, stream):
            assert args._obj.m == m

        clpk_gemm_i8_scaled = clpk_gated_ffn
    served = ff.ServedFeedForward(ff.FeedForward(64, 128, 8))
    served.K = Quantiser()
    served.forward(x)
    assert len(read) == 2 and torch.equal(read[0], bits(x))


# ---- where x and dy lie ------------------------------------------------------------------------------------------

def test_tensors_elsewhere_are_refused_before_any_call(calls):
    """"meta" stands for another GPU, or for host memory under a layer on a GPU: a device that is not the layer's."""
    layer = ff.FeedForward(64, 128, 8)
    served = ff.ServedFeedForward(layer)
    calls.clear()
    for run in (layer.forward, served.forward):
        for m in (0, 1, 4):
            with pytest.raises(ValueError, match="x must be on cpu"):
                run(values(m, 64).to("meta"))
    layer.forward(values(4, 64))
    calls.clear()
    with pytest.raises(ValueError, match="dy must be on cpu"):
        layer.backward(values(4, 64).to("meta"))
    assert not calls


def test_a_stream_of_another_gpu_is_refused(monkeypatch):
    """Launches go to the current GPU, which cannot read the layer's tensors if that is another one."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: type("Stream", (), {"cuda_stream": 77}))
    assert ff._stream(torch.device("cuda", 1)) == 77
    with pytest.raises(ValueError, match="cuda:0.*cuda:1"):
        ff._stream(torch.device("cuda", 0))


@pytest.mark.parametrize("shape,strides", [((4, 64, 1), (64, 1, 1)), ((4, 64, 3), (64, 1, 256)), ((64,), (1,)), ((), ())])
def test_x_that_is_no_matrix_is_refused(calls, shape, strides):
    """One of three dimensions whose second one has the layer's width is not its first slice."""
    layer = ff.FeedForward(64, 128, 8)
    served = ff.ServedFeedForward(layer)
    calls.clear()
    x = torch.as_strided(values(1, 1024), shape, strides)
    for run in (layer.forward, served.forward):
        with pytest.raises(ValueError, match="x must be bf16"):
            run(x)
    assert not calls


# ---- a call that fails -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("failing", ["clpk_gated_ffn", "clpk_gemm"])
def test_no_backward_pass_of_a_forward_pass_that_failed(calls, failing):
    """The kept g and u are those of an earlier x then, or of this one without a y: gradients would mix the two."""
    layer = ff.FeedForward(64, 128, 8)
    layer.forward(values(8, 64))

    def fails(args, stream):
        raise N.ClpkError(N.ERR_BAD_ARG, "refused", failing)
    setattr(calls, failing, fails)
    with pytest.raises(N.ClpkError):
        layer.forward(values(4, 64))
    delattr(calls, failing)
    with pytest.raises(RuntimeError, match="without forward"):
        layer.backward(values(4, 64))
    layer.forward(values(4, 64))
    layer.backward(values(4, 64))


# ---- workspace ---------------------------------------------------------------------------------------------------

def needed(K, m, d, f):
    need = C.c_size_t(0)
    K.clpk_gated_ffn_backward_workspace_bytes(N.DT_BF16, m, d, f, C.byref(need))
    return need.value


@pytest.mark.parametrize("d,f,tokens", [(1024, 2816, 1024), (512, 1408, 1024), (2048, 2816, 640), (4096, 4096, 264), (4096, 11008, 512), (136, 264, 300),
                                        (8, 8, 1), (64, 128, 65), (1024, 2816, 704), (8, 1408, 2000), (2048, 8, 700)])
def test_the_workspace_does_for_every_number_of_tokens(calls, K, d, f, tokens):
    """Fewer tokens can need more than all of them: their sums are cut into more parts."""
    layer = ff.FeedForward(d, f, tokens)
    layer.x = values(0, d)
    layer.backward(values(0, d))
    args, = [a[0] for a in calls.of("clpk_gated_ffn_backward")]
    most = max(needed(K, m, d, f) for m in range(tokens + 1))
    assert args["workspace_bytes"] == max(most, 16) and layer.workspace.data_ptr() == args["d_workspace"]


@pytest.mark.parametrize("d,f", [(1024, 2816), (4096, 4096), (1, 1), (333, 77), (64, 11008), (2048, 40)])
def test_the_need_grows_within_64_tokens(K, d, f):
    """As the header says: up to a number of tokens, the most is that of a multiple of 64 or of the number itself."""
    need = [needed(K, m, d, f) for m in range(1500)]
    assert all(need[m] >= need[m - 1] for m in range(1, 1500) if (m - 1) % 64)


# ---- waits that ran out --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("word", range(4))
def test_a_wait_that_ran_out_is_told(calls, word):
    layer = ff.FeedForward(64, 128, 8)
    for checked in (layer, ff.ServedFeedForward(layer)):
        checked.check()
        if word < checked.status.numel():
            checked.status[word] = 0x303
            with pytest.raises(N.ClpkError) as e:
                checked.check()
            assert e.value.code == N.ERR_TIMEOUT and str(0x303) in str(e.value)


@pytest.mark.parametrize("step,which", [(1, 0), (3, 0), (2, 1)])
def test_a_wait_that_ran_out_in_any_step_of_a_fit(calls, step, which):
    """Every call clears its status word, so that of a step is gone with the next one."""
    layers = ff.FeedForward(64, 128, 8), ff.FeedForward(64, 128, 8)
    for t in layers:
        t.y.zero_()
    steps = [0, 0]

    def gated(args, stream):
        i = [t.wg.data_ptr() for t in layers].index(args._obj.d_wg)
        steps[i] += 1
        layers[i].status[0] = 0x301 if (steps[i], i) == (step, which) else 0
    calls.clpk_gated_ffn = gated
    with pytest.raises(N.ClpkError, match=str(0x301)):
        ff.fit(*layers, steps=3, rate=0.1)
