"""What of the feed-forward operators can be told without a GPU: their structures, workspace sizes, and that calls without one fail."""
import ctypes as C
import random
import re
import subprocess
from pathlib import Path

import pytest

from clpeak_b200 import native as N

ROOT = Path(__file__).resolve().parent.parent
STRUCTS = {"clpk_gemm_i8_scaled_args_t": N.GemmI8ScaledArgs, "clpk_gated_ffn_args_t": N.GatedFfnArgs, "clpk_gated_ffn_backward_args_t": N.GatedFfnBackwardArgs}
CALLS = [("clpk_gemm_i8_scaled", N.GemmI8ScaledArgs), ("clpk_gated_ffn", N.GatedFfnArgs), ("clpk_gated_ffn_backward", N.GatedFfnBackwardArgs)]


def test_structures_are_the_headers(tmp_path):
    """Names, offsets and sizes as a C compiler has them."""
    lines = []
    for name, struct in STRUCTS.items():
        lines += [f'printf("{name} . %zu\\n", sizeof({name}));'] + [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in struct._fields_]
    src = tmp_path / "offsets.c"
    src.write_text('#include <stdio.h>\n#include "clpeak_b200_kernels.h"\nint main(void){%s return 0;}\n' % "".join(lines))
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "offsets")], check=True)
    for line in subprocess.run([str(tmp_path / "offsets")], capture_output=True, text=True, check=True).stdout.split("\n")[:-1]:
        name, field, at = line.split()
        struct = STRUCTS[name]
        assert int(at) == (C.sizeof(struct) if field == "." else getattr(struct, field).offset), line


def test_activations_are_numbered_as_in_the_header():
    text = (ROOT / "include" / "clpeak_b200_kernels.h").read_text()
    header = {name: int(v) for name, v in re.findall(r"#define CLPK_(ACT_\w+)\s+(\d+)", text)}
    assert header.pop("ACT_COUNT") == len(header) == 5
    assert all(getattr(N, name) == v for name, v in header.items())


@pytest.mark.parametrize("m,d,f,parts", [(0, 64, 8, 0), (1, 64, 1, 0), (3, 8, 8, 0), (8192, 2048, 8192, 0), (1 << 20, 64, 16384, 0), (4000, 520, 1000, 0),
                                         (147, 656, 7749, 1), (8000, 96, 200, 2)])
def test_workspace_of_the_backward_pass(K, m, d, f, parts):
    """Two matrices of 16-bit gradients with rows of 16 bytes, more than 4 GiB of them too; and where a sum over K is cut, an fp32
    result for each part: at most 32 of them, of dx (1) or of dWg and dWu (2), with rows in whole 256s."""
    gradients = 2 * m * -(-f // 8) * 8 * 2
    for dtype in (N.DT_BF16, N.DT_F16):
        need = C.c_size_t(99)
        K.clpk_gated_ffn_backward_workspace_bytes(dtype, m, d, f, C.byref(need))
        one = (0, -(-m // 256) * 256 * d * 4, 2 * -(-f // 256) * 256 * d * 4)[parts]
        assert need.value == gradients if parts == 0 else (need.value - gradients) % one == 0 and 2 <= (need.value - gradients) // one <= 32
    with pytest.raises(N.ClpkError, match="not BF16 or F16"):
        K.clpk_gated_ffn_backward_workspace_bytes(N.DT_I8, m, d, f, C.byref(C.c_size_t()))
    with pytest.raises(N.ClpkError, match="NULL"):
        K.clpk_gated_ffn_backward_workspace_bytes(N.DT_BF16, m, d, f, None)


@pytest.mark.parametrize("m,d,f", [(2 ** 32 - 1, 64, 64), (64, 2 ** 32 - 1, 64), (64, 64, 2 ** 32 - 1), (2 ** 31 - 256, 2 ** 29 - 64, 8), (8, 2 ** 29 - 64, 2 ** 29 - 64),
                                   (2 ** 24, 2 ** 17, 8)])
def test_sizes_that_cannot_be_counted(K, m, d, f):
    need = C.c_size_t(99)
    with pytest.raises(N.ClpkError, match="too large") as e:
        K.clpk_gated_ffn_backward_workspace_bytes(N.DT_BF16, m, d, f, C.byref(need))
    assert e.value.code == N.ERR_BAD_ARG and need.value == 0


@pytest.mark.parametrize("m,d,f", [(2 ** 22, 2 ** 18, 8), (8, 2 ** 18, 2 ** 22), (2 ** 30, 1, 1), (1, 1, 2 ** 28), (1, 2 ** 28, 1), (1, 1, 1)])
def test_the_largest_sizes_have_a_workspace(K, m, d, f):
    need = C.c_size_t(0)
    K.clpk_gated_ffn_backward_workspace_bytes(N.DT_BF16, m, d, f, C.byref(need))
    gradients = 2 * m * -(-f // 8) * 8 * 2
    assert gradients <= need.value < gradients + (1 << 41)


def test_no_call_without_a_gpu(K):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for call, args in [(getattr(K, name), (C.byref(struct()), None)) for name, struct in CALLS] + [(K.clpk_quantize_rows_i8, (None, None, None, 0, 0, 0, 0, N.DT_F32, None))]:
        with pytest.raises(N.ClpkError) as e:
            call(*args)
        assert e.value.code in (N.ERR_NO_DEVICE, N.ERR_CUDA, N.ERR_UNSUPPORTED)


@pytest.mark.skipif(N._calls() is None, reason="built without the interpreter's headers")
@pytest.mark.parametrize("name,struct", CALLS)
def test_the_same_answer_as_through_ctypes(K, name, struct):
    """Structures by reference, arrays of them, and structures of another call."""
    def outcome(f, args):
        try:
            return f(*args)
        except Exception as e:                                      # noqa: BLE001: whatever either raises
            return type(e), str(e)
    array = (struct * 2)()
    for args in [(C.byref(struct()), 0), (C.byref(struct()), None), (C.byref(array[1]), 0), (C.byref(array), 0), (struct(), 0), (None, 0), (C.byref(N.GemmArgs()), 0),
                 (C.byref(C.c_int()), 0), (C.byref(struct()),), (0, 0), (C.byref(array[0], C.sizeof(struct)), 0), (C.byref(struct()), -1)]:
        assert outcome(getattr(K, name), args) == outcome(lambda *a: K.call(name, *a), args)


def parts_that_may_be(m, d, f):
    """Bytes of fp32 results that the products of the backward pass may be cut into: one of dx and dW, in tiles of 128 or 256 columns,
    where the tiles are fewer than the 74 pairs of the chip and a part has eight blocks of 64 at least."""
    up = lambda a, b: -(-a // b)                                    # noqa: E731
    legal = {0}
    for columns in (128, 256):
        for rows, blocks, products in ((m, 2 * up(f, 64), 1), (f, up(m, 64), 2)):
            if products * up(rows, 256) * up(d, columns) < 74:
                legal |= {products * parts * up(rows, 256) * 256 * up(d, 4) * 4 * 4 for parts in (2, 3, 4, 6, 8, 12, 16, 24, 32) if blocks >= 8 * parts}
    return legal


def test_every_workspace_is_what_its_parts_take(K):
    rng = random.Random(3)
    size = lambda most: round(most ** rng.random())                 # noqa: E731: even over its logarithm
    cases = [(size(1 << 22), size(1 << 14), size(1 << 16)) for _ in range(4000)]
    cases += [(2 ** 22, 2 ** 18, 8), (8, 2 ** 18, 2 ** 22), (2 ** 30, 1, 1), (1, 1, 2 ** 28), (1, 2 ** 28, 1), (1, 1, 1)]
    cut = 0
    for m, d, f in cases:
        need = C.c_size_t(0)
        K.clpk_gated_ffn_backward_workspace_bytes(N.DT_F16, m, d, f, C.byref(need))
        parts = need.value - 2 * m * -(-f // 8) * 8 * 2
        assert parts in parts_that_may_be(m, d, f), (m, d, f, parts)
        cut += parts > 0
    assert cut > 200
