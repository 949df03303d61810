"""What of the operators that train a block can be told without a GPU: their structures, workspace sizes, and that calls without one fail."""
import ctypes as C
import random
import subprocess
from pathlib import Path

import pytest

from clpeak_b200 import native as N

ROOT = Path(__file__).resolve().parent.parent
STRUCTS = {"clpk_layer_norm_args_t": N.LayerNormArgs, "clpk_layer_norm_backward_args_t": N.LayerNormBackwardArgs, "clpk_adamw_tensor_t": N.AdamwTensor,
           "clpk_adamw_args_t": N.AdamwArgs, "clpk_grouped_gemm_args_t": N.GroupedGemmArgs, "clpk_grouped_gemm_backward_args_t": N.GroupedGemmBackwardArgs}
CALLS = [("clpk_layer_norm", N.LayerNormArgs), ("clpk_layer_norm_backward", N.LayerNormBackwardArgs), ("clpk_adamw", N.AdamwArgs),
         ("clpk_grouped_gemm", N.GroupedGemmArgs), ("clpk_grouped_gemm_backward", N.GroupedGemmBackwardArgs)]


def test_structures_are_the_headers(tmp_path):
    """Names, offsets and sizes as a C compiler has them."""
    lines = []
    for name, struct in STRUCTS.items():
        lines += [f'printf("{name} . %zu\\n", sizeof({name}));'] + [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in struct._fields_]
    src = tmp_path / "offsets.c"
    src.write_text('#include <stdio.h>\n#include "clpeak_b200_kernels.h"\nint main(void){printf("block . %%d\\n", CLPK_ADAMW_BLOCK);%s return 0;}\n' % "".join(lines))
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "offsets")], check=True)
    for line in subprocess.run([str(tmp_path / "offsets")], capture_output=True, text=True, check=True).stdout.split("\n")[:-1]:
        name, field, at = line.split()
        if name == "block":
            assert int(at) == N.ADAMW_BLOCK
            continue
        struct = STRUCTS[name]
        assert int(at) == (C.sizeof(struct) if field == "." else getattr(struct, field).offset), line


def norm_need(K, m, d):
    need = C.c_size_t(99)
    K.clpk_layer_norm_backward_workspace_bytes(m, d, C.byref(need))
    return need.value


def test_workspace_of_the_norms_gradients(K):
    """Whole parts of two rows of fp32, as many as rows at most, and what does for m rows does for fewer."""
    rng = random.Random(1)
    for _ in range(300):
        m, d = round((1 << 20) ** rng.random()), round((1 << 16) ** rng.random())
        need = norm_need(K, m, d)
        assert need % (8 * d) == 0 and 1 <= need // (8 * d) <= min(m, 148)
        assert norm_need(K, max(1, m - rng.randint(0, m)), d) <= need
    assert norm_need(K, 0, 8) > 0
    for m, d in ((2 ** 31, 8), (8, 2 ** 30 + 1), (8, 0)):
        with pytest.raises(N.ClpkError):
            norm_need(K, m, d)
    with pytest.raises(N.ClpkError, match="NULL"):
        K.clpk_layer_norm_backward_workspace_bytes(1, 1, None)


def test_no_call_without_a_gpu(K):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for name, struct in CALLS:
        with pytest.raises(N.ClpkError) as e:
            getattr(K, name)(C.byref(struct()), None)
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
    for args in [(C.byref(struct()), 0), (C.byref(struct()), None), (C.byref(array[1]), 0), (struct(), 0), (None, 0), (C.byref(N.GemmArgs()), 0), (C.byref(struct()),),
                 (C.byref(array[0], C.sizeof(struct)), 0), (C.byref(struct()), -1)]:
        assert outcome(getattr(K, name), args) == outcome(lambda *a: K.call(name, *a), args)


def test_adamw_keeps_what_its_table_points_to():
    """The lists that a program gives are its own to change; the tensors behind the table's addresses stay."""
    import torch

    from clpeak_b200 import block
    params, grads = [torch.ones(8), torch.ones(3)], [torch.zeros(8), torch.zeros(3)]
    kept = [t.data_ptr() for t in params + grads]
    step = block.AdamW(params, grads, "i8")
    params.clear()
    grads[0] = torch.zeros(8)
    assert [t.data_ptr() for t in [*step.params, *step.grads]] == kept
    assert [(t.d_param, t.d_grad) for t in step.table] == list(zip(kept[:2], kept[2:]))
