"""The sizes that the feed-forward operators are tested at on a GPU take every choice that their planning code makes: it is compiled
into a program of its own and asked how it cuts the tests' sizes, and sizes drawn over the whole range."""
import random
import shutil
import subprocess
from pathlib import Path

import pytest

from clpeak_b200 import build
from tests import test_gpu_feed_forward as G

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def plans():
    """[(form, tokens, k, n)] -> how each is cut.  The program fails where a launch would not fit its memory, or a tile would have no cluster."""
    if not (shutil.which("nvcc") or Path("/usr/local/cuda/bin/nvcc").exists()):
        pytest.skip("no nvcc")
    src, exe = ROOT / "tests" / "host_check" / "feed_forward_plans.cu", ROOT / "tests" / "_build" / "feed_forward_plans"
    exe.parent.mkdir(exist_ok=True)
    deps = [src, *build.CSRC.glob("*.cuh"), *build.CSRC.glob("*.h"), build.CSRC / "kernels" / "feed_forward.cu", ROOT / "include" / "clpeak_b200_kernels.h"]
    if not exe.exists() or exe.stat().st_mtime < max(p.stat().st_mtime for p in deps):
        subprocess.run([build._nvcc(), "-gencode", "arch=compute_100a,code=compute_100a", "-Xcicc", "-O0", "-O1", "-std=c++17", "-I", str(build.CSRC),
                        "-o", str(exe), str(src)], check=True)

    def ask(cases):
        r = subprocess.run([str(exe)], input="".join(f"{f} {m} {k} {n}\n" for f, m, k, n in cases), capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, f"{r.returncode} of the cases do not fit"
        return r.stdout.splitlines()
    return ask


def listed(argument):
    """The sizes of a test of test_gpu_feed_forward.py, from its own marks."""
    return [tuple(v) for mark in getattr(G, argument).pytestmark if mark.name == "parametrize" and "," in mark.args[0] for v in mark.args[1]]


def sizes_of_the_tests():
    """(form, tokens, k, n) of every test there; forms as in feed_forward_plans.cu."""
    gated = listed("test_gated_sizes") + listed("test_gated_splits") + listed("test_gated_large") + listed("test_gated_in_every_width") + G.PAIRS_GATED
    gated_8 = listed("test_gated_8_bits") + [(m, 2 * d, f) for m, d, f in listed("test_gated_8_bits_splits") + listed("test_gated_in_every_width")] + G.PAIRS_GATED_8
    scaled = listed("test_scaled_product") + listed("test_scaled_product_splits") + listed("test_scaled_product_in_every_width") + G.PAIRS_SCALED
    gradients = listed("test_backward_sizes") + listed("test_backward_splits") + listed("test_backward_large") + listed("test_backward_in_every_number_of_parts")
    return [(form, *size) for form, sizes in (("g", gated), ("i", gated_8), ("s", scaled), ("b", gradients)) for size in sizes]


def drawn(n):
    rng = random.Random(4)
    size = lambda most: round(most ** rng.random())             # noqa: E731: even over its logarithm
    return [(rng.choice("gisbb"), size(16384), size(16384), size(20000)) for _ in range(n)]


def test_every_choice_is_tested(plans):
    some, many = sizes_of_the_tests(), drawn(200000)
    assert len(some) > 150
    taken = {(case[0], plan) for case, plan in zip(some, plans(some), strict=True)}
    missing = {}
    for case, plan in zip(many, plans(many), strict=True):
        if (case[0], plan) not in taken:
            missing.setdefault((case[0], plan), case)
    assert not missing


def test_the_largest_sizes_fit(plans):
    plans([(form, m, k, n) for form in "gisb" for m in (1, 64, 65, 96, 97, 128, 129, 1 << 20) for k in (1, 64, 131071) for n in (1, 129, 1 << 20)])
