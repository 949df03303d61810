"""A product kernel of the feed-forward layer whose waits run out ends with an error status -- and not before the loads that it has
asked for have landed: its shared memory is another CTA's then.  The function that waits for them is run here against a model of a
ring whose consumer has given up anywhere; on a GPU only a fault would show it."""
import re
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "clpeak_b200" / "csrc"

MODEL = r"""
#include <cstdint>
#include <cstdio>
#define __device__
#define __forceinline__ inline
static uint32_t g_stages, g_issued, g_unarmed;
static uint64_t ring[16];                           // of a stage: the phases that are complete
// Use n of the ring is stage n % stages, phase n / stages.  A wait for a phase that is not complete lasts until its load lands, which it
// does if it was asked for.
static bool warp_wait(uint64_t *bar, uint32_t parity)
{
    if ((*bar & 1) != parity)
        return true;
    const uint32_t stage = (uint32_t)(bar - ring), use = (uint32_t)*bar * g_stages + stage;
    if (use >= g_issued) {
        g_unarmed++;
        return false;
    }
    ++*bar;
    return true;
}
FUNCTION
int main()
{
    unsigned cases = 0, bad = 0;
    for (g_stages = 1; g_stages <= 12; g_stages++)
        for (g_issued = 0; g_issued <= 5 * g_stages + 1; g_issued++)
            // a stage is asked for again only when its last use was consumed, hence had landed; of the uses after that any may have
            for (uint32_t sure = g_issued > g_stages ? g_issued - g_stages : 0, set = 0; set < 1u << (g_issued - sure); set++) {
                for (uint32_t s = 0; s < 16; s++)
                    ring[s] = 0;
                for (uint32_t use = 0; use < g_issued; use++)
                    if (use < sure || (set >> (use - sure) & 1))
                        ring[use % g_stages] = use / g_stages + 1;
                g_unarmed = 0;
                ring_settled(ring, g_stages, g_issued);
                bool landed = g_unarmed == 0;
                for (uint32_t use = sure; use < g_issued; use++)
                    landed &= ring[use % g_stages] == use / g_stages + 1;
                cases++;
                bad += !landed;
            }
    std::printf("%u %u\n", cases, bad);
}
"""


def test_all_loads_have_landed():
    source = (CSRC / "clpk_pair.cuh").read_text()
    function = re.search(r"__device__ __forceinline__ void ring_settled\(.*?\n\}\n", source, re.S).group(0)
    out = ROOT / "tests" / "_build"
    out.mkdir(exist_ok=True)
    (out / "ring_settled.cpp").write_text(MODEL.replace("FUNCTION", function))
    subprocess.run(["g++", "-O1", "-std=c++17", "-o", str(out / "ring_settled"), str(out / "ring_settled.cpp")], check=True)
    cases, bad = map(int, subprocess.run([str(out / "ring_settled")], check=True, capture_output=True, text=True).stdout.split())
    assert cases > 10000 and bad == 0


@pytest.mark.parametrize("kernel", ["clpk_linear.cuh", "clpk_linear_few.cuh"])
def test_the_kernels_wait_for_them(kernel):
    """Before the barrier of the whole CTA that stands ahead of its end."""
    source = (CSRC / kernel).read_text()
    assert "ring_settled(sh->full, p.stages, issued)" in source
    assert source.index("ring_settled(") < source.rindex("__syncthreads()") and source.index("issued++") < source.index("ring_settled(")
