"""The products of groups, by their source: every wait has its limit and tells what ran out, loads land before the CTA's memory goes away,
and no pair waits for another."""
import re
from pathlib import Path

SOURCE = (Path(__file__).resolve().parent.parent / "clpeak_b200" / "csrc" / "kernels" / "grouped_gemm.cu").read_text()
KERNEL = SOURCE[SOURCE.index("grouped_kernel(const __grid_constant__"):SOURCE.index("// ---- host side")]


def test_every_wait_has_a_limit_and_a_word_of_its_own():
    waits = re.findall(r"if \((?:use > 0 && )?!warp_wait\([^\n]*\)\) \{\s*if \(lane == 0\)\s*atomicCAS\(p\.status, 0u, (0x4\w\wu)\);", KERNEL)
    assert len(waits) == KERNEL.count("warp_wait(") == 5 and len(set(waits)) == 5
    assert "mbar_try_wait" not in KERNEL and "kBadOffsets = 0x401u" in SOURCE and "0x401u" not in waits


def test_loads_have_landed_before_the_end():
    end = KERNEL.rindex("__syncthreads()")
    assert KERNEL.index("ring_settled(sh->full, kGroupedStages, issued)") < end
    # a tail's loads land on a barrier of the CTA's own, which the warp that writes zeros waits for
    assert KERNEL.count("&sh->tail[s]") >= 5 and KERNEL.index("warp_wait(&sh->tail[s]") < end


def test_pairs_do_not_wait_for_one_another():
    """Sums of several pairs are finished by the one that comes last: it is told so by the counter, in a loop that only another pair's
    progress can prolong."""
    loops = re.findall(r"while \(true\)", SOURCE)
    assert len(loops) == 1
    body = SOURCE[SOURCE.index("add_blocks(unsigned long long *done"):]
    body = body[:body.index("\n}\n")]
    assert "while (true)" in body and "atomicCAS(done, old" in body and "if (seen == old)" in body
