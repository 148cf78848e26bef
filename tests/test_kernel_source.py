"""Rules of the CUDA sources that no compiler and no passing run can show: read on the CPU."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "audiocraft.cpp_b200", "csrc")
# instructions after which memory that others wrote is read
WAITS = ("cp.async.wait_group", "cp.async.wait_all", "cp.async.bulk.wait_group", "mbarrier.try_wait", "mbarrier.test_wait",
         "bar.sync", "barrier.cluster.wait", "griddepcontrol.wait", "tcgen05.wait::ld", "ld.acquire")


def statements(text):
    """Every asm statement of a source: its text from `asm` to the closing parenthesis."""
    for m in re.finditer(r"\basm\b\s*(volatile)?\s*\(", text):
        depth, i, quoted = 1, m.end(), False
        while depth:
            c = text[i]
            if c == "\\":
                i += 1
            elif c == '"':
                quoted = not quoted
            elif not quoted:
                depth += (c == "(") - (c == ")")
            i += 1
        yield text[m.start():i]


FILES = sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")))


@pytest.mark.parametrize("name", FILES)
def test_waits_order_memory_for_the_compiler(name):
    # without the clobber the compiler may move plain loads of what arrived above the wait
    text = open(os.path.join(CSRC, name)).read()
    for s in statements(text):
        if any(w in s for w in WAITS):
            assert "volatile" in s and '"memory"' in s, " ".join(s.split())


@pytest.mark.parametrize("name", ["gemm_f8.cu", "rank_ckpt8.cu"])
def test_products_drain_their_copies_and_mmas_on_every_path(name):
    # a role whose own waits all held still has copies or MMAs in flight if the role after it gave up
    text = open(os.path.join(CSRC, name)).read()
    for call in ("drain_ring(", "drain_mma("):
        at = text.index(call)
        before = text[:at].rstrip()
        assert before.endswith("}") and text.count(call) == 1, "not the unconditional end of its role's loop"
