"""Arguments at the edge of what the 8-bit checkpoint, layer norm and 8-bit GEMM entry points take, as
far as that needs no GPU (the addresses are made up and never read)."""
import os
import re

import pytest

import actrain as A

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20


@pytest.mark.parametrize("over", [dict(limit=0), dict(limit=10 ** 11), dict(src=0), dict(src=P + 8), dict(dst=0),
                                  dict(status=0), dict(status=P + 2)], ids=str)
def test_copy_wait_probe_refuses(over):
    a = dict(src=P, dst=P, limit=1000, status=P)
    a.update(over)
    with pytest.raises(A.ActError) as err:
        A.copy_wait_probe(a["src"], a["dst"], a["limit"], a["status"])
    assert err.value.code == A.ACT_ERR_INVALID


def test_copy_wait_probe_constants_match_the_header():
    text = open(os.path.join(ROOT, "include", "actrain.h")).read()
    value = dict(re.findall(r"#define ACT_(COPY_PROBE_\w+) (\d+)", text))
    assert value == dict(COPY_PROBE_BYTES=str(A.COPY_PROBE_BYTES), COPY_PROBE_CODE=str(A.COPY_PROBE_CODE))
    inside = open(os.path.join(ROOT, "audiocraft.cpp_b200", "csrc", "kernels.h")).read()
    assert f"COPY_PROBE_CODE = {A.COPY_PROBE_CODE}, COPY_PROBE_BYTES = {A.COPY_PROBE_BYTES};" in inside
