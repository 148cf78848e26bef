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


# ------------------------------------------------------------------------------ tensors without rows
# An empty tensor of torch has the address 0: where there are no rows, arguments with rows may be NULL.
def empty8(**over):
    v = dict(type=A.CKPT_E4M3, q=0, ldq=64, scale=0, lds=0)
    v.update(over)
    return A.ckpt8(**v)


NO_ROWS = {
    "store": lambda: A.ckpt8_store(0, A.TYPE_F32, 0, 64, empty8()),
    "store_square": lambda: A.ckpt8_store(0, A.TYPE_BF16, 0, 64, empty8(), block_rows=128),
    "load": lambda: A.ckpt8_load(empty8(), 0, 64, 0, A.TYPE_F16),
    "layernorm_fwd": lambda: A.layernorm_fwd(0, A.TYPE_F32, 0, 64, P, P, 0, A.TYPE_F16, 0, 0),
    "layernorm_fwd_8": lambda: A.layernorm_fwd(0, A.TYPE_F32, 0, 64, P, P, 0, A.TYPE_F16, 0, 0, y8=empty8(), x8=empty8()),
    "layernorm_bwd": lambda: A.layernorm_bwd(0, A.TYPE_F32, 0, A.TYPE_F32, P, 0, 0, 0, 64, 0, A.TYPE_F32, P, P, P, 1 << 24,
                                             accumulate=True),
    "layernorm_bwd_8": lambda: A.layernorm_bwd(0, A.TYPE_F32, 0, A.TYPE_F32, P, 0, 0, 0, 64, 0, A.TYPE_F32, 0, 0, P, 1 << 24,
                                               x8=empty8()),
    "gelu_fwd": lambda: A.gelu_ckpt8_fwd(0, A.TYPE_F16, 0, 64, 0, A.TYPE_F16, empty8()),
    "gelu_fwd_8": lambda: A.gelu_ckpt8_fwd(0, A.TYPE_F16, 0, 64, 0, A.TYPE_F16, empty8(), g8=empty8()),
    "gelu_bwd": lambda: A.gelu_ckpt8_bwd(0, A.TYPE_F16, empty8(), 0, 64, 0, A.TYPE_F16),
    "gelu_bwd_8": lambda: A.gelu_ckpt8_bwd(0, A.TYPE_F16, empty8(), 0, 64, 0, A.TYPE_F16, dz8=empty8()),
    "rank": lambda: A.rank_gemm_ckpt8(0, A.TYPE_F16, 16, empty8(), 0, 64, P, P, accumulate=True),
    "gemm": lambda: A.gemm_f8(empty8(), A.ckpt8(A.CKPT_E4M3, P, 64, P, 1), 0, 64, 64, 0, A.TYPE_F16, P),
}


@pytest.mark.parametrize("name", NO_ROWS)
def test_empty_tensors_are_no_work(name):
    NO_ROWS[name]()


def test_other_checks_hold_without_rows():
    w8 = A.ckpt8(A.CKPT_E4M3, P, 64, P, 1)
    for call in (lambda: A.ckpt8_store(0, A.TYPE_F32, 0, 64, None),
                 lambda: A.ckpt8_store(0, A.TYPE_F32, 0, 64, empty8(type=5)),
                 lambda: A.ckpt8_store(2, A.TYPE_F32, 0, 64, empty8()),
                 lambda: A.ckpt8_store(0, A.TYPE_F32, 0, 64, empty8(ldq=63)),
                 lambda: A.ckpt8_load(empty8(), 0, 64, 0, A.TYPE_Q8_0),
                 lambda: A.layernorm_fwd(0, A.TYPE_F32, 0, 64, P + 1, P, 0, A.TYPE_F16, 0, 0),
                 lambda: A.layernorm_fwd(0, A.TYPE_F32, 0, 9000, P, P, 0, A.TYPE_F16, 0, 0),
                 lambda: A.layernorm_bwd(0, A.TYPE_F32, P, A.TYPE_F32, P, 0, 0, 0, 64, 0, A.TYPE_F32, P, P, P, 1 << 24,
                                         x8=empty8()),
                 lambda: A.layernorm_bwd(0, A.TYPE_F32, 0, A.TYPE_F32, P, 0, 0, 0, 64, 0, A.TYPE_F32, P, P, 0, 1 << 24),
                 lambda: A.gelu_ckpt8_fwd(0, A.TYPE_F16, 0, 64, 0, A.TYPE_F16, None),
                 lambda: A.rank_gemm_ckpt8(0, A.TYPE_F16, 65, empty8(), 0, 64, P, P),
                 lambda: A.rank_gemm_ckpt8(0, A.TYPE_F16, 16, empty8(), 0, 64, 0, P),
                 lambda: A.gemm_f8(empty8(), w8, 0, 64, 64, 0, A.TYPE_F16, 0),
                 lambda: A.gemm_f8(empty8(), empty8(lds=1), 0, 64, 64, 0, A.TYPE_F16, P),
                 lambda: A.gemm_f8(empty8(), w8, 0, 64, 64, 0, A.TYPE_F16, P, bias=P + 2)):
        with pytest.raises(A.ActError) as err:
            call()
        assert err.value.code == A.ACT_ERR_INVALID
