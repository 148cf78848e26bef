"""Refusals of the 8-bit checkpoint, layer norm and 8-bit GEMM entry points: every bad argument is
reported before any device work, so none of this needs a GPU (the addresses are made up)."""
import numpy as np
import pytest
import torch

import actrain as A
import eight_bit as E

P = 1 << 20  # an aligned address that is never read


def view(**over):
    v = dict(type=A.CKPT_E4M3, q=P, ldq=64, scale=P, lds=8)
    v.update(over)
    return A.ckpt8(**v)


def store(**o):
    a = dict(x=P, x_type=A.TYPE_F32, rows=8, cols=64, out=view())
    a.update(o)
    A.ckpt8_store(**a)


def load(**o):
    a = dict(src=view(), rows=8, cols=64, y=P, y_type=A.TYPE_F32)
    a.update(o)
    A.ckpt8_load(**a)


def ln_fwd(**o):
    a = dict(x=P, x_type=A.TYPE_F32, rows=8, dim=64, w=P, b=P, y=P, y_type=A.TYPE_F16, mean=P, rstd=P)
    a.update(o)
    A.layernorm_fwd(**a)


def ln_bwd(**o):
    a = dict(dy=P, dy_type=A.TYPE_F32, x=P, x_type=A.TYPE_F32, w=P, mean=P, rstd=P, rows=8, dim=64, dx=P,
             dx_type=A.TYPE_F32, dw=P, db=P, workspace=P, workspace_bytes=1 << 24)
    a.update(o)
    A.layernorm_bwd(**a)


def gelu_fwd(**o):
    a = dict(z=P, z_type=A.TYPE_F16, rows=8, cols=64, g=P, g_type=A.TYPE_F16, z8=view())
    a.update(o)
    A.gelu_ckpt8_fwd(**a)


def gelu_bwd(**o):
    a = dict(dg=P, dg_type=A.TYPE_F16, z8=view(), rows=8, cols=64, dz=P, dz_type=A.TYPE_F16)
    a.update(o)
    A.gelu_ckpt8_bwd(**a)


def rank(**o):
    a = dict(u=P, u_type=A.TYPE_F16, nb=16, x8=view(), rows=8, cols=64, c=P, status=P)
    a.update(o)
    A.rank_gemm_ckpt8(**a)


def gemm(**o):
    a = dict(x8=view(), w8=view(lds=1), M=8, N=64, K=64, y=P, y_type=A.TYPE_F16, status=P)
    a.update(o)
    A.gemm_f8(**a)


BAD = [
    (store, dict(x=0)), (store, dict(x=P + 2)), (store, dict(x_type=A.TYPE_Q8_0)), (store, dict(rows=-1)),
    (store, dict(cols=0, ldx=8)), (store, dict(ldx=63)), (store, dict(block_rows=64)), (store, dict(out=None)),
    (store, dict(out=view(q=0))), (store, dict(out=view(scale=0))), (store, dict(out=view(scale=P + 2))),
    (store, dict(out=view(ldq=63))), (store, dict(out=view(lds=7))), (store, dict(out=view(type=0))),
    (store, dict(out=view(type=3))), (store, dict(rows=1 << 31, out=view(lds=1 << 31))),
    (load, dict(y=0)), (load, dict(y=P + 1, y_type=A.TYPE_F16)), (load, dict(src=None)), (load, dict(ldy=63)),
    (load, dict(src=view(lds=7))), (load, dict(block_rows=2)),
    (ln_fwd, dict(x=0)), (ln_fwd, dict(dim=0, ldx=8, ldy=8)), (ln_fwd, dict(dim=8193)), (ln_fwd, dict(eps=-1.0)),
    (ln_fwd, dict(eps=float("nan"))), (ln_fwd, dict(eps=float("inf"))), (ln_fwd, dict(y=0)), (ln_fwd, dict(mean=0)),
    (ln_fwd, dict(rstd=0)), (ln_fwd, dict(w=P + 1)), (ln_fwd, dict(b=P + 2)), (ln_fwd, dict(ldx=63)),
    (ln_fwd, dict(ldy=63)), (ln_fwd, dict(y8=view(ldq=63))), (ln_fwd, dict(x8=view(lds=7))),
    (ln_fwd, dict(y_type=A.TYPE_Q8_0)), (ln_fwd, dict(rows=-1)),
    (ln_bwd, dict(x=0)), (ln_bwd, dict(x8=view())), (ln_bwd, dict(dy=0)), (ln_bwd, dict(dx=0)),
    (ln_bwd, dict(workspace=0)), (ln_bwd, dict(workspace=P + 8)), (ln_bwd, dict(workspace_bytes=0)),
    (ln_bwd, dict(accumulate=2)), (ln_bwd, dict(dim=9000)), (ln_bwd, dict(lddx=63)), (ln_bwd, dict(add=P + 2)),
    (ln_bwd, dict(dw=P + 2)), (ln_bwd, dict(db=P + 2)), (ln_bwd, dict(mean=0)), (ln_bwd, dict(rstd=0)),
    (ln_bwd, dict(dx_type=7)), (ln_bwd, dict(x=0, x8=view(lds=7))),
    (gelu_fwd, dict(z=0)), (gelu_fwd, dict(g=0)), (gelu_fwd, dict(z8=None)), (gelu_fwd, dict(g8=view(ldq=1))),
    (gelu_fwd, dict(g_type=A.TYPE_F32)), (gelu_fwd, dict(cols=0, ldz=4, ldg=4)),
    (gelu_bwd, dict(dg=0)), (gelu_bwd, dict(dz=0)), (gelu_bwd, dict(z8=None)), (gelu_bwd, dict(dz8=view(lds=1))),
    (gelu_bwd, dict(dz_type=A.TYPE_F32)), (gelu_bwd, dict(lddz=63)),
    (rank, dict(nb=0)), (rank, dict(nb=65)), (rank, dict(u=0)), (rank, dict(x8=None)), (rank, dict(c=0)),
    (rank, dict(c=P + 2)), (rank, dict(status=0)), (rank, dict(status=P + 2)), (rank, dict(ldu=15)),
    (rank, dict(ldc=63)), (rank, dict(x8=view(q=P + 8))), (rank, dict(x8=view(ldq=72))), (rank, dict(cols=0, ldc=1)),
    (rank, dict(accumulate=3)), (rank, dict(x8=view(lds=7))),
    (gemm, dict(x8=None)), (gemm, dict(w8=None)), (gemm, dict(x8=view(type=A.CKPT_I8))),
    (gemm, dict(w8=view(type=A.CKPT_I8))), (gemm, dict(K=0)), (gemm, dict(N=0, ldy=1)), (gemm, dict(M=-1)),
    (gemm, dict(y=0)), (gemm, dict(y=P + 1)), (gemm, dict(status=0)), (gemm, dict(bias=P + 2)), (gemm, dict(ldy=63)),
    (gemm, dict(x8=view(q=P + 4))), (gemm, dict(w8=view(ldq=72))), (gemm, dict(w8=view(lds=0))),
    (gemm, dict(w8=view(ldq=48))), (gemm, dict(N=129, w8=view(lds=1))), (gemm, dict(w_mn_major=2)),
    (gemm, dict(accumulate=-1)), (gemm, dict(y_type=A.TYPE_Q8_0)), (gemm, dict(x8=view(lds=7))),
]


@pytest.mark.parametrize("call,over", BAD, ids=[f"{c.__name__}-{'-'.join(map(str, o))}-{i}"
                                                for i, (c, o) in enumerate(BAD)])
def test_bad_arguments_are_refused(call, over):
    with pytest.raises(A.ActError) as err:
        call(**over)
    assert err.value.code == A.ACT_ERR_INVALID
    assert "act_" in str(err.value) or "_ckpt8_" in str(err.value)


@pytest.mark.parametrize("call,over", [(store, {}), (load, {}), (ln_fwd, {}), (ln_bwd, dict(dw=0, db=0)),
                                       (gelu_fwd, {}), (gelu_bwd, {}), (rank, dict(accumulate=True))],
                         ids=["store", "load", "ln_fwd", "ln_bwd", "gelu_fwd", "gelu_bwd", "rank"])
def test_no_rows_is_no_work(call, over):
    call(rows=0, **over)


def test_no_rows_is_no_work_for_the_gemm():
    gemm(M=0)


def test_workspace_query():
    assert A.layernorm_bwd_workspace(8, 64) >= 2 * 64 * 4
    for rows, dim in ((-1, 64), (8, 0), (8, 8193)):
        with pytest.raises(A.ActError):
            A.layernorm_bwd_workspace(rows, dim)


def test_struct_layout_matches_c(tmp_path):
    import ctypes
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "layout.c"
    fields = [f for f, _ in A.Ckpt8._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "actrain.h"\nint main(void){printf("%zu", '
                   'sizeof(act_ckpt8));\n' +
                   "".join(f'printf(" %zu", offsetof(act_ckpt8, {f}));\n' for f in fields) + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I" + os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(A.Ckpt8)] + [getattr(A.Ckpt8, f).offset for f in fields]


def test_plain_e4m3_codes_match_torch():
    # the oracle's own rounding and decoding, against an independent implementation of the format
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((64, 128)) * np.exp2(rng.integers(-14, 9, (64, 128)))).clip(-448, 448)
    x[0, 0] = 448.0  # every block's scale stays at most 1: divide it out
    q, s = E.encode(x, A.CKPT_E4M3)
    v = torch.from_numpy(x / E.spread(s, x.shape)).float()
    want = v.to(torch.float8_e4m3fn)
    exact = (v.double().numpy() == x / E.spread(s, x.shape))  # fp32 holds most of them
    got = want.view(torch.uint8).numpy()
    np.testing.assert_array_equal(q[exact], got[exact])
    np.testing.assert_array_equal(E.decode(q, np.ones_like(s), A.CKPT_E4M3)[exact], want.double().numpy()[exact])
