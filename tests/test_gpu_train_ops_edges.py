"""The 8-bit checkpoint, layer norm and product operators at the edge of what they take, against their
definitions in 64 bits (tests/eight_bit.py)."""
import numpy as np
import pytest
import torch

import actrain as A
import eight_bit as E
from test_gpu_train_ops import U, Eight, Mat, assert_close, out_mat, status_word, stream

pytestmark = pytest.mark.gpu


def test_empty_tensors_zero_the_sums_over_their_rows():
    x, st = torch.empty(0, 64, device="cuda"), status_word()
    assert x.data_ptr() == 0
    w, sums, c = torch.ones(64, device="cuda"), torch.full((2, 64), 5.0, device="cuda"), out_mat(16, 64, "f32", 3)
    x8 = A.ckpt8(A.CKPT_I8, 0, 64, 0, 0)
    room = A.layernorm_bwd_workspace(0, 64)
    space = torch.empty(room // 4, device="cuda")
    for keep in (True, False):
        for kept in (None, x8):
            A.layernorm_bwd(0, A.TYPE_F32, 0, A.TYPE_F32, w.data_ptr(), 0, 0, 0, 64, 0, A.TYPE_F32, sums[0].data_ptr(),
                            sums[1].data_ptr(), space.data_ptr(), room, accumulate=keep, x8=kept, stream=stream())
            A.rank_gemm_ckpt8(0, A.TYPE_F32, 16, x8, 0, 64, c.ptr, st.data_ptr(), accumulate=keep, ldc=c.ld,
                              stream=stream())
            torch.cuda.synchronize()
            assert bool((sums == (5.0 if keep else 0.0)).all())
            assert np.all(c.np() == (3.0 if keep else 0.0)) and c.untouched() and st.item() == 0


@pytest.mark.parametrize("rows,cols,nb", [(70, 300, 20), (200, 5000, 3)])
@pytest.mark.parametrize("ut", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", [A.CKPT_I8, A.CKPT_E4M3], ids=["i8", "e4m3"])
def test_infinite_u_gives_what_the_formula_gives(rows, cols, nb, ut, kind):
    # infinity times a value is an infinity of its sign, times 0 NaN; infinities of both signs add up to NaN
    rng = np.random.default_rng(rows + nb)
    X, V = rng.standard_normal((rows, cols)), rng.standard_normal((rows, nb))
    X[:, 5:9], X[:, 9] = 0.0, np.abs(X[:, 9])
    V[3, 0], V[69, 1], V[11, 2], V[12, 2] = np.inf, -np.inf, np.inf, np.nan
    if nb > 3:
        V[20, 3], V[21, 3], V[22, 19], V[23, 19] = np.inf, -np.inf, np.inf, np.inf
    q, s = E.encode(X, kind)
    x = Eight(rows, cols, kind, 1, -cols % 16, data=(q, s))
    for pad, off in ((0, 0), (3, 1)):
        u, c, st = Mat(V, ut, pad, off), out_mat(nb, cols, "f32"), status_word()
        A.rank_gemm_ckpt8(u.ptr, E.KINDS[ut], nb, x.v, rows, cols, c.ptr, st.data_ptr(), alpha=0.5, ldu=u.ld,
                          stream=stream())
        torch.cuda.synchronize()
        K, V_, got = E.decode(q, s, kind), u.np(), c.np()
        finite = np.isfinite(V_).all(0)
        with np.errstate(invalid="ignore"):
            want = 0.5 * np.stack([(V_[:, j, None] * K).sum(0) for j in range(nb)])
        np.testing.assert_array_equal(got[~finite], want[~finite])
        size = 0.5 * (np.abs(V_[:, finite]).T @ np.abs(K))
        # rows terms in any order, twice that for truncating adds; the product with alpha
        assert_close(got[finite], want[finite], (2 * rows + 4) * U * size + 2.0 ** -140, "c")
        assert st.item() == 0
