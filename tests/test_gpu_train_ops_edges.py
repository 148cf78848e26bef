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


def nearest_kept(x, kind, block=1):
    """Codes and scales of the definition, and what they stand for; finite values are limited first to the
    largest that a code and a scale stand for in fp32 (the next code would be 2^128)."""
    limit = 127 * 2.0 ** 121 if kind == A.CKPT_I8 else 240 * 2.0 ** 120
    x = np.where(np.isfinite(x), np.clip(x, -limit, limit), x)
    q, s = E.encode(x, kind, block)
    return q, s, E.decode(q, s, kind, block)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("kind", [A.CKPT_I8, A.CKPT_E4M3], ids=["i8", "e4m3"])
@pytest.mark.parametrize("layout", [(0, 0), (3, 1)], ids=["dense", "odd"])
def test_the_largest_finite_values_stay_finite(t, kind, layout):
    # a mask of the type's lowest value in an activation: its checkpoint is finite, and so are the gradients
    rng = np.random.default_rng(3)
    pad, off = layout
    big = torch.finfo(torch.float32 if t == "f32" else torch.bfloat16).max
    X = rng.standard_normal((9, 300))
    X[0, :40], X[1, 40:90], X[2, ::3], X[3, 7] = big, -big, -big, 0.99 * big
    X[4, :], X[5, :4], X[6, 130] = -big, [big, np.inf, np.nan, -big], 0.8 * big
    X[7, 200:204] = 0.9375 * 2.0 ** 128, 0.96875 * 2.0 ** 128, 0.984375 * 2.0 ** 128, 0.9921875 * 2.0 ** 128
    z = Mat(X, t, pad, off)
    for block in (1, 128):
        e, y = Eight(9, 300, kind, block, pad, off), out_mat(9, 300, "f32", pad, off)
        A.ckpt8_store(z.ptr, E.KINDS[t], 9, 300, e.v, block_rows=block, ldx=z.ld, stream=stream())
        A.ckpt8_load(e.v, 9, 300, y.ptr, A.TYPE_F32, block_rows=block, ldy=y.ld, stream=stream())
        torch.cuda.synchronize()
        q, s, v = nearest_kept(z.np(), kind, block)
        np.testing.assert_array_equal(e.codes().cpu().numpy(), q)
        np.testing.assert_array_equal(e.scales(), s)
        np.testing.assert_array_equal(y.np(), v)
        assert np.array_equal(np.isfinite(y.np()), np.isfinite(z.np()))
    q, s, v = nearest_kept(z.np(), kind)
    # the norm's checkpoint of the same rows, and of rows of one column (whose variance is 0)
    st, x8, y8 = Mat(np.zeros((2, 9)), "f32"), Eight(9, 300, kind, 1, pad, off), out_mat(9, 300, "f32")
    A.layernorm_fwd(z.ptr, E.KINDS[t], 9, 300, 0, 0, y8.ptr, A.TYPE_F32, st.ptr, st.ptr + 4 * st.ld, ldx=z.ld, x8=x8.v,
                    stream=stream())
    torch.cuda.synchronize()
    np.testing.assert_array_equal(x8.codes().cpu().numpy(), q)
    np.testing.assert_array_equal(x8.scales(), s)
    one = Mat(np.array([[big], [-big], [0.5], [0.9 * big]]), t)
    st, x8, y = Mat(np.zeros((2, 4)), "f32"), Eight(4, 1, kind), out_mat(4, 1, "f32")
    A.layernorm_fwd(one.ptr, E.KINDS[t], 4, 1, 0, 0, y.ptr, A.TYPE_F32, st.ptr, st.ptr + 4 * st.ld, x8=x8.v,
                    stream=stream())
    torch.cuda.synchronize()
    np.testing.assert_array_equal(x8.np(), nearest_kept(one.np(), kind)[2])
    # GELU there and back: its own 8-bit result too; the gradient at the kept values is 1 or 0 out there
    z8, g8, g, dz = Eight(9, 300, kind, 1, pad, off), Eight(9, 300, kind, 1, pad, off), out_mat(9, 300, "f32"), \
        out_mat(9, 300, t, pad, off)
    ones = Mat(np.ones((9, 300)), t, pad, off)
    A.gelu_ckpt8_fwd(z.ptr, E.KINDS[t], 9, 300, 0, E.KINDS[t], z8.v, g8=g8.v, ldz=z.ld, stream=stream())
    A.ckpt8_load(g8.v, 9, 300, g.ptr, A.TYPE_F32, stream=stream())
    A.gelu_ckpt8_bwd(ones.ptr, E.KINDS[t], z8.v, 9, 300, dz.ptr, E.KINDS[t], lddg=ones.ld, lddz=dz.ld, stream=stream())
    torch.cuda.synchronize()
    np.testing.assert_array_equal(z8.codes().cpu().numpy(), q)
    far = np.abs(z.np()) > 1e30
    right = np.isfinite(z.np())
    np.testing.assert_array_equal(dz.np()[far & right], (z.np() > 0)[far & right].astype(float))
    np.testing.assert_array_equal(np.isfinite(dz.np()), np.isfinite(v))
    up = far & right & (z.np() > 0)
    assert np.all(np.isfinite(g.np()[up])) and np.all(np.abs(g.np()[up] / z.np()[up] - 1) <= 2.0 ** -4)
