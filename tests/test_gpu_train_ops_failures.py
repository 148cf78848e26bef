"""The products' bounded waits and their status word, and what a call does after one ran out."""
import numpy as np
import pytest
import torch

import actrain as A
import eight_bit as E
from test_gpu_train_ops import U, Eight, Mat, assert_close, operands, out_mat, product, status_word, stream

pytestmark = pytest.mark.gpu


def test_a_wait_that_runs_out_sets_the_status_and_lets_its_copies_land():
    src = torch.randint(0, 256, (A.COPY_PROBE_BYTES,), dtype=torch.uint8, device="cuda")
    dst, st = torch.zeros_like(src), status_word()
    A.copy_wait_probe(src.data_ptr(), dst.data_ptr(), 5000, st.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    assert st.item() == A.COPY_PROBE_CODE and torch.equal(src, dst)
    # the first code stays
    st.fill_(41)
    A.copy_wait_probe(src.data_ptr(), dst.data_ptr(), 5000, st.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    assert st.item() == 41


@pytest.mark.parametrize("M,N,K", [(200, 300, 400), (130, 256, 6144), (2500, 1300, 520)])
def test_products_end_with_a_status_already_set_and_are_right_with_a_fresh_one(M, N, K):
    rng = np.random.default_rng(M)
    x, w = operands(rng, M, N, K, False)
    y, u, c = out_mat(M, N, "f32"), Mat(rng.standard_normal((M, 24)), "f32"), out_mat(24, K, "f32")
    for code in (31, 0):
        st = status_word()
        st.fill_(code)
        A.gemm_f8(x.v, w.v, M, N, K, y.ptr, A.TYPE_F32, st.data_ptr(), stream=stream())
        A.rank_gemm_ckpt8(u.ptr, A.TYPE_F32, 24, x.v, M, K, c.ptr, st.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        assert st.item() == code
    want, size = product(x, w, False)
    # K (M) products summed in any order, twice that for truncating adds
    assert_close(y.np(), want, (2 * K + 6) * U * size, "y")
    assert_close(c.np(), u.np().T @ x.np(), (2 * M + 4) * U * (np.abs(u.np()).T @ np.abs(x.np())) + 2.0 ** -140, "c")
