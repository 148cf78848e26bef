"""The 8-bit checkpoint, layer norm and product operators at the edge of what they take, against their
definitions in 64 bits (tests/eight_bit.py)."""
import numpy as np
import pytest
import torch

import actrain as A
import eight_bit as E
from test_gpu_train_ops import Eight, Mat, out_mat, status_word, stream

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
