"""Layer norm with weight gradients, 8-bit checkpoints, GELU and rank product that read them, and
the 8-bit GEMM, against their definitions in 64 bits (tests/eight_bit.py).

Tolerances are counted, not fitted.  u = 2^-24 is half a step of fp32; a result rounded to a type
may move by half that type's step (eight_bit.rounding).  A sum of n terms in any order is off by
at most n u times the sum of the terms' sizes; twice that where the tensor cores truncate.
"""
import numpy as np
import pytest
import torch

import actrain as A
import eight_bit as E

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ALL = ["f32", "f16", "bf16"]


def stream():
    return torch.cuda.current_stream().cuda_stream


class Mat:
    """A matrix on the GPU with a row stride, a start that is `off` elements past an aligned address,
    and a filling around it that must survive."""

    def __init__(self, x, kind, pad=0, off=0, fill=7.0):
        x = np.asarray(x, np.float64)
        self.rows, self.cols, self.kind = x.shape[0], x.shape[1], kind
        self.ld = self.cols + pad
        self.buf = torch.full((off + self.rows * self.ld + 64,), fill, dtype=TORCH[kind], device="cuda")
        self.fill, self.off = self.buf[0].clone() if self.buf.numel() else None, off
        self.view = self.buf[off:off + self.rows * self.ld].view(self.rows, self.ld)[:, :self.cols]
        self.view.copy_(torch.from_numpy(x).to("cuda").to(TORCH[kind]))
        self.ptr = self.buf.data_ptr() + off * self.buf.element_size()

    def np(self):
        return self.view.double().cpu().numpy()

    def untouched(self):
        mask = torch.ones_like(self.buf, dtype=torch.bool)
        mask[self.off:self.off + self.rows * self.ld].view(self.rows, self.ld)[:, :self.cols] = False
        return bool((self.buf[mask] == self.fill).all())


def out_mat(rows, cols, kind, pad=0, off=0):
    return Mat(np.full((rows, cols), 3.0), kind, pad, off)


class Eight:
    """An 8-bit tensor on the GPU; codes start as NaN."""

    def __init__(self, rows, cols, kind, block=1, pad=0, off=0, extra=0, data=None):
        self.rows, self.cols, self.kind, self.block = rows, cols, kind, block
        self.ldq, self.off = cols + pad, off
        self.lds = -(-rows // block) + extra
        self.nan = 127 if kind == A.CKPT_E4M3 else 128
        self.q = torch.full((off + rows * self.ldq + 64,), self.nan, dtype=torch.uint8, device="cuda")
        self.scale = torch.full((-(-cols // 128), self.lds), float("nan"), device="cuda")
        if data is not None:
            q, s = data
            self.codes().copy_(torch.from_numpy(q))
            self.scale[:, :s.shape[1]] = torch.from_numpy(s.astype(np.float32)).to("cuda")
        self.v = A.ckpt8(kind, self.q.data_ptr() + off, self.ldq, self.scale.data_ptr(), self.lds)

    def codes(self):
        return self.q[self.off:self.off + self.rows * self.ldq].view(self.rows, self.ldq)[:, :self.cols]

    def scales(self):
        return self.scale[:, :-(-self.rows // self.block)].double().cpu().numpy()

    def np(self):
        return E.decode(self.codes().cpu().numpy().copy(), self.scales(), self.kind, self.block)

    def untouched(self):
        mask = torch.ones_like(self.q, dtype=torch.bool)
        mask[self.off:self.off + self.rows * self.ldq].view(self.rows, self.ldq)[:, :self.cols] = False
        used = -(-self.rows // self.block)
        return bool((self.q[mask] == self.nan).all()) and bool(torch.isnan(self.scale[:, used:]).all())


def up16(n):
    return -n % 16


def assert_close(got, want, allowed, what=""):
    assert got.shape == want.shape
    with np.errstate(invalid="ignore"):
        off = np.abs(got - want) - allowed
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    worst = np.nanmax(off) if np.any(~np.isnan(off)) else -1.0  # nothing, or NaN in both throughout
    assert worst <= 0, f"{what}: {np.nansum(off > 0)} of {off.size} off, by up to {worst:.3g} more than allowed"


def rounded(x, kind):
    return torch.from_numpy(np.asarray(x, np.float64)).to(TORCH[kind]).double().numpy()


def wild(rng, rows, cols):
    """Rows of very different sizes, some zero blocks."""
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-12, 12, (rows, 1)))
    x[rng.random((rows, cols)) < 0.02] *= 40
    if rows > 2 and cols > 130:
        x[2, :128] = 0
    return x


# ------------------------------------------------------------------------------ store and load
SHAPES = [(1, 1), (1, 128), (3, 129), (5, 127), (130, 257), (257, 1000), (4, 4096), (1000, 4)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("kind", [A.CKPT_I8, A.CKPT_E4M3], ids=["i8", "e4m3"])
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("layout", [(0, 0), (3, 1), (4, 8)], ids=["dense", "odd", "strided"])
def test_store_and_load_are_exact(rows, cols, kind, block, layout):
    rng = np.random.default_rng(rows * 31 + cols)
    pad, off = layout
    for t in ALL:
        x = Mat(wild(rng, rows, cols), t, pad, off)
        e = Eight(rows, cols, kind, block, pad, off, extra=2)
        A.ckpt8_store(x.ptr, E.KINDS[t], rows, cols, e.v, block_rows=block, ldx=x.ld, stream=stream())
        torch.cuda.synchronize()
        q, s = E.encode(x.np(), kind, block)
        np.testing.assert_array_equal(e.scales(), s)
        np.testing.assert_array_equal(e.codes().cpu().numpy(), q)
        assert e.untouched()
        want = E.decode(q, s, kind, block)
        for u in ALL:
            y = out_mat(rows, cols, u, pad, off)
            A.ckpt8_load(e.v, rows, cols, y.ptr, E.KINDS[u], block_rows=block, ldy=y.ld, stream=stream())
            torch.cuda.synchronize()
            np.testing.assert_array_equal(y.np(), rounded(want, u))
            assert y.untouched()


@pytest.mark.parametrize("kind", [A.CKPT_I8, A.CKPT_E4M3], ids=["i8", "e4m3"])
@pytest.mark.parametrize("block", [1, 128])
def test_store_of_special_values(kind, block):
    top = E.TOP[kind]
    x = np.zeros((9, 300))
    x[0, :] = np.linspace(-1, 1, 300) * top                  # the largest value is exactly top: s = 1
    x[1, :] = np.nextafter(np.float32(top), np.float32(1e9))  # one step past it: s = 2
    x[2, 5], x[2, 130] = np.inf, -np.inf                      # stored as NaN, the rest of the block as ever
    x[2, 6], x[2, 131], x[2, 299] = 3.0, 1e-3, np.nan
    x[3, :] = 2.0 ** -140                                     # subnormal: s = 2^-126
    x[4, :3] = 3e38, -3e38, 1.0
    x[5, :] = np.nan                                          # nothing finite: s = 2^-126
    x[6, ::2] = -0.0
    x[7, :] = (np.arange(300) - 150 + 0.5) * top / 127        # halves: ties to even in I8
    x[8, 7] = 1e-38
    m = Mat(x, "f32")
    e = Eight(9, 300, kind, block)
    A.ckpt8_store(m.ptr, A.TYPE_F32, 9, 300, e.v, block_rows=block, stream=stream())
    torch.cuda.synchronize()
    q, s = E.encode(m.np(), kind, block)
    np.testing.assert_array_equal(e.scales(), s)
    got = e.codes().cpu().numpy()
    if kind == A.CKPT_E4M3:  # the sign of a code that stands for 0 follows x; of NaN it is free
        got = np.where((got & 127) == 127, 127, got)
    np.testing.assert_array_equal(got, q)
    np.testing.assert_array_equal(e.np(), E.decode(q, s, kind, block))


# ------------------------------------------------------------------------------ layer norm
DIMS = [1, 2, 3, 100, 127, 128, 129, 256, 257, 512, 513, 1000, 1024, 1025, 1536, 2047, 2049, 4096, 5000, 8192]


def check_codes(e, y, slack, what):
    """8 bits of a computed y, known to `slack`: either neighbour next to a border is right."""
    top, s = E.TOP[e.kind], E.spread(e.scales(), y.shape)
    half = s * 0.5 if e.kind == A.CKPT_I8 else np.maximum(np.abs(y) * 2.0 ** -4, s * 2.0 ** -10)
    assert_close(e.np(), y, half + 2 * slack, what)
    assert np.all(np.abs(y) <= top * s * (1 + 2.0 ** -20) + slack), what
    want = E.block_scales(y, e.kind)
    assert np.all((e.scales() == want) | (np.abs(np.log2(e.scales() / want)) <= 1)), what
    assert np.mean(e.scales() != want) < 0.02 or e.scales().size < 50, what


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("layout", [(0, 0), (5, 1), (4, 4)], ids=["dense", "odd", "strided"])
def test_layernorm_forward(dim, layout):
    rng = np.random.default_rng(dim)
    pad, off = layout
    rows, eps = 11, 1e-5
    for t, u in (("f32", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("f32", "f32"), ("f16", "bf16")):
        x = Mat(wild(rng, rows, dim) + rng.standard_normal((rows, 1)), t, pad, off)
        w, b = (Mat(1 + 0.3 * rng.standard_normal((1, dim)), "f32", 0, off),
                Mat(0.3 * rng.standard_normal((1, dim)), "f32", 0, off))
        y = out_mat(rows, dim, u, pad, off)
        st = Mat(np.zeros((2, rows)), "f32")
        kind = A.CKPT_I8 if t == "f32" else A.CKPT_E4M3
        y8, x8 = Eight(rows, dim, A.CKPT_E4M3, 1, pad, off, 1), Eight(rows, dim, kind, 1, pad, off, 3)
        bare = u == "f32" and t == "f32"
        A.layernorm_fwd(x.ptr, E.KINDS[t], rows, dim, 0 if bare else w.ptr, 0 if bare else b.ptr, y.ptr, E.KINDS[u],
                        st.ptr, st.ptr + 4 * st.ld, eps=eps, ldx=x.ld, ldy=y.ld, y8=y8.v, x8=x8.v, stream=stream())
        torch.cuda.synchronize()
        X = x.np()
        W, B = (np.ones((1, dim)), np.zeros((1, dim))) if bare else (w.np(), b.np())
        mean, rstd = E.norm_stats(X, eps)
        # sums of dim terms: 4 values of a lane, up to 8 blocks, 5 shuffles, 16 warps add up to at
        # most 40 roundings on any path; mean and each difference from it one more each
        size = np.abs(X).max(1)
        dmean = 42 * U * np.abs(X).mean(1)
        assert_close(st.np()[0], mean, dmean + U * np.abs(mean), "mean")
        # variance: 42 roundings of its own, each difference off by dmean + u |x - mean|
        spread = np.abs(X - mean[:, None]).mean(1)
        dvar = 46 * U * rstd ** -2 + 2 * dmean * spread + dmean ** 2 + 2 * U * size * spread
        drstd = 0.5 * rstd ** 3 * dvar * 1.01 + 4 * U * rstd + np.where(dvar > 0.1 * rstd ** -2, np.inf, 0)
        assert_close(st.np()[1], rstd, drstd, "rstd")
        h = (X - mean[:, None]) * rstd[:, None]
        Y = h * W + B
        dh = (dmean[:, None] + U * np.abs(X - mean[:, None])) * rstd[:, None] + \
            np.abs(X - mean[:, None]) * drstd[:, None] + 2 * U * np.abs(h)
        slack = dh * np.abs(W) + 2 * U * (np.abs(h * W) + np.abs(Y))
        assert_close(y.np(), Y, slack + E.rounding(u, np.abs(Y) + slack), f"y {t} {u}")
        q, s = E.encode(X, kind)
        np.testing.assert_array_equal(x8.codes().cpu().numpy(), q)
        np.testing.assert_array_equal(x8.scales(), s)
        if np.all(np.isfinite(slack)):
            check_codes(y8, Y, slack, "y8")
        assert y.untouched() and y8.untouched() and x8.untouched() and st.untouched()


def test_layernorm_forward_without_y_and_with_bad_rows():
    # a row with NaN or infinity spoils itself alone; y may be left out beside y8
    rng = np.random.default_rng(3)
    X = rng.standard_normal((6, 700))
    X[1, 3], X[4, 600] = np.nan, np.inf
    x = Mat(X, "f32")
    st, y8 = Mat(np.zeros((2, 6)), "f32"), Eight(6, 700, A.CKPT_E4M3)
    y = out_mat(6, 700, "f32")
    for out, t in ((0, 0), (y.ptr, A.TYPE_F32)):
        A.layernorm_fwd(x.ptr, A.TYPE_F32, 6, 700, 0, 0, out, t, st.ptr, st.ptr + 24, y8=y8.v, stream=stream())
    torch.cuda.synchronize()
    bad = np.array([False, True, False, False, True, False])
    assert np.isnan(y.np()[bad]).all() and np.isfinite(y.np()[~bad]).all()
    assert np.isnan(y8.np()[bad]).all() and np.isfinite(y8.np()[~bad]).all()


def backward(x, x8, dy, w, mean, rstd, dxk, add, acc, layout, want_sums=(True, True)):
    rows, dim = dy.rows, dy.cols
    pad, off = layout
    dx = out_mat(rows, dim, dxk, pad, off) if add is not True else Mat(0.5 * np.ones((rows, dim)), dxk, pad, off)
    addp = dx.ptr if add is True else 0
    sums = Mat(np.full((2, dim), 2.0), "f32")
    room = A.layernorm_bwd_workspace(rows, dim)
    space = torch.full((room // 4,), float("nan"), device="cuda")
    A.layernorm_bwd(dy.ptr, E.KINDS[dy.kind], 0 if x8 else x.ptr, E.KINDS[x.kind], w.ptr if w else 0, mean.ptr,
                    rstd.ptr, rows, dim, dx.ptr, E.KINDS[dxk], sums.ptr if want_sums[0] else 0,
                    sums.ptr + 4 * sums.ld if want_sums[1] else 0, space.data_ptr(), room, accumulate=acc, add=addp,
                    x8=x8.v if x8 else None, lddy=dy.ld, ldx=x.ld, lddx=dx.ld, stream=stream())
    torch.cuda.synchronize()
    assert dx.untouched() and sums.untouched()
    return dx.np(), sums.np()


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("layout", [(0, 0), (5, 1), (4, 4)], ids=["dense", "odd", "strided"])
def test_layernorm_backward(dim, layout):
    rng = np.random.default_rng(dim + 1)
    pad, off = layout
    for i, (t, u, v, kept) in enumerate([("f32", "f32", "f32", None), ("f16", "bf16", "f16", None),
                                         ("bf16", "bf16", "bf16", A.CKPT_I8), ("f32", "f16", "f32", A.CKPT_E4M3),
                                         ("f16", "f16", "bf16", None)]):
        rows = (1, 37, 300, 5, 70)[i]
        # the wild values leave f16's range: the second case spreads NaN, the last one is tame
        x = Mat(rng.standard_normal((rows, dim)) if i == 4 else wild(rng, rows, dim), t, pad, off)
        dy = Mat(rng.standard_normal((rows, dim)), u, pad, off)
        w = Mat(1 + 0.3 * rng.standard_normal((1, dim)), "f32", 0, off) if i != 1 else None
        X = x.np()
        mean, rstd = E.norm_stats(X, 1e-3)
        mm, rr = Mat(mean[None], "f32"), Mat(rstd[None], "f32")
        x8 = None
        if kept is not None:
            q, s = E.encode(X, kept)
            x8 = Eight(rows, dim, kept, 1, pad, off, 2, data=(q, s))
            X = E.decode(q, s, kept)
        add, acc = i % 2 == 1, i >= 2
        dx, sums = backward(x, x8, dy, w, mm, rr, v, add, acc, layout)
        W = w.np() if w else np.ones((1, dim))
        M, R, D = mm.np()[0], rr.np()[0], dy.np()
        wx, ww, wb = E.norm_back(D, X, W, M, R)
        # h: a subtraction and a product; sums over the row as in the forward (45 roundings and h's
        # own, 48); c1, c2 and the last three operations a few more
        h, d = np.abs((X - M[:, None]) * R[:, None]), np.abs(D * W)
        hs = h + np.abs(M * R)[:, None] * 0
        allowed = U * R[:, None] * (8 * d + 56 * d.mean(1, keepdims=True) +
                                    60 * hs * (d * hs).mean(1, keepdims=True)) + 4 * U * (np.abs(wx) + add)
        want = wx + (0.5 if add else 0.0)
        assert_close(dx, want, allowed + E.rounding(v, np.abs(want) + allowed), f"dx {i}")
        # rows of a group one after the other (at most all of them), then groups, CTAs and slices
        path = min(rows, rows / 16 + 2) + 16 + 148 / 8 + 8 + 4
        assert_close(sums[0], ww + (2 if acc else 0), U * (path + 4) * ((np.abs(D) * h).sum(0) + 4), f"dw {i}")
        assert_close(sums[1], wb + (2 if acc else 0), U * (path + 4) * (np.abs(D).sum(0) + 4), f"db {i}")


def test_layernorm_backward_over_many_rows():
    # more rows than the grid takes at once: every CTA walks
    rng = np.random.default_rng(11)
    rows, dim = 5003, 200
    x, dy = Mat(wild(rng, rows, dim), "f32"), Mat(rng.standard_normal((rows, dim)), "f32")
    mean, rstd = E.norm_stats(x.np(), 1e-3)
    mm, rr = Mat(mean[None], "f32"), Mat(rstd[None], "f32")
    dx, sums = backward(x, None, dy, None, mm, rr, "f32", False, False, (0, 0))
    again = backward(x, None, dy, None, mm, rr, "f32", False, False, (0, 0))
    np.testing.assert_array_equal(dx, again[0])
    np.testing.assert_array_equal(sums, again[1])
    X, M, R, D = x.np(), mm.np()[0], rr.np()[0], dy.np()
    wx, ww, wb = E.norm_back(D, X, np.ones((1, dim)), M, R)
    h = np.abs((X - M[:, None]) * R[:, None])
    assert_close(sums[0], ww, U * 400 * (np.abs(D) * h).sum(0), "dw")
    assert_close(sums[1], wb, U * 400 * np.abs(D).sum(0), "db")
    only, _ = backward(x, None, dy, None, mm, rr, "f32", False, False, (0, 0), want_sums=(False, False))
    np.testing.assert_array_equal(only, dx)
    _, s = backward(x, None, dy, None, mm, rr, "f32", False, False, (0, 0), want_sums=(False, True))
    assert np.all(s[0] == 2.0) and np.array_equal(s[1], sums[1])


def test_layernorm_backward_of_no_rows_zeroes_the_sums():
    d = torch.ones(64, device="cuda")
    sums = torch.full((2, 64), 5.0, device="cuda")
    p = d.data_ptr()
    args = (p, A.TYPE_F32, p, A.TYPE_F32, 0, p, p, 0, 64, p, A.TYPE_F32, sums[0].data_ptr(), sums[1].data_ptr())
    space = torch.empty(4096, device="cuda")
    A.layernorm_bwd(*args, space.data_ptr(), 16384, accumulate=True, stream=stream())
    torch.cuda.synchronize()
    assert bool((sums == 5.0).all())
    A.layernorm_bwd(*args, space.data_ptr(), 16384, stream=stream())
    torch.cuda.synchronize()
    assert bool((sums == 0.0).all()) and bool((d == 1.0).all())


def test_layernorm_gradient_against_differences():
    rng = np.random.default_rng(2)
    rows, dim, eps, step = 3, 9, 1e-2, 1e-5
    X, D = rng.standard_normal((rows, dim)), rounded(rng.standard_normal((rows, dim)), "f32")
    W = 1 + 0.3 * rng.standard_normal((1, dim))
    x, dy, w = Mat(X, "f32"), Mat(D, "f32"), Mat(W, "f32")
    X, W = x.np(), w.np()

    def loss(X, W):
        m, r = E.norm_stats(X, eps)
        return float((((X - m[:, None]) * r[:, None] * W) * D).sum())

    mean, rstd = E.norm_stats(X, eps)
    dx, sums = backward(x, None, dy, w, Mat(mean[None], "f32"), Mat(rstd[None], "f32"), "f32", False, False, (0, 0))
    nx, nw = np.zeros_like(X), np.zeros_like(W)
    for a, n, f in ((X, nx, lambda z: loss(z, W)), (W, nw, lambda z: loss(X, z))):
        for i in np.ndindex(*a.shape):
            up, dn = a.copy(), a.copy()
            up[i] += step
            dn[i] -= step
            n[i] = (f(up) - f(dn)) / (2 * step)
    # differences: third derivative * step^2 (1e-10 times O(10)) and 2^-53 * |loss| / step (1e-10);
    # the kernel: statistics rounded to fp32 and some 60 roundings of values up to about 4
    np.testing.assert_allclose(dx, nx, atol=1e-8 + 100 * U * 4)
    np.testing.assert_allclose(sums[0][None], nw, atol=1e-8 + 100 * U * 4)


# ------------------------------------------------------------------------------ GELU
def gelu_flush(z):
    """The hardware exponential flushes below 2^-126 (from |z| = 13.2 on): what z times it, and Q < e / 2,
    lose at most."""
    return np.where(np.abs(z) > 13.2, (np.abs(z) + 1) * 2.0 ** -126, 0.0)


def gelu_slack(z):
    """Relative error of Phi and phi: the fit and its evaluation 2^-21 (the polynomial's eight steps, the
    reciprocal), the hardware exponential 2 + 1.173 z^2 / 2 steps of 2^-23 by CUDA's own bound."""
    return 2.0 ** -21 + 2.0 ** -23 * (3 + 0.6 * z * z)


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 129), (64, 1000), (300, 512)])
@pytest.mark.parametrize("kind", [A.CKPT_I8, A.CKPT_E4M3], ids=["i8", "e4m3"])
@pytest.mark.parametrize("layout", [(0, 0), (3, 1), (8, 4)], ids=["dense", "odd", "strided"])
def test_gelu_with_checkpoint(rows, cols, kind, layout):
    rng = np.random.default_rng(rows + cols)
    pad, off = layout
    for t in ALL:
        z = Mat(rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-6, 4, (rows, 1))), t, pad, off)
        Z = z.np()
        g = out_mat(rows, cols, t, pad, off)
        z8, g8 = Eight(rows, cols, kind, 1, pad, off, 1), Eight(rows, cols, A.CKPT_E4M3, 1, pad, off)
        A.gelu_ckpt8_fwd(z.ptr, E.KINDS[t], rows, cols, g.ptr, E.KINDS[t], z8.v, g8=g8.v, ldz=z.ld, ldg=g.ld,
                         stream=stream())
        torch.cuda.synchronize()
        q, s = E.encode(Z, kind)
        np.testing.assert_array_equal(z8.codes().cpu().numpy(), q)
        np.testing.assert_array_equal(z8.scales(), s)
        G = E.gelu(Z)
        # beyond |z| = 13 the exponential, Q and the result are subnormal: each rounds by up to 2^-150
        # whatever its size, and z multiplies the first two's
        slack = np.abs(G) * gelu_slack(Z) + (2 * np.abs(Z) + 1) * 2.0 ** -150 + gelu_flush(Z)
        assert_close(g.np(), G, slack + E.rounding(t, G), f"g {t}")
        check_codes(g8, G, slack, "g8")
        assert g.untouched() and z8.untouched() and g8.untouched()
        # backward at the kept values
        K = E.decode(q, s, kind)
        dg = Mat(rng.standard_normal((rows, cols)), t, pad, off)
        dz, dz8 = out_mat(rows, cols, t, pad, off), Eight(rows, cols, A.CKPT_E4M3, 1, pad, off)
        D = dg.np()
        want = D * E.gelu_grad(K)
        slack = np.abs(D) * (E.phi(K) + np.abs(K) * np.exp(-K * K / 2) * 0.4) * (gelu_slack(K) + 8 * U)
        # and subnormal: the exponential within one step of 2^-149, times z; Q, their sum and the product with
        # dg half a step each
        slack = slack + (np.abs(D) * (np.abs(K) + 2) + 1) * 2.0 ** -149 + np.abs(D) * gelu_flush(K)
        A.gelu_ckpt8_bwd(dg.ptr, E.KINDS[t], z8.v, rows, cols, dz.ptr, E.KINDS[t], dz8=dz8.v, lddg=dg.ld, lddz=dz.ld,
                         stream=stream())
        torch.cuda.synchronize()
        assert_close(dz.np(), want, slack + E.rounding(t, want), f"dz {t}")
        check_codes(dz8, want, slack, "dz8")
        assert dz.untouched() and dz8.untouched()
        # in place, and the 8-bit result alone
        A.gelu_ckpt8_bwd(dg.ptr, E.KINDS[t], z8.v, rows, cols, dg.ptr, E.KINDS[t], lddg=dg.ld, lddz=dg.ld,
                         stream=stream())
        first = dz8.codes().clone()
        A.gelu_ckpt8_fwd(z.ptr, E.KINDS[t], rows, cols, 0, E.KINDS[t], z8.v, g8=dz8.v, ldz=z.ld, stream=stream())
        torch.cuda.synchronize()
        np.testing.assert_array_equal(dg.np(), dz.np())
        np.testing.assert_array_equal(dz8.codes().cpu().numpy(), g8.codes().cpu().numpy())
        assert first.shape == dz8.codes().shape


def test_results_in_whole_numbers():
    # the 8-bit forms of the results come as I8 too
    rng = np.random.default_rng(12)
    rows, cols = 20, 300
    x = Mat(rng.standard_normal((rows, cols)), "f32")
    y, st, y8 = out_mat(rows, cols, "f32"), Mat(np.zeros((2, rows)), "f32"), Eight(rows, cols, A.CKPT_I8)
    A.layernorm_fwd(x.ptr, A.TYPE_F32, rows, cols, 0, 0, y.ptr, A.TYPE_F32, st.ptr, st.ptr + 4 * st.ld, y8=y8.v,
                    stream=stream())
    g, g8, z8, dz8 = out_mat(rows, cols, "f32"), *(Eight(rows, cols, A.CKPT_I8) for _ in range(3))
    A.gelu_ckpt8_fwd(x.ptr, A.TYPE_F32, rows, cols, g.ptr, A.TYPE_F32, z8.v, g8=g8.v, stream=stream())
    dz = out_mat(rows, cols, "f32")
    A.gelu_ckpt8_bwd(g.ptr, A.TYPE_F32, z8.v, rows, cols, dz.ptr, A.TYPE_F32, dz8=dz8.v, stream=stream())
    torch.cuda.synchronize()
    for wide, eight in ((y, y8), (g, g8), (dz, dz8)):  # exactly the codes of the fp32 result beside them
        q, s = E.encode(wide.np(), A.CKPT_I8)
        np.testing.assert_array_equal(eight.codes().cpu().numpy(), q)
        np.testing.assert_array_equal(eight.scales(), s)


def test_gelu_of_infinities():
    z, g, z8 = Mat(np.array([[np.inf, -np.inf, np.nan, 1e38, -1e38]]), "f32"), out_mat(1, 5, "f32"), Eight(1, 5, A.CKPT_I8)
    A.gelu_ckpt8_fwd(z.ptr, A.TYPE_F32, 1, 5, g.ptr, A.TYPE_F32, z8.v, stream=stream())
    torch.cuda.synchronize()
    got = g.np()[0]
    assert got[0] == np.inf and got[1] == 0 and np.isnan(got[2]) and got[3] == z.np()[0, 3] and got[4] == 0


def test_gelu_over_the_whole_range():
    Z = np.concatenate([np.linspace(-14, 14, 20001), [0.0, -0.0, 60.0, -60.0, 1e30, -1e30]])[None]
    z = Mat(Z, "f32")
    Z = z.np()
    g, z8 = out_mat(1, Z.shape[1], "f32"), Eight(1, Z.shape[1], A.CKPT_I8)
    A.gelu_ckpt8_fwd(z.ptr, A.TYPE_F32, 1, Z.shape[1], g.ptr, A.TYPE_F32, z8.v, stream=stream())
    torch.cuda.synchronize()
    G = E.gelu(Z)
    # below 2^-126 the hardware exponential may flush; 2^-120 covers z times it
    assert_close(g.np(), G, np.abs(G) * gelu_slack(np.clip(Z, -14, 14)) + 2.0 ** -120, "gelu")


def test_gelu_gradient_against_differences():
    Z = np.linspace(-4, 4, 161)[None]
    q, s = E.encode(Z, A.CKPT_I8)
    z8 = Eight(1, 161, A.CKPT_I8, data=(q, s))
    K = E.decode(q, s, A.CKPT_I8)
    one, dz = Mat(np.ones((1, 161)), "f32"), out_mat(1, 161, "f32")
    A.gelu_ckpt8_bwd(one.ptr, A.TYPE_F32, z8.v, 1, 161, dz.ptr, A.TYPE_F32, stream=stream())
    torch.cuda.synchronize()
    num = (E.gelu(K + 1e-5) - E.gelu(K - 1e-5)) / 2e-5
    np.testing.assert_allclose(dz.np(), num, atol=1e-9 + 2.0 ** -19)


def test_nan_in_a_checkpoint_reaches_the_gradient():
    Z = np.zeros((2, 140))
    Z[0, 3], Z[1, 139] = np.nan, np.inf
    z, dz = Mat(Z, "f32"), out_mat(2, 140, "f32")
    for kind in (A.CKPT_I8, A.CKPT_E4M3):
        z8 = Eight(2, 140, kind)
        g = out_mat(2, 140, "f32")
        A.gelu_ckpt8_fwd(z.ptr, A.TYPE_F32, 2, 140, g.ptr, A.TYPE_F32, z8.v, stream=stream())
        A.gelu_ckpt8_bwd(g.ptr, A.TYPE_F32, z8.v, 2, 140, dz.ptr, A.TYPE_F32, stream=stream())
        torch.cuda.synchronize()
        want = np.zeros((2, 140), bool)
        want[0, 3] = want[1, 139] = True
        np.testing.assert_array_equal(np.isnan(dz.np()), want)


# ------------------------------------------------------------------------------ rank product
def status_word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("rows,cols,nb", [(1, 1, 1), (1, 128, 16), (63, 130, 3), (64, 256, 64), (65, 1000, 17),
                                          (129, 127, 33), (750, 1024, 16), (1500, 384, 64), (3001, 260, 8)])
@pytest.mark.parametrize("kind", [A.CKPT_I8, A.CKPT_E4M3], ids=["i8", "e4m3"])
@pytest.mark.parametrize("ut", ALL)
def test_rank_product(rows, cols, nb, kind, ut):
    rng = np.random.default_rng(rows + cols + nb)
    X = wild(rng, rows, cols)
    q, s = E.encode(X, kind)
    for pad, off, acc in ((0, 0, False), (3, 1, True)):
        x = Eight(rows, cols, kind, 1, up16(cols) + 16 * pad, 0, extra=pad, data=(q, s))
        u = Mat(rng.standard_normal((rows, nb)), ut, pad, off)
        c = Mat(rng.standard_normal((nb, cols)), "f32", pad, off)
        was, st = c.np(), status_word()
        A.rank_gemm_ckpt8(u.ptr, E.KINDS[ut], nb, x.v, rows, cols, c.ptr, st.data_ptr(), alpha=0.75, accumulate=acc,
                          ldu=u.ld, ldc=c.ld, stream=stream())
        torch.cuda.synchronize()
        K, V = E.decode(q, s, kind), u.np()
        want = 0.75 * (V.T @ K)
        size = 0.75 * (np.abs(V).T @ np.abs(K))
        if acc:
            want, size = want + was, size + np.abs(was)
        # rows terms in any order, twice that for truncating adds; the product with alpha and the add
        assert_close(c.np(), want, (2 * rows + 4) * U * size + 2.0 ** -140, "c")
        assert c.untouched() and st.item() == 0


@pytest.mark.parametrize("rows,cols,nb,pad,off", [(200, 4737, 8, 4, 4), (200, 4737, 24, 8, 8), (65, 4992, 64, 0, 0),
                                                  (513, 130, 40, 4, 12), (1, 4800, 16, 8, 4), (63, 5001, 19, 1, 2)])
@pytest.mark.parametrize("kind", [A.CKPT_I8, A.CKPT_E4M3], ids=["i8", "e4m3"])
@pytest.mark.parametrize("ut", ALL)
def test_rank_product_of_wide_inputs_and_placed_u(rows, cols, nb, pad, off, kind, ut):
    """256 columns a CTA, and U at 16-byte, 8-byte and odd places."""
    rng = np.random.default_rng(rows + cols + nb + pad + off)
    q, s = E.encode(wild(rng, rows, cols), kind)
    x = Eight(rows, cols, kind, 1, up16(cols), 0, data=(q, s))
    u, c, st = Mat(rng.standard_normal((rows, nb)), ut, pad, off), out_mat(nb, cols, "f32"), status_word()
    for _ in range(2):
        A.rank_gemm_ckpt8(u.ptr, E.KINDS[ut], nb, x.v, rows, cols, c.ptr, st.data_ptr(), ldu=u.ld, ldc=c.ld,
                          stream=stream())
    torch.cuda.synchronize()
    K, V = E.decode(q, s, kind), u.np()
    # rows terms in any order, twice that for truncating adds
    assert_close(c.np(), V.T @ K, (2 * rows + 4) * U * (np.abs(V).T @ np.abs(K)) + 2.0 ** -140, "c")
    assert c.untouched() and st.item() == 0


def test_rank_product_of_no_rows():
    c = Mat(np.ones((4, 40)), "f32", 3)
    x, st = Eight(1, 40, A.CKPT_I8, 1, 8), status_word()
    u = torch.ones(4, device="cuda")
    A.rank_gemm_ckpt8(u.data_ptr(), A.TYPE_F32, 4, x.v, 0, 40, c.ptr, st.data_ptr(), accumulate=True, ldc=c.ld,
                      stream=stream())
    torch.cuda.synchronize()
    assert np.all(c.np() == 1)
    A.rank_gemm_ckpt8(u.data_ptr(), A.TYPE_F32, 4, x.v, 0, 40, c.ptr, st.data_ptr(), ldc=c.ld, stream=stream())
    torch.cuda.synchronize()
    assert np.all(c.np() == 0) and c.untouched()


def test_rank_product_spreads_nan_where_the_formula_does():
    rng = np.random.default_rng(8)
    rows, cols, nb = 300, 400, 20
    X, V = rng.standard_normal((rows, cols)), rng.standard_normal((rows, nb))
    X[17, 5], V[40, 3], V[41, 4] = np.nan, np.nan, np.inf
    q, s = E.encode(X, A.CKPT_E4M3)
    x = Eight(rows, cols, A.CKPT_E4M3, 1, 0, data=(q, s))
    u, c, st = Mat(V, "f32"), out_mat(nb, cols, "f32"), status_word()
    A.rank_gemm_ckpt8(u.ptr, A.TYPE_F32, nb, x.v, rows, cols, c.ptr, st.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    got = c.np()
    want = np.zeros((nb, cols), bool)
    want[:, 5] = want[3] = want[4] = True
    np.testing.assert_array_equal(~np.isfinite(got), want)


# ------------------------------------------------------------------------------ GEMM
GEMM = [(1, 1, 1), (1, 128, 128), (2, 130, 127), (3, 64, 1000), (4, 1000, 129), (8, 256, 1536), (9, 384, 300),
        (16, 1000, 256), (17, 513, 640), (32, 129, 384), (33, 128, 200), (100, 260, 128), (128, 256, 512),
        (129, 300, 385), (257, 1000, 513), (300, 1536, 256), (750, 512, 1024)]


def operands(rng, M, N, K, mn, pad=0):
    X = wild(rng, M, K)
    Wm = rng.standard_normal((K, N) if mn else (N, K)) * 0.05 * np.exp(rng.standard_normal((1, 1)))
    xq, xs = E.encode(X, A.CKPT_E4M3)
    wq, ws = E.encode(Wm, A.CKPT_E4M3, 128)
    x = Eight(M, K, A.CKPT_E4M3, 1, up16(K) + 16 * pad, 0, extra=pad, data=(xq, xs))
    w = Eight(Wm.shape[0], Wm.shape[1], A.CKPT_E4M3, 128, up16(Wm.shape[1]) + 16 * pad, 0, extra=pad, data=(wq, ws))
    return x, w


def product(x, w, mn):
    X, W = x.np(), w.np()
    B = W if mn else W.T
    return X @ B, np.abs(X) @ np.abs(B)


@pytest.mark.parametrize("M,N,K", GEMM)
@pytest.mark.parametrize("mn", [False, True], ids=["k_major", "mn_major"])
def test_gemm(M, N, K, mn):
    rng = np.random.default_rng(M + 3 * N + 7 * K)
    for u, pad, off, bias, acc in (("f32", 0, 0, False, False), ("f16", 0, 0, True, True), ("bf16", 1, 3, True, False),
                                   ("f32", 3, 1, False, True)):
        x, w = operands(rng, M, N, K, mn, pad)
        y = Mat(rng.standard_normal((M, N)), u, pad, off)
        b = Mat(rng.standard_normal((1, N)), "f32", 0, off) if bias else None
        was, st = y.np(), status_word()
        A.gemm_f8(x.v, w.v, M, N, K, y.ptr, E.KINDS[u], st.data_ptr(), w_mn_major=mn, bias=b.ptr if b else 0,
                  accumulate=acc, ldy=y.ld, stream=stream())
        torch.cuda.synchronize()
        want, size = product(x, w, mn)
        if bias:
            want, size = want + b.np(), size + np.abs(b.np())
        if acc:
            want, size = want + was, size + np.abs(was)
        # K products summed in any order, twice that for truncating adds; each block's two scales,
        # bias and the old value one rounding each
        slack = (2 * K + 6) * U * size
        if u == "f16":
            slack = np.where(np.abs(want) + slack > 65504, np.inf, slack)
        assert_close(y.np(), np.where(np.isfinite(slack), want, y.np()), slack + E.rounding(u, want), f"{u} {pad}")
        assert y.untouched() and st.item() == 0


# few tiles and many k-blocks: clusters share a tile's reduction (slices of unequal length, a ragged last one)
FEW_TILES = [(20, 130, 4100), (130, 256, 6144), (100, 1000, 3001), (257, 129, 2600)]


@pytest.mark.parametrize("M,N,K", FEW_TILES)
@pytest.mark.parametrize("mn", [False, True], ids=["k_major", "mn_major"])
def test_gemm_of_few_tiles(M, N, K, mn):
    test_gemm(M, N, K, mn)


def test_gemm_takes_any_scale_and_keeps_nan_in_its_place():
    rng = np.random.default_rng(4)
    for M in (5, 200):
        N, K = 300, 400
        x, w = operands(rng, M, N, K, False)
        x.scale.mul_(1.37)
        w.scale.mul_(0.73)
        y, st = out_mat(M, N, "f32"), status_word()
        A.gemm_f8(x.v, w.v, M, N, K, y.ptr, A.TYPE_F32, st.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        want, size = product(x, w, False)
        assert_close(y.np(), want, (2 * K + 6) * U * size, "scales")
        x.codes()[2, 7] = 127        # NaN in one row of X, one column of W, and one scale of each
        w.codes()[11, 399] = 127
        x.scale[1, 4] = float("inf")
        w.scale[2, 1] = float("nan")
        A.gemm_f8(x.v, w.v, M, N, K, y.ptr, A.TYPE_F32, st.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        bad = np.zeros((M, N), bool)
        bad[2], bad[:, 11], bad[4], bad[:, 128:256] = True, True, True, True
        np.testing.assert_array_equal(~np.isfinite(y.np()), bad)


def test_gemm_with_a_scale_table_that_underflows():
    # zero blocks carry 2^-126: the product of two such scales is 0, and so is the block's part
    M, N, K = 40, 200, 300
    x = Eight(M, K, A.CKPT_E4M3, 1, up16(K), data=E.encode(np.zeros((M, K)), A.CKPT_E4M3))
    w = Eight(N, K, A.CKPT_E4M3, 128, up16(K), data=E.encode(np.zeros((N, K)), A.CKPT_E4M3, 128))
    y, st = out_mat(M, N, "f16"), status_word()
    A.gemm_f8(x.v, w.v, M, N, K, y.ptr, A.TYPE_F16, st.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    assert np.all(y.np() == 0)


# ------------------------------------------------------------------------------ far offsets
def far(rows, ld, dtype):
    return torch.empty((rows - 1) * ld + 512, dtype=dtype, device="cuda")


def rows_of(buf, rows, cols, ld):
    return buf.as_strided((rows, cols), (ld, 1))


def test_rows_more_than_32_bits_apart():
    # strides of 1.5 G elements: row 2 starts beyond 2^31 elements and 2^32 bytes
    rows, cols, ld = 3, 300, 1_500_000_000
    rng = np.random.default_rng(5)
    X = rounded(rng.standard_normal((rows, cols)), "bf16")
    x, q, y = far(rows, ld, torch.bfloat16), far(rows, ld, torch.uint8), far(rows, ld, torch.bfloat16)
    rows_of(x, rows, cols, ld).copy_(torch.from_numpy(X))
    scale = torch.zeros(3, rows, device="cuda")
    v = A.ckpt8(A.CKPT_E4M3, q.data_ptr(), ld, scale.data_ptr(), rows)
    A.ckpt8_store(x.data_ptr(), A.TYPE_BF16, rows, cols, v, ldx=ld, stream=stream())
    A.ckpt8_load(v, rows, cols, y.data_ptr(), A.TYPE_BF16, ldy=ld, stream=stream())
    torch.cuda.synchronize()
    want = E.decode(*E.encode(X, A.CKPT_E4M3), A.CKPT_E4M3)
    np.testing.assert_array_equal(rows_of(y, rows, cols, ld).double().cpu().numpy(), want)
    # norm there and back, GELU there and back, all through the far rows
    st, sums = torch.zeros(2, rows, device="cuda"), torch.zeros(2, cols, device="cuda")
    A.layernorm_fwd(x.data_ptr(), A.TYPE_BF16, rows, cols, 0, 0, y.data_ptr(), A.TYPE_BF16, st[0].data_ptr(),
                    st[1].data_ptr(), ldx=ld, ldy=ld, stream=stream())
    torch.cuda.synchronize()
    mean, rstd = E.norm_stats(X, 1e-5)
    H = (X - mean[:, None]) * rstd[:, None]
    np.testing.assert_allclose(rows_of(y, rows, cols, ld).double().cpu().numpy(), H, rtol=2.0 ** -7, atol=1e-5)
    room = A.layernorm_bwd_workspace(rows, cols)
    space = torch.empty(room // 4, device="cuda")
    A.layernorm_bwd(x.data_ptr(), A.TYPE_BF16, 0, 0, 0, st[0].data_ptr(), st[1].data_ptr(), rows, cols, y.data_ptr(),
                    A.TYPE_BF16, sums[0].data_ptr(), sums[1].data_ptr(), space.data_ptr(), room, x8=v, lddy=ld,
                    lddx=ld, stream=stream())
    torch.cuda.synchronize()
    dx, dw, db = E.norm_back(X, want, np.ones((1, cols)), mean, rstd)
    np.testing.assert_allclose(rows_of(y, rows, cols, ld).double().cpu().numpy(), dx, rtol=2.0 ** -7, atol=1e-4)
    np.testing.assert_allclose(sums[1].double().cpu().numpy(), db, atol=1e-5)
    A.gelu_ckpt8_fwd(x.data_ptr(), A.TYPE_BF16, rows, cols, y.data_ptr(), A.TYPE_BF16, v, ldz=ld, ldg=ld,
                     stream=stream())
    torch.cuda.synchronize()
    np.testing.assert_allclose(rows_of(y, rows, cols, ld).double().cpu().numpy(), E.gelu(X), rtol=2.0 ** -7, atol=1e-5)
    A.gelu_ckpt8_bwd(x.data_ptr(), A.TYPE_BF16, v, rows, cols, y.data_ptr(), A.TYPE_BF16, lddg=ld, lddz=ld,
                     stream=stream())
    torch.cuda.synchronize()
    np.testing.assert_allclose(rows_of(y, rows, cols, ld).double().cpu().numpy(), X * E.gelu_grad(want),
                               rtol=2.0 ** -7, atol=1e-5)
    # products: C and Y with far rows, X with far rows
    u = torch.from_numpy(X[:, :3].copy()).to("cuda").float()
    word, c = status_word(), far(3, ld, torch.float32)
    A.ckpt8_store(x.data_ptr(), A.TYPE_BF16, rows, cols, v, ldx=ld, stream=stream())
    A.rank_gemm_ckpt8(u.data_ptr(), A.TYPE_F32, 3, v, rows, cols, c.data_ptr(), word.data_ptr(), ldc=ld,
                      stream=stream())
    torch.cuda.synchronize()
    np.testing.assert_allclose(rows_of(c, 3, cols, ld).double().cpu().numpy(), X[:, :3].T @ want, atol=1e-5)
    del c
    w = Eight(40, cols, A.CKPT_E4M3, 128, up16(cols), data=E.encode(rng.standard_normal((40, cols)), A.CKPT_E4M3, 128))
    out = far(rows, ld, torch.bfloat16)
    A.gemm_f8(v, w.v, rows, 40, cols, out.data_ptr(), A.TYPE_BF16, word.data_ptr(), ldy=ld, stream=stream())
    torch.cuda.synchronize()
    np.testing.assert_allclose(rows_of(out, rows, 40, ld).double().cpu().numpy(), want @ w.np().T, rtol=2.0 ** -7,
                               atol=1e-4)


def test_gemm_of_rows_more_than_32_bits_apart_on_the_tensor_cores():
    rows, cols, ld = 200, 256, 1 << 25
    rng = np.random.default_rng(6)
    qx, sx = E.encode(rng.standard_normal((rows, cols)), A.CKPT_E4M3)
    q = far(rows, ld, torch.uint8)
    rows_of(q, rows, cols, ld).copy_(torch.from_numpy(qx))
    scale = torch.from_numpy(sx.astype(np.float32)).to("cuda")
    v = A.ckpt8(A.CKPT_E4M3, q.data_ptr(), ld, scale.data_ptr(), rows)
    w = Eight(300, cols, A.CKPT_E4M3, 128, up16(cols), data=E.encode(rng.standard_normal((300, cols)), A.CKPT_E4M3, 128))
    y, word = out_mat(rows, 300, "f32"), status_word()
    A.gemm_f8(v, w.v, rows, 300, cols, y.ptr, A.TYPE_F32, word.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    X = E.decode(qx, sx, A.CKPT_E4M3)
    assert_close(y.np(), X @ w.np().T, (2 * cols + 6) * U * (np.abs(X) @ np.abs(w.np()).T), "far")
    assert word.item() == 0


# ------------------------------------------------------------------------------ how they are called
def test_host_memory_is_refused():
    host = np.zeros(4096, np.float32)
    dev = torch.zeros(4096, device="cuda")
    e = Eight(4, 64, A.CKPT_I8)
    with pytest.raises(A.ActError) as err:
        A.ckpt8_store(host.ctypes.data, A.TYPE_F32, 4, 64, e.v, stream=stream())
    assert err.value.code == A.ACT_ERR_INVALID and "device memory" in str(err.value)
    with pytest.raises(A.ActError):
        A.layernorm_fwd(dev.data_ptr(), A.TYPE_F32, 4, 64, 0, 0, dev.data_ptr(), A.TYPE_F32, dev.data_ptr(),
                        host.ctypes.data, stream=stream())


def block_pass(t, s):
    """A pre-norm feed-forward block with an adapter on its first projection, trained: every operator in
    the order a step runs them."""
    rows, d, f, r = t["rows"], t["d"], t["f"], t["r"]
    A.layernorm_fwd(t["x"].ptr, A.TYPE_F32, rows, d, t["w"].ptr, t["b"].ptr, 0, 0, t["st"].ptr,
                    t["st"].ptr + 4 * t["st"].ld, y8=t["y8"].v, x8=t["x8"].v, stream=s)
    A.gemm_f8(t["y8"].v, t["w1"].v, rows, f, d, t["z"].ptr, A.TYPE_F16, t["status"].data_ptr(), stream=s)
    A.gelu_ckpt8_fwd(t["z"].ptr, A.TYPE_F16, rows, f, 0, A.TYPE_F16, t["z8"].v, g8=t["g8"].v, stream=s)
    A.gemm_f8(t["g8"].v, t["w2"].v, rows, d, f, t["out"].ptr, A.TYPE_F32, t["status"].data_ptr(), stream=s)
    A.ckpt8_store(t["dout"].ptr, A.TYPE_F32, rows, d, t["d8"].v, stream=s)
    A.gemm_f8(t["d8"].v, t["w2"].v, rows, f, d, t["dg"].ptr, A.TYPE_BF16, t["status"].data_ptr(), w_mn_major=True,
              stream=s)
    A.gelu_ckpt8_bwd(t["dg"].ptr, A.TYPE_BF16, t["z8"].v, rows, f, t["dg"].ptr, A.TYPE_BF16, dz8=t["dz8"].v, stream=s)
    A.rank_gemm_ckpt8(t["u"].ptr, A.TYPE_F16, r, t["y8"].v, rows, d, t["dA"].ptr, t["status"].data_ptr(), stream=s)
    A.gemm_f8(t["dz8"].v, t["w1"].v, rows, d, f, t["dh"].ptr, A.TYPE_F32, t["status"].data_ptr(), w_mn_major=True,
              stream=s)
    A.layernorm_bwd(t["dh"].ptr, A.TYPE_F32, 0, 0, t["w"].ptr, t["st"].ptr, t["st"].ptr + 4 * t["st"].ld, rows, d,
                    t["dx"].ptr, A.TYPE_F32, t["sums"].ptr, t["sums"].ptr + 4 * t["sums"].ld,
                    t["space"].data_ptr(), t["space"].numel() * 4, add=t["dout"].ptr, x8=t["x8"].v, stream=s)


def block_tensors(rng, rows, d, f, r):
    t = dict(rows=rows, d=d, f=f, r=r, status=status_word())
    t["x"] = Mat(wild(rng, rows, d) * 0.01 + rng.standard_normal((rows, d)), "f32")
    t["w"], t["b"] = Mat(1 + 0.2 * rng.standard_normal((1, d)), "f32"), Mat(0.2 * rng.standard_normal((1, d)), "f32")
    t["dout"], t["u"] = Mat(rng.standard_normal((rows, d)), "f32"), Mat(rng.standard_normal((rows, r)), "f16")
    t["st"], t["sums"] = out_mat(2, rows, "f32"), out_mat(2, d, "f32")
    e = lambda n: Eight(rows, n, A.CKPT_E4M3, 1, up16(n))  # noqa: E731
    t["y8"], t["g8"], t["d8"], t["dz8"] = e(d), e(f), e(d), e(f)
    t["x8"], t["z8"] = Eight(rows, d, A.CKPT_I8, 1, up16(d)), Eight(rows, f, A.CKPT_I8, 1, up16(f))
    for k, n, m in (("w1", f, d), ("w2", d, f)):
        t[k] = Eight(n, m, A.CKPT_E4M3, 128, up16(m), data=E.encode(rng.standard_normal((n, m)) / np.sqrt(m),
                                                                    A.CKPT_E4M3, 128))
    t["z"], t["dg"] = out_mat(rows, f, "f16"), out_mat(rows, f, "bf16")
    t["out"], t["dh"], t["dx"], t["dA"] = (out_mat(rows, d, "f32"), out_mat(rows, d, "f32"), out_mat(rows, d, "f32"),
                                           out_mat(r, d, "f32"))
    t["space"] = torch.empty(A.layernorm_bwd_workspace(rows, d) // 4, device="cuda")
    return t


KEPT = ["out", "dx", "dA", "sums", "st", "z", "dg", "dh"]


def block_reference(t):
    """The same pass in 64 bits from the kernels' own 8-bit operands and rounded intermediates, one
    operator at a time."""
    X, W, B = t["x"].np(), t["w"].np(), t["b"].np()
    mean, rstd = t["st"].np()
    y8, g8, d8, dz8 = (t[k].np() for k in ("y8", "g8", "d8", "dz8"))
    w1, w2, D = t["w1"].np(), t["w2"].np(), t["dout"].np()
    h = (X - mean[:, None]) * rstd[:, None]
    ref = dict(y8=h * W + B, z=y8 @ w1.T, g8=E.gelu(t["z"].np()), out=g8 @ w2.T, d8=D, dA=t["u"].np().T @ y8,
               dz8=(d8 @ w2) * E.gelu_grad(t["z8"].np()), dh=dz8 @ w1)
    dx, dw, db = E.norm_back(t["dh"].np(), t["x8"].np(), W, mean, rstd)
    ref.update(dx=dx + D, sums=np.stack([dw, db]))
    return ref


@pytest.mark.parametrize("rows,d,f,r", [(3, 64, 256, 4), (70, 200, 520, 16), (300, 256, 1024, 16)])
def test_a_feed_forward_block_runs_through_all_operators(rows, d, f, r):
    t = block_tensors(np.random.default_rng(rows), rows, d, f, r)
    block_pass(t, stream())
    torch.cuda.synchronize()
    ref = block_reference(t)
    assert t["status"].item() == 0
    rel = lambda k: np.linalg.norm(t[k].np() - ref[k]) / np.linalg.norm(ref[k])  # noqa: E731
    # per operator and in the 2-norm: one rounding of the result's type (e4m3 2^-4, f16 2^-11), fp32
    # sums of up to f terms (2 f u, times up to 30 for terms that cancel), GELU 2^-20; dz8 also holds
    # dg's rounding to bf16
    sums = 2 * f * U * 30
    for k, bound in (("y8", 2.0 ** -4), ("z", 2.0 ** -11 + sums), ("g8", 2.0 ** -4 + 2.0 ** -18), ("out", sums),
                     ("d8", 2.0 ** -4), ("dA", sums), ("dz8", 2.0 ** -4 + 2.0 ** -7), ("dh", sums), ("dx", sums),
                     ("sums", sums)):
        assert rel(k) <= bound, (k, rel(k), bound)


def test_passes_captured_into_graphs_and_on_other_streams_agree_with_eager_ones():
    rng = np.random.default_rng(77)
    t = block_tensors(rng, 200, 256, 512, 16)
    block_pass(t, stream())
    torch.cuda.synchronize()
    eager = {k: t[k].np() for k in KEPT}
    other = torch.cuda.Stream()
    for k in KEPT:
        t[k].view.fill_(9.0)
    torch.cuda.synchronize()
    block_pass(t, other.cuda_stream)
    other.synchronize()
    for k in KEPT:
        np.testing.assert_array_equal(t[k].np(), eager[k], err_msg=k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=other):
        block_pass(t, torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        for k in KEPT:
            t[k].view.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        for k in KEPT:
            np.testing.assert_array_equal(t[k].np(), eager[k], err_msg=k)


def test_two_passes_at_once_on_two_streams():
    rng = np.random.default_rng(78)
    ts = [block_tensors(rng, 150, 384, 640, 8) for _ in range(2)]
    want = []
    for t in ts:
        block_pass(t, stream())
        torch.cuda.synchronize()
        want.append({k: t[k].np() for k in KEPT})
        for k in KEPT:
            t[k].view.fill_(9.0)
    streams = [torch.cuda.Stream() for _ in ts]
    torch.cuda.synchronize()
    for _ in range(3):
        for t, s in zip(ts, streams):
            block_pass(t, s.cuda_stream)
    torch.cuda.synchronize()
    for t, w in zip(ts, want):
        for k in KEPT:
            np.testing.assert_array_equal(t[k].np(), w[k], err_msg=k)
