"""The 8-bit checkpoint, layer norm, GELU and product operators on tensors of more rows than a launch takes at
once, where every loop over row groups, tiles and k-blocks turns several times (the sizes that reach
that on 148 SMs stand beside each list).  The definitions in 64 bits run as plain torch operations."""
import numpy as np
import pytest
import torch

import actrain as A
import eight_bit as E
from test_gpu_train_ops import TORCH, U, Eight, status_word, stream

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rand(g, *n):
    return torch.randn(*n, device="cuda", generator=g, dtype=torch.float64)


TABLE = torch.from_numpy(E.E4M3)


def value(codes, kind):
    """What codes [..] stand for before scaling, in 64 bits."""
    if kind == A.CKPT_I8:
        v = codes.view(torch.int8).double()
        return torch.where(v == -128, torch.nan, v)
    return TABLE.to("cuda")[codes.long()]


def spread(scale, shape, block=1):
    rows, cols = shape
    at = torch.arange(rows, device="cuda") // block
    return scale.double()[:, at].t()[:, torch.arange(cols, device="cuda") // 128]


def read(e):
    """The values of an 8-bit tensor, in 64 bits."""
    return value(e.codes(), e.kind) * spread(e.scale, (e.rows, e.cols), e.block)


def scales_of(x, kind, block=1):
    """The definition's scales [ceil(cols / 128)][ceil(rows / block)], finite x in 64 bits."""
    rows, cols = x.shape
    nr, nc = -(-rows // block), -(-cols // 128)
    wide = torch.zeros(nr * block, nc * 128, dtype=torch.float64, device="cuda")
    wide[:rows, :cols] = x.abs()
    most = wide.view(nr, block, nc, 128).amax(dim=(1, 3))
    e = torch.frexp(most / E.TOP[kind])[1].double()  # most / top lies in [2^(e - 1), 2^e)
    e = torch.where(most <= E.TOP[kind] * torch.exp2(e - 1), e - 1, e)
    e = torch.where(most == 0, -126.0, e).clamp(min=-126)
    return torch.exp2(e).t()


def kept(x, kind, block=1):
    """x as its 8-bit form stands for it: scales, and x / s rounded to nearest even, times s."""
    s = scales_of(x, kind, block)
    w = spread(s, x.shape, block)
    v = x / w
    if kind == A.CKPT_I8:
        return torch.round(v) * w, s
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step * w, s


def phi(z):
    # erfc keeps its relative accuracy in the tail; 1 + erf, and functions made of it, are off by 1e-16 there
    return 0.5 * torch.special.erfc(-z * 0.7071067811865476)


def half_step(t, y):
    return torch.clamp(y.abs() * E.HALF[t], min=E.TINY[t])


def check(got, want, allowed, what):
    off = (got.double() - want).abs() - allowed
    assert bool((off <= 0).all()), f"{what}: {int((off > 0).sum())} of {off.numel()} off, by up to {off.max().item():.3g} more"


def eight(rows, cols, kind, block=1, pitched=False):
    return Eight(rows, cols, kind, block, -cols % 16 if pitched else 0)


# ------------------------------------------------------------------------------ store and load
# 148 SMs x 8 blocks x 8 warps, four rows of a block column each: 37888 rows of 128 columns
@pytest.mark.parametrize("rows,cols", [(90001, 100), (40003, 260)])
@pytest.mark.parametrize("kind", [A.CKPT_I8, A.CKPT_E4M3], ids=["i8", "e4m3"])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_store_and_load_of_many_rows(rows, cols, kind, t):
    x = (rand(gen(rows), rows, cols) * torch.exp2(torch.arange(rows, device="cuda") % 17 - 8.0)[:, None]).to(TORCH[t])
    e, y = eight(rows, cols, kind), torch.empty(rows, cols, device="cuda")
    A.ckpt8_store(x.data_ptr(), E.KINDS[t], rows, cols, e.v, stream=stream())
    A.ckpt8_load(e.v, rows, cols, y.data_ptr(), A.TYPE_F32, stream=stream())
    torch.cuda.synchronize()
    want, s = kept(x.double(), kind)
    assert torch.equal(e.scale.double(), s) and torch.equal(y.double(), want)


def test_store_of_more_square_blocks_than_grid_rows():
    # 65535 block rows in a grid: the last ones are a second turn
    rows, cols = 65537 * 128 + 5, 3
    x = rand(gen(1), rows, cols).float()
    e, y = eight(rows, cols, A.CKPT_E4M3, 128), torch.empty(rows, cols, device="cuda")
    A.ckpt8_store(x.data_ptr(), A.TYPE_F32, rows, cols, e.v, block_rows=128, stream=stream())
    A.ckpt8_load(e.v, rows, cols, y.data_ptr(), A.TYPE_F32, block_rows=128, stream=stream())
    torch.cuda.synchronize()
    want, s = kept(x.double(), A.CKPT_E4M3, 128)
    assert torch.equal(e.scale.double(), s) and torch.equal(y.double(), want)


# ------------------------------------------------------------------------------ GELU
def gelu_slack(z):
    """Relative error of the normal tail and of the density, and what the hardware exponential flushes below
    2^-126.  The fit evaluated in fp32 with a reciprocal one step off 5.6e-7 (test_tail_fit.py), the
    exponential 2^-22 (its stated bound), their product 2^-24: together below 2^-20.  The exponent is z^2
    times a constant that is off by 0.224 * 2^-24, rounded twice: z^2 / 2 * 2.224 * 2^-24."""
    return 2.0 ** -20 + 0.5561 * 2.0 ** -23 * z * z, (z.abs() + 2) * 2.0 ** -126


@pytest.mark.parametrize("rows,cols,t", [(90001, 100, "f32"), (40003, 260, "f16"), (40003, 260, "bf16")])
@pytest.mark.parametrize("kind", [A.CKPT_I8, A.CKPT_E4M3], ids=["i8", "e4m3"])
def test_gelu_of_many_rows(rows, cols, t, kind):
    g = gen(rows + 1)
    z, dg = (1.5 * rand(g, rows, cols)).to(TORCH[t]), rand(g, rows, cols).to(TORCH[t])
    out, dz = torch.empty_like(z), torch.empty_like(z)
    z8 = eight(rows, cols, kind)
    A.gelu_ckpt8_fwd(z.data_ptr(), E.KINDS[t], rows, cols, out.data_ptr(), E.KINDS[t], z8.v, stream=stream())
    A.gelu_ckpt8_bwd(dg.data_ptr(), E.KINDS[t], z8.v, rows, cols, dz.data_ptr(), E.KINDS[t], stream=stream())
    torch.cuda.synchronize()
    Z = z.double()
    want, s = kept(Z, kind)
    assert torch.equal(z8.scale.double(), s) and torch.equal(read(z8), want)
    rel, flush = gelu_slack(Z)
    G = Z * phi(Z)
    slack = G.abs() * rel + flush
    check(out, G, slack + half_step(t, G.abs() + slack), "g")
    rel, flush = gelu_slack(want)
    density = torch.exp(-want * want / 2) * 0.3989422804014327
    D = dg.double() * (phi(want) + want * density)
    slack = dg.double().abs() * ((phi(want) + (want * density).abs()) * (rel + 8 * U) + flush)
    check(dz, D, slack + half_step(t, D.abs() + slack), "dz")


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 129), (64, 1000), (9001, 512)])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", [A.CKPT_I8, A.CKPT_E4M3], ids=["i8", "e4m3"])
@pytest.mark.parametrize("pad,off", [(0, 0), (3, 1), (8, 4)], ids=["dense", "odd", "strided"])
def test_gelu_backward_into_8_bits_alone(rows, cols, t, kind, pad, off):
    # dz left out beside dz8: the same codes as with it
    g = gen(rows + cols)
    z = rand(g, rows, cols).to(TORCH[t])
    dg = torch.zeros(off + rows * (cols + pad), dtype=TORCH[t], device="cuda")
    dg = dg[off:].view(rows, cols + pad)[:, :cols]
    dg.copy_(rand(g, rows, cols))
    z8 = eight(rows, cols, kind)
    A.ckpt8_store(z.data_ptr(), E.KINDS[t], rows, cols, z8.v, stream=stream())
    dz = torch.empty(rows, cols, dtype=TORCH[t], device="cuda")
    for fmt in (A.CKPT_E4M3, A.CKPT_I8):
        both, alone = (Eight(rows, cols, fmt, 1, pad, off) for _ in range(2))
        A.gelu_ckpt8_bwd(dg.data_ptr(), E.KINDS[t], z8.v, rows, cols, dz.data_ptr(), E.KINDS[t], dz8=both.v,
                         lddg=cols + pad, stream=stream())
        A.gelu_ckpt8_bwd(dg.data_ptr(), E.KINDS[t], z8.v, rows, cols, 0, E.KINDS[t], dz8=alone.v, lddg=cols + pad,
                         stream=stream())
        torch.cuda.synchronize()
        assert torch.equal(both.codes(), alone.codes()) and torch.equal(both.scale, alone.scale)
        assert alone.untouched() and both.untouched()
        # and they are the gradient's: half a step of the format at most, and what the gradient itself may be off
        want = dg.double() * (phi(read(z8)) + read(z8) * torch.exp(-read(z8) ** 2 / 2) * 0.3989422804014327)
        w = spread(alone.scale, (rows, cols))
        half = 0.5 * w if fmt == A.CKPT_I8 else torch.maximum(want.abs() * 2.0 ** -4, w * 2.0 ** -10)
        check(read(alone), want, half + dg.double().abs() * 2.0 ** -16, "dz8")


# ------------------------------------------------------------------------------ layer norm
# rows of all groups that run at once, at most (8 blocks of 256 threads an SM): 9472 up to 512 columns, 4736 up
# to 1024, 2368 up to 2048, 1184 up to 4096, 592 beyond
NORM = [(20011, 130), (10007, 700), (5003, 1500), (5003, 1900), (2600, 2900), (1301, 5000)]


def norm_want(x, w, b, eps):
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    return mean, rstd, d * rstd * w + b


@pytest.mark.parametrize("rows,dim", NORM)
@pytest.mark.parametrize("t,kind", [("f32", A.CKPT_E4M3), ("bf16", A.CKPT_I8)], ids=["f32-e4m3", "bf16-i8"])
def test_layernorm_of_many_rows(rows, dim, t, kind):
    g = gen(rows + dim)
    x = (rand(g, rows, dim) * (1 + torch.arange(rows, device="cuda") % 5)[:, None] + rand(g, rows, 1)).to(TORCH[t])
    w, b = (1 + 0.3 * rand(g, dim)).float(), (0.3 * rand(g, dim)).float()
    y, st = torch.empty(rows, dim, device="cuda"), torch.empty(2, rows, device="cuda")
    x8, y8 = eight(rows, dim, kind), eight(rows, dim, A.CKPT_E4M3)
    A.layernorm_fwd(x.data_ptr(), E.KINDS[t], rows, dim, w.data_ptr(), b.data_ptr(), y.data_ptr(), A.TYPE_F32,
                    st[0].data_ptr(), st[1].data_ptr(), eps=1e-5, y8=y8.v, x8=x8.v, stream=stream())
    torch.cuda.synchronize()
    X, W, B = x.double(), w.double(), b.double()
    mean, rstd, Y = norm_want(X, W, B, 1e-5)
    # as in test_gpu_train_ops: a sum takes at most 42 roundings on any path
    size = X.abs()
    dmean = 42 * U * size.mean(1, keepdim=True)
    off = (X - mean).abs()
    check(st[0], mean[:, 0], (dmean + U * mean.abs())[:, 0], "mean")
    far = off.mean(1, keepdim=True)
    dvar = 46 * U * rstd ** -2 + 2 * dmean * far + dmean ** 2 + 2 * U * size.amax(1, keepdim=True) * far
    drstd = 0.5 * rstd ** 3 * dvar * 1.01 + 4 * U * rstd
    check(st[1], rstd[:, 0], drstd[:, 0], "rstd")
    h = (X - mean) * rstd
    dh = (dmean + U * off) * rstd + off * drstd + 2 * U * h.abs()
    slack = dh * W.abs() + 2 * U * ((h * W).abs() + Y.abs())
    check(y, Y, slack + half_step("f32", Y.abs() + slack), "y")
    want, s = kept(X, kind)
    assert torch.equal(x8.scale.double(), s) and torch.equal(read(x8), want)
    # y8 is the 8-bit form of the fp32 result beside it, exactly
    want, s = kept(y.double(), A.CKPT_E4M3)
    assert torch.equal(y8.scale.double(), s) and torch.equal(read(y8), want)


@pytest.mark.parametrize("rows,dim", NORM)
@pytest.mark.parametrize("t,kind", [("f32", None), ("bf16", A.CKPT_I8), ("f16", A.CKPT_E4M3)], ids=["f32", "i8", "e4m3"])
def test_layernorm_backward_of_many_rows(rows, dim, t, kind):
    g = gen(rows - dim)
    x, dy = rand(g, rows, dim).to(TORCH[t]), rand(g, rows, dim).to(TORCH[t])
    w = (1 + 0.3 * rand(g, dim)).float()
    mean, rstd, _ = norm_want(x.double(), 1.0, 0.0, 1e-5)
    st = torch.stack([mean[:, 0], rstd[:, 0]]).float()
    x8 = None
    if kind:
        x8 = eight(rows, dim, kind)
        A.ckpt8_store(x.data_ptr(), E.KINDS[t], rows, dim, x8.v, stream=stream())
    dx, sums = torch.full((rows, dim), 0.5, device="cuda"), torch.full((2, dim), 2.0, device="cuda")
    room = A.layernorm_bwd_workspace(rows, dim)
    space = torch.empty(room // 4, device="cuda")
    A.layernorm_bwd(dy.data_ptr(), E.KINDS[t], 0 if kind else x.data_ptr(), E.KINDS[t], w.data_ptr(), st[0].data_ptr(),
                    st[1].data_ptr(), rows, dim, dx.data_ptr(), A.TYPE_F32, sums[0].data_ptr(), sums[1].data_ptr(),
                    space.data_ptr(), room, accumulate=True, add=dx.data_ptr(), x8=x8.v if x8 else None, stream=stream())
    torch.cuda.synchronize()
    X = read(x8) if kind else x.double()
    M, R = st.double()[0][:, None], st.double()[1][:, None]
    D, h = dy.double(), (X - M) * R
    d = D * w.double()
    want = R * (d - d.mean(1, keepdim=True) - h * (d * h).mean(1, keepdim=True)) + 0.5
    # as in test_gpu_train_ops, and h's own roundings where x is not small against its mean
    ha = h.abs() + (M * R).abs()
    allowed = U * R * (8 * d.abs() + 56 * d.abs().mean(1, keepdim=True) +
                       60 * ha * (d.abs() * ha).mean(1, keepdim=True)) + 5 * U * (want.abs() + 1)
    check(dx, want, allowed, "dx")
    path = rows / 148 + 2 + 16 + 148 / 8 + 8 + 4  # rows of a block one after the other, groups, blocks, slices
    check(sums[0], (D * h).sum(0) + 2, U * (path + 6) * ((D.abs() * ha).sum(0) + 4), "dw")
    check(sums[1], D.sum(0) + 2, U * (path + 4) * (D.abs().sum(0) + 4), "db")


# ------------------------------------------------------------------------------ rank product
# Blocks of 64 rows: sixteen slices of a narrow X (24000 rows: 23 or 24 blocks each, so five or six times
# 256 rows and three turns of the ring), and 256 columns a block from 4737 columns on, six slices of 21
@pytest.mark.parametrize("rows,cols,nb", [(24001, 130, 16), (24001, 300, 64), (24001, 300, 5), (8003, 4900, 64),
                                          (8003, 4900, 17)])
@pytest.mark.parametrize("kind", [A.CKPT_I8, A.CKPT_E4M3], ids=["i8", "e4m3"])
@pytest.mark.parametrize("ut", ["f32", "f16", "bf16"])
def test_rank_product_of_many_rows(rows, cols, nb, kind, ut):
    g = gen(rows + cols + nb)
    x8, st = eight(rows, cols, kind, pitched=True), status_word()
    x8.codes().copy_(torch.randint(-127, 128, (rows, cols), device="cuda", generator=g, dtype=torch.int8).view(torch.uint8)
                     if kind == A.CKPT_I8 else
                     torch.randint(0, 127, (rows, cols), device="cuda", generator=g, dtype=torch.uint8) |
                     (torch.randint(0, 2, (rows, cols), device="cuda", generator=g, dtype=torch.uint8) << 7))
    x8.scale.copy_(torch.exp2(torch.randint(-9, -3, x8.scale.shape, device="cuda", generator=g).double()))
    u, c = rand(g, rows, nb).to(TORCH[ut]), torch.full((nb, cols), 1.5, device="cuda")
    for turn in range(2):
        A.rank_gemm_ckpt8(u.data_ptr(), E.KINDS[ut], nb, x8.v, rows, cols, c.data_ptr(), st.data_ptr(), alpha=0.5,
                          accumulate=turn == 0, stream=stream())
        torch.cuda.synchronize()
        X, V = read(x8), u.double()
        want, size = 0.5 * (V.t() @ X), 0.5 * (V.abs().t() @ X.abs())
        if turn == 0:
            want, size = want + 1.5, size + 1.5
        # inside 256 rows in any order, twice that for truncating adds; then 256 rows, slices one after the
        # other, the product with alpha and the old value
        assert rows < 256 * 100
        check(c, want, (2 * 256 + 100 + 16 + 4) * U * size, "c")
        assert st.item() == 0


# ------------------------------------------------------------------------------ GEMM
# 128-wide tiles in two rounds (312 tiles), 256-wide ones in one (114) and two (240, ragged both ways), and three
# rounds of either (M, N, K with the rule of gemm_f8)
BIG = [(3000, 1540, 300), (2400, 1500, 1000), (3000, 2500, 129), (2999, 2500, 520), (6001, 1793, 257), (9000, 1050, 400)]


def rounds(M, N, bn):
    tiles = -(-M // 128) * -(-N // bn)
    return -(-tiles // 148)


def test_sizes_of_the_large_products_reach_both_tile_widths_in_several_rounds():
    wide = [rounds(M, N, 256) for M, N, _ in BIG if rounds(M, N, 256) * 256 <= rounds(M, N, 128) * 128]
    narrow = [rounds(M, N, 128) for M, N, _ in BIG if rounds(M, N, 256) * 256 > rounds(M, N, 128) * 128]
    assert min(wide) == 1 and max(wide) >= 2 and max(narrow) >= 3


@pytest.mark.parametrize("M,N,K", BIG)
@pytest.mark.parametrize("mn", [False, True], ids=["k_major", "mn_major"])
def test_gemm_of_many_tiles(M, N, K, mn):
    g = gen(M + N + K)
    x8, w8, st = eight(M, K, A.CKPT_E4M3, 1, True), eight(*((K, N) if mn else (N, K)), A.CKPT_E4M3, 128, True), status_word()
    x = (rand(g, M, K) * torch.exp2(torch.arange(M, device="cuda") % 11 - 5.0)[:, None]).float()
    w = (0.05 * rand(g, w8.rows, w8.cols)).float()
    A.ckpt8_store(x.data_ptr(), A.TYPE_F32, M, K, x8.v, stream=stream())
    A.ckpt8_store(w.data_ptr(), A.TYPE_F32, w8.rows, w8.cols, w8.v, block_rows=128, stream=stream())
    X, W, bias = read(x8), read(w8), rand(g, N).float()
    W = W if mn else W.t()
    plain, size = X @ W, X.abs() @ W.abs()
    for t, pad, keep, add in (("f32", 4, False, None), ("bf16", 0, True, bias), ("f16", 3, False, bias), ("f32", 1, True, None)):
        held = torch.full((M, N + pad), 0.25, dtype=TORCH[t], device="cuda")
        y = held[:, :N]
        A.gemm_f8(x8.v, w8.v, M, N, K, y.data_ptr(), E.KINDS[t], st.data_ptr(), w_mn_major=mn,
                  bias=add.data_ptr() if add is not None else 0, accumulate=keep, ldy=N + pad, stream=stream())
        torch.cuda.synchronize()
        want, most = plain, size
        if add is not None:
            want, most = want + add.double(), most + add.double().abs()
        if keep:
            want, most = want + 0.25, most + 0.25
        # 128 products of a block in any order, twice that for truncating adds; the blocks one after the other,
        # a block's two scales, bias and the old value one rounding each
        slack = (2 * 128 + K / 128 + 8) * U * most
        check(y, want, slack + half_step(t, want.abs() + slack), f"{t} {pad}")
        assert bool((held[:, N:] == 0.25).all()) and st.item() == 0
