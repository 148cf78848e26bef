"""Plain 64-bit forms of the 8-bit tensors, layer norm, GELU and products, for the tests of the
operators that use them (numpy; the definition, not the kernels' way of computing it)."""
import math

import numpy as np

import actrain as A

TOP = {A.CKPT_I8: 127.0, A.CKPT_E4M3: 448.0}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # half a step, relative
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half the subnormal step
KINDS = {"f32": A.TYPE_F32, "f16": A.TYPE_F16, "bf16": A.TYPE_BF16}


def e4m3_table():
    """The value of each of the 256 codes (sign, 4 exponent bits of bias 7, 3 mantissa bits; 0x7f NaN)."""
    v = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        v[c] = math.copysign(x, -1 if c & 128 else 1) if (c & 127) != 127 else math.nan
    return v


E4M3 = e4m3_table()


def block_scales(x, kind, block_rows=1):
    """[ceil(cols/128)][ceil(rows/block_rows)] smallest powers of two s >= 2^-126 with max |finite x| <= top s."""
    rows, cols = x.shape
    nc, nr = -(-cols // 128), -(-rows // block_rows)
    out = np.zeros((nc, nr))
    for c in range(nc):
        for r in range(nr):
            b = x[r * block_rows:(r + 1) * block_rows, c * 128:(c + 1) * 128]
            b = np.abs(b[np.isfinite(b)])
            most = b.max() if b.size else 0.0
            e = -126
            if most > 0:
                e = max(-126, math.frexp(most / TOP[kind])[1] - 1)  # most / top is in [2^e, 2^(e + 1))
                while most > TOP[kind] * 2.0 ** e:
                    e += 1
            out[c, r] = 2.0 ** e
    return out


def spread(scale, shape, block_rows=1):
    """Each element's scale."""
    return np.repeat(np.repeat(scale.T, block_rows, 0)[:shape[0]], 128, 1)[:, :shape[1]]


def encode(x, kind, block_rows=1):
    """(codes uint8, scales) of x in 64 bits."""
    x = np.asarray(x, np.float64)
    scale = block_scales(x, kind, block_rows)
    bad = ~np.isfinite(x)
    v = np.where(bad, 0, x) / spread(scale, x.shape, block_rows)
    if kind == A.CKPT_I8:
        q = np.rint(v).astype(np.int64)
        q[bad] = -128
        return (q & 255).astype(np.uint8), scale
    a = np.abs(v)
    step = 2.0 ** (np.floor(np.log2(np.maximum(a, 2.0 ** -6))) - 3)
    r = np.rint(a / step) * step
    e = np.floor(np.log2(np.maximum(r, 2.0 ** -6)))
    code = np.where(r < 2.0 ** -6, r * 2 ** 9, (e + 7) * 8 + (r / 2.0 ** e - 1) * 8).astype(np.int64)
    code |= np.where(np.signbit(v), 128, 0)
    code[bad] = 127
    return code.astype(np.uint8), scale


def decode(q, scale, kind, block_rows=1):
    """The values codes stand for, in 64 bits."""
    if kind == A.CKPT_I8:
        v = q.view(np.int8).astype(np.float64)
        v[v == -128] = np.nan
    else:
        v = E4M3[q]
    return v * spread(np.asarray(scale, np.float64), q.shape, block_rows)


def rounding(kind, y):
    """How far one rounding to `kind` may move each y."""
    return np.maximum(np.abs(y) * HALF[kind], TINY[kind])


def norm_stats(x, eps):
    mean = x.mean(1)
    return mean, 1 / np.sqrt(((x - mean[:, None]) ** 2).mean(1) + eps)


def norm_back(dy, x, w, mean, rstd):
    """(dx, dw, db) of sum(dy * y)."""
    h = (x - mean[:, None]) * rstd[:, None]
    d = dy * w
    dx = rstd[:, None] * (d - d.mean(1, keepdims=True) - h * (d * h).mean(1, keepdims=True))
    return dx, (dy * h).sum(0), dy.sum(0)


_erfc = np.vectorize(math.erfc)


def phi(z):
    return 0.5 * _erfc(-z / math.sqrt(2))


def gelu(z):
    return z * phi(z)


def gelu_grad(z):
    return phi(z) + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
