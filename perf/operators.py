"""The training operators around an adapted projection, as they are measured.

Layer norm with the gradient of its weight and bias, activation checkpoints in 8 bits (stored,
loaded, and read by the backward passes of layer norm, GELU and an adapter's rank product) and
the product of two 8-bit floating-point matrices with a scale for each block of 128.

An 8-bit tensor here is codes and scales.  A block is 128 neighbouring columns of one row (or of
128 rows, for a weight) and has one scale, the smallest power of two s with max|x| <= top * s
(top: 448 for e4m3, 127 for whole numbers; s >= 2^-126).  A code is x / s rounded to nearest even.
Dividing by a power of two is exact, so code and scale follow from x alone.
Scales lie block-major: [ceil(cols / 128)][rows].
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
FORMATS = {"i8": (127.0, 7, 127.0 / 128.0), "e4m3": (448.0, 9, 0.875)}  # top = mantissa * 2^exponent
EPS = 1e-5


def _lib():
    """The framework's binding; its folder is no package name, so it goes on the path."""
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "audiocraft.cpp_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import actrain
    return actrain


# --------------------------------------------------------------------------------------- cases
def listed():
    ln, ck, ge, ra, ge8 = "layernorm", "ckpt8", "gelu", "rank_gemm", "gemm_f8"
    return [
        # one token of each of 4 sequences through a 1536-wide norm: latency only
        dict(name="ln fwd 4x1536 f16", op=ln, rows=4, cols=1536, xt="f16", yt="f16", fmt="", back=False, out8=False),
        # the norms of one 30 s clip at an odd length, trained, with the input kept as it is
        dict(name="ln step 749x1024 f32", op=ln, rows=749, cols=1024, xt="f32", yt="f16", fmt="", back=True, out8=False),
        # a batch of 16 x 1500 frames with the input kept in 8 bits until the backward pass
        dict(name="ln step 24000x1536 bf16 i8", op=ln, rows=24000, cols=1536, xt="bf16", yt="bf16", fmt="i8", back=True,
             out8=False),
        # an activation put away in 8 bits and brought back, at a width that ends inside a block
        dict(name="ckpt8 1501x1000 f32 i8", op=ck, rows=1501, cols=1000, xt="f32", yt="f32", fmt="i8", block=1),
        # a frozen weight laid out for the 8-bit product in blocks of 128 x 128, and back
        dict(name="ckpt8 6144x1536 f32 e4m3 b128", op=ck, rows=6144, cols=1536, xt="f32", yt="bf16", fmt="e4m3",
             block=128),
        # the feed-forward activation of 8 clips, its result also as the next product's operand
        dict(name="gelu step 6000x4096 f16 i8 +8", op=ge, rows=6000, cols=4096, xt="f16", fmt="i8", out8=True),
        # the same for 8 x 1500 frames of the wider model
        dict(name="gelu step 12000x6144 bf16 e4m3", op=ge, rows=12000, cols=6144, xt="bf16", fmt="e4m3", out8=False),
        # gradient of a rank-16 adapter from the kept input of 8 clips
        dict(name="rank 6000x1024 r16 f16 e4m3", op=ra, rows=6000, cols=1024, nb=16, ut="f16", fmt="e4m3"),
        # the largest rank on the widest activation, fp32 gradients of U
        dict(name="rank 24000x6144 r64 f32 i8", op=ra, rows=24000, cols=6144, nb=64, ut="f32", fmt="i8"),
        # one token of each of 4 sequences through a projection: the weight is read once
        dict(name="gemm 4x6144x1536 f16", op=ge8, rows=4, n=6144, k=1536, yt="f16", mn=False, bias=True),
        # one clip at an odd length and sizes that end inside tiles
        dict(name="gemm 749x4104x1000 f32", op=ge8, rows=749, n=4104, k=1000, yt="f32", mn=False, bias=False),
        # input gradient of the wider model's feed-forward projection over 16 x 1500 frames
        dict(name="gemm 24000x1536x6144 bf16 mn", op=ge8, rows=24000, n=1536, k=6144, yt="bf16", mn=True, bias=False),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layernorm", "ckpt8", "gelu", "rank_gemm", "gemm_f8"])
    kind = lambda: rng.choice(sorted(DTYPES))  # noqa: E731
    if op == "layernorm":
        back = rng.random() < 0.7
        rows, cols = _between(rng, 1, 24000), _between(rng, 8, 8192)
        rows = max(1, min(rows, 24000 * 1536 // cols))
        return dict(op=op, rows=rows, cols=cols, xt=kind(), yt=kind(), fmt=rng.choice(["", "i8", "e4m3"]), back=back,
                    out8=rng.random() < 0.3)
    if op == "ckpt8":
        rows, cols = _between(rng, 1, 24000), _between(rng, 1, 8192)
        rows = max(1, min(rows, 36000000 // cols))
        return dict(op=op, rows=rows, cols=cols, xt=kind(), yt=rng.choice(["f32", "bf16"]),
                    fmt=rng.choice(["i8", "e4m3"]), block=rng.choice([1, 1, 128]))
    if op == "gelu":
        rows, cols = _between(rng, 1, 24000), _between(rng, 1, 8192)
        rows = max(1, min(rows, 36000000 // cols))
        return dict(op=op, rows=rows, cols=cols, xt=kind(), fmt=rng.choice(["i8", "e4m3"]), out8=rng.random() < 0.4)
    if op == "rank_gemm":
        rows, cols = _between(rng, 1, 24000), _between(rng, 16, 6144)
        return dict(op=op, rows=rows, cols=cols, nb=_between(rng, 1, 64), ut=kind(), fmt=rng.choice(["i8", "e4m3"]))
    rows, n, k = _between(rng, 1, 24000), _between(rng, 16, 6144), _between(rng, 16, 6144)
    rows = max(1, min(rows, 24000 * 1536 * 6144 // (n * k)))
    return dict(op=op, rows=rows, n=n, k=k, yt=kind(), mn=rng.random() < 0.4, bias=rng.random() < 0.5)


def work(case):
    op, rows = case["op"], case["rows"]
    if op == "gemm_f8":
        n, k = case["n"], case["k"]
        scales = 4 * (rows * -(-k // 128) + -(-n // 128) * -(-k // 128))
        return {"bytes": rows * k + n * k + scales + rows * n * BYTES[case["yt"]] + (4 * n if case["bias"] else 0),
                "flops": 2 * rows * n * k}
    cols = case["cols"]
    eight = rows * cols + 4 * rows * -(-cols // 128)  # codes and scales
    if op == "layernorm":
        x, y = rows * cols * BYTES[case["xt"]], rows * cols * BYTES[case["yt"]]
        total, flops = x + y + 8 * rows + 8 * cols, 8 * rows * cols
        total += eight if case["out8"] else 0
        if case["fmt"]:
            total += eight
        if case["back"]:  # dy and the kept input in, dx and the two sums over the rows out
            total += y + (eight if case["fmt"] else x) + x + 8 * rows + 12 * cols
            flops += 12 * rows * cols
        return {"bytes": total, "flops": flops}
    if op == "ckpt8":
        if case["block"] == 128:
            eight = rows * cols + 4 * -(-rows // 128) * -(-cols // 128)
        return {"bytes": rows * cols * (BYTES[case["xt"]] + BYTES[case["yt"]]) + 2 * eight, "flops": 4 * rows * cols}
    if op == "gelu":
        return {"bytes": 4 * rows * cols * BYTES[case["xt"]] + 2 * eight + (eight if case["out8"] else 0),
                "flops": 60 * rows * cols}
    return {"bytes": eight + rows * case["nb"] * BYTES[case["ut"]] + 4 * case["nb"] * cols,
            "flops": 2 * rows * cols * case["nb"]}


# --------------------------------------------------------------------------------- 8-bit tensors
def _power(e):
    """2^e in 32 bits for whole e in [-126, 127], exactly."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _store(x, fmt, block):
    """x [rows][cols] in 32 bits -> codes and the block-major scales."""
    rows, cols = x.shape
    _, exponent, mantissa = FORMATS[fmt]
    nb, nr = -(-cols // 128), -(-rows // block)
    padded = torch.zeros(nr * block, nb * 128, device=x.device)
    padded[:rows, :cols] = x
    blocks = padded.view(nr, block, nb, 128)
    top = blocks.abs().amax(dim=(1, 3))
    m, e = torch.frexp(top)
    e = (e.to(torch.int32) - exponent + (m > mantissa).to(torch.int32)).clamp(min=-126)
    e = torch.where(top == 0, torch.full_like(e, -126), e)
    q = (blocks * _power(-e)[:, None, :, None]).view(nr * block, nb * 128)[:rows, :cols]
    q = q.to(torch.float8_e4m3fn) if fmt == "e4m3" else torch.round(q).to(torch.int8)
    return q, _power(e).t().contiguous()


def _load(q, scale, block):
    """Codes and scales -> the values they stand for, in 32 bits (exact)."""
    rows, cols = q.shape
    s = scale.t().repeat_interleave(block, 0)[:rows].repeat_interleave(128, 1)[:, :cols]
    return q.float() * s


def _pitched(q):
    """The codes with rows that start on 16-byte boundaries, as the products want their operands."""
    rows, cols = q.shape
    held = torch.zeros(rows, -(-cols // 16) * 16, dtype=torch.uint8, device=q.device)
    held[:, :cols] = q.view(torch.uint8)
    return held


def _values(held, fmt, cols):
    return held.view(torch.float8_e4m3fn if fmt == "e4m3" else torch.int8)[:, :cols]


# -------------------------------------------------------------------------------------- inputs
def _activation(gen, rows, cols):
    """A residual stream's values: columns of different size, a few far larger, an offset per row."""
    x = torch.randn(rows, cols, device="cuda", generator=gen)
    size = torch.exp(0.5 * torch.randn(cols, device="cuda", generator=gen))
    size = torch.where(torch.rand(cols, device="cuda", generator=gen) < 0.01, size * 12, size)
    return x * size + 0.3 * torch.randn(rows, 1, device="cuda", generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    rows, op = case["rows"], case["op"]
    rand = lambda *n: torch.randn(*n, device="cuda", generator=gen)  # noqa: E731
    s = dict(case=case)
    if op == "layernorm":
        cols = case["cols"]
        s["x"] = _activation(gen, rows, cols).to(DTYPES[case["xt"]])
        s["w"], s["b"] = 1 + 0.2 * rand(cols), 0.2 * rand(cols)
        s["dy"] = (0.1 * rand(rows, cols)).to(DTYPES[case["yt"]])
    elif op == "ckpt8":
        x = 0.02 * rand(rows, case["cols"]) if case["block"] == 128 else _activation(gen, rows, case["cols"])
        s["x"] = x.to(DTYPES[case["xt"]])
    elif op == "gelu":
        s["z"] = (1.5 * _activation(gen, rows, case["cols"])).to(DTYPES[case["xt"]])
        s["dg"] = (0.1 * rand(rows, case["cols"])).to(DTYPES[case["xt"]])
    elif op == "rank_gemm":
        q, scale = _store(_activation(gen, rows, case["cols"]), case["fmt"], 1)
        s["q"], s["scale"] = _pitched(q), scale
        s["u"] = (0.1 * rand(rows, case["nb"])).to(DTYPES[case["ut"]])
        s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    else:
        n, k = case["n"], case["k"]
        q, s["xs"] = _store(_activation(gen, rows, k), "e4m3", 1)
        s["xq"] = _pitched(q)
        w, s["ws"] = _store(0.02 * rand(*((k, n) if case["mn"] else (n, k))), "e4m3", 128)
        s["wq"] = _pitched(w)
        s["bias"] = 0.1 * rand(n) if case["bias"] else None
        s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    return s


# ---------------------------------------------------------------------------------- plain forms
def _plain_layernorm(s):
    c, x = s["case"], s["x"].float()
    mean = x.mean(1)
    rstd = 1 / torch.sqrt((x - mean[:, None]).square().mean(1) + EPS)
    y = (x - mean[:, None]) * rstd[:, None] * s["w"] + s["b"]
    out = dict(y=y.to(DTYPES[c["yt"]]), mean=mean, rstd=rstd)
    if c["out8"]:
        out["y8"] = _load(*_store(y, "e4m3", 1), 1).to(torch.bfloat16)
    kept = _store(x, c["fmt"], 1) if c["fmt"] else None
    if not c["back"]:
        if kept:
            out["x8"] = _load(*kept, 1).to(torch.bfloat16)
        return out
    x = _load(*kept, 1) if kept else x
    dy = s["dy"].float()
    xhat = (x - mean[:, None]) * rstd[:, None]
    dxhat = dy * s["w"]
    dx = rstd[:, None] * (dxhat - dxhat.mean(1, keepdim=True) - xhat * (dxhat * xhat).mean(1, keepdim=True))
    out.update(dx=dx.to(DTYPES[c["xt"]]), dw=(dy * xhat).sum(0), db=dy.sum(0))
    return out


def _plain_gelu(s):
    c, z = s["case"], s["z"].float()
    kind = DTYPES[c["xt"]]
    g = z * 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
    out = dict(g=g.to(kind))
    if c["out8"]:
        out["g8"] = _load(*_store(g, "e4m3", 1), 1).to(torch.bfloat16)
    z = _load(*_store(z, c["fmt"], 1), 1)
    slope = 0.5 * torch.special.erfc(-z * math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    out["dz"] = (s["dg"].float() * slope).to(kind)
    return out


def _plain(s):
    c, op = s["case"], s["case"]["op"]
    if op == "layernorm":
        return _plain_layernorm(s)
    if op == "gelu":
        return _plain_gelu(s)
    if op == "ckpt8":
        q, scale = _store(s["x"].float(), c["fmt"], c["block"])
        return dict(y=_load(q, scale, c["block"]).to(DTYPES[c["yt"]]), scale=scale)
    if op == "rank_gemm":
        x = _load(_values(s["q"], c["fmt"], c["cols"]), s["scale"], 1)
        return dict(c=0.5 * (s["u"].float().t() @ x))
    x = _load(_values(s["xq"], "e4m3", c["k"]), s["xs"], 1)
    w = _load(_values(s["wq"], "e4m3", c["n"] if c["mn"] else c["k"]), s["ws"], 128)
    y = x @ (w if c["mn"] else w.t())
    if c["bias"]:
        y = y + s["bias"]
    return dict(y=y.to(DTYPES[c["yt"]]))


# ------------------------------------------------------------------------------ framework's calls
def _new8(A, rows, cols, fmt, block=1):
    """Room for an 8-bit tensor and the binding's view of it."""
    q = torch.empty(rows, -(-cols // 16) * 16, dtype=torch.uint8, device="cuda")
    scale = torch.empty(-(-cols // 128), -(-rows // block), device="cuda")
    return q, scale, _view8(A, q, scale, fmt)


def _view8(A, q, scale, fmt):
    return A.ckpt8(A.CKPT_E4M3 if fmt == "e4m3" else A.CKPT_I8, q.data_ptr(), q.shape[1], scale.data_ptr(),
                   scale.shape[1])


def _loaded(A, view, rows, cols, stream, kind="bf16", block=1):
    y = torch.empty(rows, cols, dtype=DTYPES[kind], device="cuda")
    A.ckpt8_load(view, rows, cols, y.data_ptr(), _kind(A, kind), block_rows=block, stream=stream)
    return y


def _kind(A, name):
    return {"f32": A.TYPE_F32, "f16": A.TYPE_F16, "bf16": A.TYPE_BF16}[name]


def _own_layernorm(A, s, stream):
    c = s["case"]
    rows, cols, xt, yt = c["rows"], c["cols"], _kind(A, c["xt"]), _kind(A, c["yt"])
    y = torch.empty(rows, cols, dtype=DTYPES[c["yt"]], device="cuda")
    stats = torch.empty(2, rows, device="cuda")
    mean, rstd = stats[0], stats[1]
    out = dict(y=y, mean=mean, rstd=rstd)
    y8 = _new8(A, rows, cols, "e4m3") if c["out8"] else None
    x8 = _new8(A, rows, cols, c["fmt"]) if c["fmt"] else None
    A.layernorm_fwd(s["x"].data_ptr(), xt, rows, cols, s["w"].data_ptr(), s["b"].data_ptr(), y.data_ptr(), yt,
                    mean.data_ptr(), rstd.data_ptr(), eps=EPS, y8=y8 and y8[2], x8=x8 and x8[2], stream=stream)
    if y8:
        out["y8"] = _loaded(A, y8[2], rows, cols, stream)
    if not c["back"]:
        if x8:
            out["x8"] = _loaded(A, x8[2], rows, cols, stream)
        return out
    dx = torch.empty(rows, cols, dtype=DTYPES[c["xt"]], device="cuda")
    sums = torch.empty(2, cols, device="cuda")
    room = A.layernorm_bwd_workspace(rows, cols)
    space = torch.empty(room, dtype=torch.uint8, device="cuda")
    A.layernorm_bwd(s["dy"].data_ptr(), yt, 0 if x8 else s["x"].data_ptr(), xt, s["w"].data_ptr(), mean.data_ptr(),
                    rstd.data_ptr(), rows, cols, dx.data_ptr(), xt, sums[0].data_ptr(), sums[1].data_ptr(),
                    space.data_ptr(), room, x8=x8 and x8[2], stream=stream)
    out.update(dx=dx, dw=sums[0], db=sums[1])
    return out


def _own_gelu(A, s, stream):
    c = s["case"]
    rows, cols, kind = c["rows"], c["cols"], _kind(A, c["xt"])
    g = torch.empty(rows, cols, dtype=DTYPES[c["xt"]], device="cuda")
    z8 = _new8(A, rows, cols, c["fmt"])
    g8 = _new8(A, rows, cols, "e4m3") if c["out8"] else None
    A.gelu_ckpt8_fwd(s["z"].data_ptr(), kind, rows, cols, g.data_ptr(), kind, z8[2], g8=g8 and g8[2], stream=stream)
    out = dict(g=g)
    if g8:
        out["g8"] = _loaded(A, g8[2], rows, cols, stream)
    dz = torch.empty_like(g)
    A.gelu_ckpt8_bwd(s["dg"].data_ptr(), kind, z8[2], rows, cols, dz.data_ptr(), kind, stream=stream)
    out["dz"] = dz
    return out


def _own(s):
    A = _lib()
    stream = torch.cuda.current_stream().cuda_stream
    c, op, rows = s["case"], s["case"]["op"], s["case"]["rows"]
    if op == "layernorm":
        return _own_layernorm(A, s, stream)
    if op == "gelu":
        return _own_gelu(A, s, stream)
    if op == "ckpt8":
        q, scale, view = _new8(A, rows, c["cols"], c["fmt"], c["block"])
        A.ckpt8_store(s["x"].data_ptr(), _kind(A, c["xt"]), rows, c["cols"], view, block_rows=c["block"], stream=stream)
        return dict(y=_loaded(A, view, rows, c["cols"], stream, c["yt"], c["block"]), scale=scale)
    if op == "rank_gemm":
        out = torch.empty(c["nb"], c["cols"], device="cuda")
        A.rank_gemm_ckpt8(s["u"].data_ptr(), _kind(A, c["ut"]), c["nb"], _view8(A, s["q"], s["scale"], c["fmt"]), rows,
                          c["cols"], out.data_ptr(), s["status"].data_ptr(), alpha=0.5, stream=stream)
        return dict(c=out)
    y = torch.empty(rows, c["n"], dtype=DTYPES[c["yt"]], device="cuda")
    A.gemm_f8(_view8(A, s["xq"], s["xs"], "e4m3"), _view8(A, s["wq"], s["ws"], "e4m3"), rows, c["n"], c["k"],
              y.data_ptr(), _kind(A, c["yt"]), s["status"].data_ptr(), w_mn_major=c["mn"],
              bias=s["bias"].data_ptr() if c["bias"] else 0, stream=stream)
    return dict(y=y)


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ------------------------------------------------------------------------------ the definition
def _exact8(x, fmt, block):
    """What codes and scales stand for, of x in 64 bits: x / s rounded to the format's steps, times s."""
    top = FORMATS[fmt][0]
    rows, cols = x.shape
    nb, nr = -(-cols // 128), -(-rows // block)
    wide = torch.zeros(nr * block, nb * 128, dtype=torch.float64, device=x.device)
    wide[:rows, :cols] = x
    most = wide.view(nr, block, nb, 128).abs().amax(dim=(1, 3))
    e = torch.ceil(torch.log2(most.clamp(min=2.0 ** -140) / top))
    for _ in range(2):  # log2 may be off by a rounding next to a border
        e = torch.where(most > top * torch.exp2(e), e + 1, e)
        e = torch.where(most <= top * torch.exp2(e - 1), e - 1, e)
    scale = torch.exp2(e.clamp(min=-126))
    s = scale.repeat_interleave(block, 0)[:rows].repeat_interleave(128, 1)[:, :cols]
    v = x / s
    if fmt == "i8":
        step = torch.ones_like(v)
    else:  # steps of 2^-3 of the binade, and of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step * s, scale.t().contiguous()


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "layernorm":
        x = s["x"].double()
        w, b, n = s["w"].double(), s["b"].double(), case["cols"]
        mean = x.sum(1, keepdim=True) / n
        var = (x - mean).pow(2).sum(1, keepdim=True) / n
        rstd = (var + EPS).rsqrt()
        # y8 is rounded to 8 bits from computed values: next to a border either neighbour is right
        out = dict(y=(x - mean) * rstd * w + b, mean=mean[:, 0], rstd=rstd[:, 0])
        if case["out8"]:
            out["y8"] = None
        if not case["back"]:
            if case["fmt"]:
                out["x8"] = _exact8(x, case["fmt"], 1)[0]
            return out
        if case["fmt"]:
            x = _exact8(x, case["fmt"], 1)[0]
        h, dy = (x - mean) * rstd, s["dy"].double()
        dh = dy * w
        out["dx"] = (dh - dh.sum(1, keepdim=True) / n - h * (dh * h).sum(1, keepdim=True) / n) * rstd
        out["dw"], out["db"] = (dy * h).sum(0), dy.sum(0)
        return out
    if op == "ckpt8":
        y, scale = _exact8(s["x"].double(), case["fmt"], case["block"])
        return dict(y=y, scale=scale)
    if op == "gelu":
        z = s["z"].double()
        out = dict(g=z * torch.special.ndtr(z))
        if case["out8"]:
            out["g8"] = None  # rounded to 8 bits from computed values
        z = _exact8(z, case["fmt"], 1)[0]
        density = torch.exp(-z.pow(2) / 2) / math.sqrt(2 * math.pi)
        out["dz"] = s["dg"].double() * (torch.special.ndtr(z) + z * density)
        return out

    def dense(held, fmt, scale, cols, block):
        q = _values(held, fmt, cols).to(torch.float32).double()
        at = torch.arange(q.shape[0], device=q.device) // block
        return q * scale.double()[:, at].t()[:, torch.arange(cols, device=q.device) // 128]

    if op == "rank_gemm":
        x = dense(s["q"], case["fmt"], s["scale"], case["cols"], 1)
        return dict(c=0.5 * torch.einsum("tr,tc->rc", s["u"].double(), x))
    x = dense(s["xq"], "e4m3", s["xs"], case["k"], 1)
    w = dense(s["wq"], "e4m3", s["ws"], case["n"] if case["mn"] else case["k"], 128)
    y = torch.einsum("mk,kn->mn" if case["mn"] else "mk,nk->mn", x, w)
    return dict(y=y + s["bias"].double() if case["bias"] else y)
