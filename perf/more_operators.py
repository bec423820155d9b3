"""Performance cases of the 4-bit linear layers of a step: weights in microscaled 4-bit floating point (E2M1
codes), the 8-bit rows that multiply them (E4M3 codes), made by a norm with the residual's addition, by SwiGLU
or from plain rows, and the product of the two.

Both formats hold blocks of 32 values along a row under one scale, a power of two: the smallest 2^e, e in
[-127, 127], at which the block's largest magnitude does not round past the code's largest (6, or 448). Codes
round to nearest, ties to even. A row's last block is filled up with zeros.

Sizes are those of the repository's benchmark and tests: hidden size 5120, an MLP of 17408, projections of
14336, 6144 and 1024; also odd ones. Each call is one layer's.
"""
from __future__ import annotations

import math

import torch

own = False

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
FP8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
DEV = "cuda"
EPS = 1e-6
MOST = 34816 * 5120          # weights of the largest matrix: an MLP's gate and up together
GRID4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # magnitudes of the E2M1 codes 0..7


def listed():
    return [
        # one token's norm, before every projection of a decode step: latency counts
        dict(name="norm8_1x5120", kind="norm8", rows=1, width=5120, delta=True),
        # the norm of a prompt's chunk
        dict(name="norm8_2048x5120", kind="norm8", rows=2048, width=5120, delta=True),
        # the MLP's activation of a verify pass, and of a prompt's chunk
        dict(name="swiglu8_5x17408", kind="act8", rows=5, width=17408, swiglu=True),
        dict(name="swiglu8_2048x17408", kind="act8", rows=2048, width=17408, swiglu=True),
        # attention outputs of a short prompt, before the output projection
        dict(name="quant8_300x6144", kind="act8", rows=300, width=6144, swiglu=False),
        # loading a model: the smallest weight (a key projection), and the largest one of a layer; a pass
        # quantises and reads the values back
        dict(name="quant4_1024x5120", kind="quant4", out=1024, width=5120),
        dict(name="quant4_34816x5120", kind="quant4", out=34816, width=5120),
        # one token's attention projection: streaming the weights
        dict(name="product_1x14336x5120", kind="product", rows=1, out=14336, width=5120),
        # speculative verify: five rows through the MLP's second matrix, a long sum
        dict(name="product_5x5120x17408", kind="product", rows=5, out=5120, width=17408),
        # a mid-sized batch of tokens on odd sizes: neither streaming nor tiles fit well
        dict(name="product_77x5001x6176", kind="product", rows=77, out=5001, width=6176),
        # a short prompt's output projection
        dict(name="product_300x5120x6144", kind="product", rows=300, out=5120, width=6144),
        # a prompt's chunk through the MLP's gate and up: the large, arithmetic-bound call
        dict(name="product_2048x34816x5120", kind="product", rows=2048, out=34816, width=5120),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["norm8", "norm8", "act8", "act8", "quant4"] + ["product"] * 6)
    if kind == "quant4":
        width = _log(rng, 32, 17408)
        return dict(kind=kind, out=_log(rng, 1, min(34816, MOST // width)), width=width)
    if kind == "product":
        width = 32 * _log(rng, 1, 544)
        out = _log(rng, 16, min(34816, MOST // width))
        return dict(kind=kind, rows=_log(rng, 1, 2048), out=out, width=width)
    rows = _log(rng, 1, 2048)
    width = rng.choice([_log(rng, 16, 17408), 32 * _log(rng, 1, 544)])
    if kind == "act8":
        return dict(kind=kind, rows=rows, width=width, swiglu=rng.choice([True, False]))
    return dict(kind=kind, rows=rows, width=width, delta=rng.choice([True, True, False]))


# ---------------------------------------------------------------------------------- inputs
def _randn(g, *shape, scale=1.0, dtype=BF):
    x = torch.empty(shape, dtype=dtype, device=DEV).normal_(generator=g)
    return x if scale == 1.0 else x.mul_(scale)


def _wide(width):
    return -(-width // 32) * 32


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    kind = case["kind"]
    if kind == "quant4":
        s = dict(case=case, w=_randn(g, case["out"], case["width"], scale=case["width"] ** -0.5),
                 values=torch.empty(case["out"], case["width"], dtype=BF, device=DEV))
        if own:
            import qengine_amd as qa
            s["wq"] = qa.alloc_mx4(case["out"], case["width"])
        return s
    n, K = case["rows"], case["width"]
    if kind == "product":
        N = case["out"]
        w = _randn(g, N, K, scale=K ** -0.5)
        # rows with a few large channels, as a residual stream has them
        x = _randn(g, n, K, dtype=F32) * torch.exp(1.5 * _randn(g, 1, K, dtype=F32).clamp(0))
        xq, xs = _rows8(x)
        s = dict(case=case, xq=xq, xs=xs, out=torch.empty(n, N, dtype=BF, device=DEV))
        if own:
            import qengine_amd as qa
            from qengine_amd import _C
            s["wq"], s["ws"] = qa.alloc_mx4(N, K), qa.alloc_mx4_ws(n, N, K)
            _C.mx4_quant(w, s["wq"])
        else:
            s["codes"], s["scales"] = _codes4(w)
        return s
    q = torch.empty(n, _wide(K), dtype=FP8, device=DEV)
    sc = torch.empty(n, _wide(K) // 32, dtype=E8, device=DEV)
    if kind == "act8":
        return dict(case=case, x=_randn(g, n, K * (2 if case["swiglu"] else 1), scale=2.0), q=q, s=sc)
    return dict(case=case, x=_randn(g, n, K, scale=3.0), w=_randn(g, K, scale=0.3),
                delta=_randn(g, n, K) if case["delta"] else None, sum=torch.empty(n, K, dtype=BF, device=DEV),
                q=q, s=sc)


def _codes4(w):
    """A weight as E2M1 codes, two in a byte (the lower half first), and scale codes: what a checkpoint holds."""
    v, e = _blocks(w.float(), 0.875, 3, False)
    a = v.abs()
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
    code = (code + 8 * (v < 0)).view(w.shape[0], -1, 2)
    return code[..., 0] | code[..., 1] << 4, (e + 127).to(torch.uint8).view(w.shape[0], -1)


# ---------------------------------------------------------------------------------- a pass
def run(s):
    return {"norm8": _norm8, "act8": _act8, "quant4": _quant4, "product": _product}[s["case"]["kind"]](s)


def _norm8(s):
    if own:
        from qengine_amd import _C
        # without a residual there is no sum to write
        _C.rmsnorm1p_mx8(s["x"], s["delta"], s["w"], s["q"], s["s"], EPS,
                         s["sum"] if s["delta"] is not None else None)
        q, sc = s["q"], s["s"]
    else:
        x = s["x"]
        if s["delta"] is not None:
            x = s["sum"].copy_((x.float() + s["delta"].float()).to(BF))
        # in 64 bits: a value next to the border between two codes
        y = x.double()
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * (1 + s["w"].double())
        q, sc = _rows8(y)
    return {"q": q, "s": sc, "sum": s["sum"]} if s["delta"] is not None else {"q": q, "s": sc}


def _act8(s):
    x, K = s["x"], s["case"]["width"]
    if own:
        from qengine_amd import _C
        (_C.swiglu_mx8 if s["case"]["swiglu"] else _C.quant_mx8)(x, s["q"], s["s"])
        return {"q": s["q"], "s": s["s"]}
    if s["case"]["swiglu"]:
        g = x[:, :K].double()
        q, sc = _rows8(g / (1 + torch.exp(-g)) * x[:, K:].double())
    else:
        q, sc = _rows8(x.float())
    return {"q": q, "s": sc}


def _quant4(s):
    if own:
        from qengine_amd import _C
        _C.mx4_quant(s["w"], s["wq"])
        _C.mx4_dequant(s["wq"], s["values"])
        return s["values"]
    v, e = _blocks(s["w"].float(), 0.875, 3, False)
    a = v.abs()
    step = 0.5 + 0.5 * (a >= 2) + (a >= 4)
    q = torch.ldexp(torch.sign(v) * (torch.round(a / step) * step), e)
    return s["values"].copy_(q.view(q.shape[0], -1)[:, :s["w"].shape[1]])


def _product(s):
    if own:
        from qengine_amd import _C
        _C.gemm_mx4(s["wq"], s["xq"], s["xs"], s["out"], s["ws"])
        return s["out"]
    table = torch.tensor(GRID4 + tuple(-x for x in GRID4), dtype=F32, device=DEV)
    n, N, K = s["case"]["rows"], s["case"]["out"], s["case"]["width"]
    w = torch.stack([table[(s["codes"] & 15).int()], table[(s["codes"] >> 4).int()]], -1)
    w = (w.view(N, -1, 32) * torch.exp2(s["scales"].float() - 127).view(N, -1, 1)).view(N, K)
    x = (s["xq"].float().view(n, -1, 32) * s["xs"].float().view(n, -1, 1)).view(n, K)
    return s["out"].copy_(x @ w.T)


def _blocks(x, border, power, low):
    """Blocks of 32 over their scale, [n, blocks, 32], and the scales' exponents, [n, blocks, 1]: the largest
    magnitude m * 2^E, 1/2 <= m < 1, stays below `border` * 2^`power` (with `low`, at it too)."""
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).view(x.shape[0], -1, 32)
    m, E = torch.frexp(x.abs().amax(-1, keepdim=True))
    e = E - power + (m > border if low else m >= border)
    e = torch.where(m == 0, -127, e).clamp(-127, 127)
    return torch.ldexp(x, -e), e


def _rows8(x):
    """Rows as E4M3 codes and their blocks' scales: magnitudes up to 464 round to 448 or below."""
    v, e = _blocks(x, 0.90625, 9, True)
    return v.float().view(x.shape[0], -1).to(FP8), torch.exp2(e.float()).view(x.shape[0], -1).to(E8)


# ---------------------------------------------------------------------------------- floors
def work(case):
    """Bytes and operations that a pass cannot do without."""
    kind, K = case["kind"], case["width"]
    if kind == "quant4":  # the weight, the codes written, the values
        return {"bytes": case["out"] * K * (2 + 17 / 32 + 2), "flops": 0}
    n = case["rows"]
    if kind == "product":
        N = case["out"]
        return {"bytes": N * K * 17 / 32 + n * K * 33 / 32 + n * N * 2, "flops": 2 * n * N * K}
    read = 2 * n * K * ((2 if case["swiglu"] else 1) if kind == "act8" else 1)
    if kind == "norm8" and case["delta"]:
        read += 4 * n * K
    return {"bytes": read + n * K * 33 / 32, "flops": 0}


# ---------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The definition in 64 bits: codes are the nearest of all values that the format has."""
    s = prepare(case, seed)
    kind, K = case["kind"], case["width"]
    if kind == "product":
        n, N = case["rows"], case["out"]
        if own:
            w = _nearest(_again(case, seed), GRID4, 7.0, False)
            w = (w[0] * w[1]).reshape(N, -1)[:, :K]
        else:
            value = torch.tensor(GRID4, dtype=F64, device=DEV)
            halves = [c.long() for c in (s["codes"] % 16, s["codes"] // 16)]
            w = torch.empty(N, K, dtype=F64, device=DEV)
            for i, c in enumerate(halves):
                w[:, i::2] = value[c % 8] * (1 - 2 * (c // 8))
            w *= torch.pow(2.0, s["scales"].double() - 127).repeat_interleave(32, 1)
        x = s["xq"].double() * s["xs"].double().repeat_interleave(32, 1)
        return x @ w.T.contiguous()
    if kind == "quant4":
        v, sc = _nearest(s["w"].double(), GRID4, 7.0, False)
        return (v * sc).reshape(case["out"], -1)[:, :K]
    x = s["x"].double()
    if kind == "norm8":
        if s["delta"] is not None:
            x = (x + s["delta"].double()).to(BF).double()
        y = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / K + EPS)
        y = y + y * s["w"].double()
    else:
        y = x[:, K:] * x[:, :K] * torch.sigmoid(x[:, :K]) if case["swiglu"] else x
    grid = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)]
    v, sc = _nearest(y, grid[:127], 464.0, True)
    got = {"q": v.reshape(len(y), -1), "s": sc.reshape(len(y), -1)}
    return {**got, "sum": x} if kind == "norm8" and s["delta"] is not None else got


def _again(case, seed):
    """The weight of a product's case, as its preparation draws it first."""
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    return _randn(g, case["out"], case["width"], scale=case["width"] ** -0.5).double()


def _nearest(x, grid, limit, at):
    """Values of `grid` nearest to x over its scale, the even one of two as near, and the scales."""
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).view(len(x), -1, 32)
    top = x.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -140) / limit))  # near: corrected by one either way
    for _ in range(2):
        over = top > limit * 2.0 ** e if at else top >= limit * 2.0 ** e
        e = e + over
    under = top <= limit * 2.0 ** (e - 1) if at else top < limit * 2.0 ** (e - 1)
    e = (e - under.double()).clamp(-127, 127)
    grid = torch.tensor(grid, dtype=F64, device=DEV)
    v = x * 2.0 ** -e
    hi = torch.searchsorted(grid, v.abs().contiguous()).clamp(1, len(grid) - 1)
    below, above = v.abs() - grid[hi - 1], grid[hi] - v.abs()
    up = (above < below) | ((above == below) & (hi % 2 == 0))
    return torch.where(up, grid[hi], grid[hi - 1]) * torch.sign(v), 2.0 ** e
