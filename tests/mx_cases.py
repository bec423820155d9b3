"""Shared by the tests of the linear layers on 4-bit weights: inputs, and the checks of rows and products."""
import torch

from oracle import mx_oracle as M

BF, F64, U8 = torch.bfloat16, torch.float64, torch.uint8
FP8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
DEV = "cuda"


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(BF)


def spread(g, n, K):
    """Rows whose blocks differ in size by many powers of two, with zeros and a block of zeros among them."""
    x = torch.randn(n, K, generator=g) * torch.exp2(torch.randint(-12, 12, (n, K), generator=g).float())
    x[torch.rand(n, K, generator=g) < 0.05] = 0
    x[0, 32:64] = 0
    return x.to(BF)


def strided(x, pad, offset=0):
    """x as rows of a wider buffer on the GPU, `offset` values in, the rest NaN."""
    big = torch.full((x.shape[0], x.shape[1] + pad + offset), float("nan"), dtype=x.dtype, device=DEV)
    view = big[:, offset: offset + x.shape[1]]
    view.copy_(x)
    return view


def out8(n, K, pad=0, pads=0):
    """Buffers of 8-bit rows, the bytes around them set, to see that they stay."""
    Kp = -(-K // 32) * 32
    q = torch.full((n, Kp + pad), 0x55, dtype=U8, device=DEV)
    s = torch.full((n, Kp // 32 + pads), 0x55, dtype=U8, device=DEV)
    return q, s, q[:, :Kp], s[:, : Kp // 32]


def check_rows(q, s, y, delta):
    """8-bit rows of the values y (64 bits), which the kernel had up to a relative error `delta`: each scale is the
    oracle's for a value that near to the block's largest, each code is as near to its value as any other, up to
    that error (2 delta: the value's own, and that of the middle between two codes)."""
    q, s = q.cpu(), s.cpu()
    b = M.blocks(y)
    lo, hi = M.scale_codes(b * (1 - delta), M.GRID8), M.scale_codes(b * (1 + delta), M.GRID8)
    got = s.view(U8).long()
    assert ((got >= lo) & (got <= hi)).all()
    v = b / M.scale_values(got)[..., None]
    have = M.values8(q, torch.full_like(s.view(U8), 127)).view(v.shape)
    best = M.GRID8[M.nearest(v, M.GRID8)]
    off = (have - v).abs() - (best - v.abs()).abs()
    assert (off <= 2 * delta * v.abs()).all(), float(off.max())


def check_product(out, x, w, K):
    """out (bf16) against the 64-bit product of the values x and w. Half a bf16 step, 2^-8 of the result. The scaled
    matrix instruction adds the products of eight neighbouring k as whole multiples of 2^(e - 13), e the largest
    sum of two codes' exponents among them (measured on MI355X: beside 2688 - 2688, whose e is 10, each of
    the other six places of its eight keeps 2^-3 and 1.5 * 2^-2, cuts (1 + 7/8) * 2^-3 to 2^-3 and 2^-4 to
    0; other eights keep 2^-10). Cut towards zero, each of at most seven products loses less than 2^-13 of the
    largest of its eight, which itself is whole (its 6 bits). The sums of eights, and what follows, are
    fp32 additions, off by at most 2^-23 of what is summed (a truncated one); no value passes through more of
    them than 16 within an instruction, one for each instruction of its chain (at most K / 128), and 32 partial
    sums."""
    x, w = x.to(DEV), w.to(DEV)
    want, size = M.product(x, w.contiguous())
    eights = torch.zeros_like(want)  # the largest product of every eight k, summed
    xa, wa = x.abs().view(len(x), -1, 8), w.abs().view(len(w), -1, 8)
    for g in range(xa.shape[1]):
        most = torch.zeros_like(want)
        for k in range(8):
            most = torch.maximum(most, xa[:, g, k, None] * wa[:, g, k])
        eights += most
    fine = 7 * 2.0 ** -13 * eights + (K // 128 + 49) * 2.0 ** -23 * size
    bound = 2.0 ** -8 * want.abs() + fine * (1 + 2.0 ** -8) + 1e-37
    diff = (out.to(DEV).to(F64) - want).abs()
    assert (diff <= bound).all(), float((diff / bound).max())


def weight(capi_or_native, w):
    """The 4-bit form of a CPU weight on the GPU, and the values it stands for."""
    import qengine_amd as qa
    wq = qa.alloc_mx4(*w.shape)
    capi_or_native.mx4_quant(w.to(DEV), wq)
    return wq, M.values4(*M.quant4(w))
