"""Oracle of the linear layers on 4-bit weights, in 64 bits on the CPU: microscaled blocks of 32 values under a
power of two, E2M1 codes for weights and E4M3 codes for rows, and the product of the two. The reference has no
counterpart. Codes are found as the nearest of all values that a format has, scales by trying them."""
from __future__ import annotations

import torch

F64 = torch.float64
BLOCK = 32
GRID4 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=F64)  # of codes 0..7; 8..15 are negative
GRID8 = torch.tensor([m * 2.0 ** -9 for m in range(8)] +
                     [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1], dtype=F64)  # 0..126


def nearest(v: torch.Tensor, grid: torch.Tensor) -> torch.Tensor:
    """Codes (without sign) of the grid values nearest to |v|, the even code of two as near; past the end, the
    last one."""
    a = v.abs().clamp(max=float(grid[-1]))
    hi = torch.searchsorted(grid, a.contiguous()).clamp(1, len(grid) - 1)
    up, down = grid[hi] - a, a - grid[hi - 1]
    return torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)


def fits(top: torch.Tensor, grid: torch.Tensor) -> torch.Tensor:
    """Whether a largest magnitude does not round past the grid's last value: below the middle between it and the
    value that would follow, or in the middle where the last one is the even one."""
    last = float(grid[-1])
    middle = last + (last - float(grid[-2])) / 2
    return top <= middle if (len(grid) - 1) % 2 == 0 else top < middle


def blocks(x: torch.Tensor) -> torch.Tensor:
    """[n, K] -> [n, blocks, 32] in 64 bits, the last block filled up with zeros."""
    x = torch.nn.functional.pad(x.to(F64), (0, -x.shape[1] % BLOCK))
    return x.view(x.shape[0], -1, BLOCK)


def scale_codes(x: torch.Tensor, grid: torch.Tensor) -> torch.Tensor:
    """Scale codes of blocks [n, b, 32]: the smallest that fits; 255 for a block with an infinity or NaN."""
    top = x.abs().amax(-1)
    code = torch.zeros(top.shape, dtype=torch.int64)
    for c in range(1, 255):  # the first that fits, from the smallest
        code += ~fits(top * 2.0 ** (127 - (c - 1)), grid)
    return torch.where(torch.isfinite(x).all(-1), code, 255)


def scale_values(code: torch.Tensor) -> torch.Tensor:
    v = torch.pow(torch.tensor(2.0, dtype=F64), code.to(F64) - 127)
    return torch.where(code == 255, torch.tensor(float("nan"), dtype=F64), v)


def quant8(x: torch.Tensor):
    """Rows [n, K] (any float type) -> E4M3 codes uint8 [n, Kp] and scale codes uint8 [n, Kp / 32]."""
    b = blocks(x)
    s = scale_codes(b, GRID8)
    v = torch.where((s == 255)[..., None], torch.zeros_like(b), b / scale_values(s)[..., None])
    q = nearest(v, GRID8) + 128 * torch.signbit(v)
    q = torch.where((s == 255)[..., None], 127, q)
    return q.view(len(x), -1).to(torch.uint8), s.to(torch.uint8)


def values8(q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """What codes and scales stand for, [n, Kp]."""
    q, s = q.view(torch.uint8).long(), s.view(torch.uint8).long()
    v = torch.cat([GRID8, torch.tensor([float("nan")], dtype=F64)])[q & 127] * (1 - 2 * (q >> 7))
    return v * scale_values(s).repeat_interleave(BLOCK, 1)


def quant4(w: torch.Tensor):
    """Weight [N, K] -> E2M1 codes uint8 [N, Kp] (one a byte) and scale codes uint8 [N, Kp / 32]."""
    b = blocks(w)
    s = scale_codes(b, GRID4)
    v = torch.where((s == 255)[..., None], torch.zeros_like(b), b / scale_values(s)[..., None])
    q = nearest(v, GRID4) + 8 * torch.signbit(v)
    return q.view(len(w), -1).to(torch.uint8), s.to(torch.uint8)


def values4(q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    q = q.long()
    return GRID4[q & 7] * (1 - 2 * (q >> 3)) * scale_values(s.long()).repeat_interleave(BLOCK, 1)


def unpack4(wq: torch.Tensor, N: int, K: int):
    """Codes and scale codes of a weight's buffer: tiles of 16 rows by 128 values in lane order (lane r + 16 g:
    row r, block g), then the scales of four tiles a dword. Padding rows and blocks are left out."""
    RT, KT = -(-N // 16), -(-K // 128)
    KS, Kb = -(-KT // 4), -(-K // BLOCK)
    raw = wq.cpu()
    body, tail = raw[: RT * KT * 1024], raw[RT * KT * 1024:]
    assert tail.numel() == RT * KS * 256
    body = body.view(RT, KT, 4, 16, 16).permute(0, 3, 1, 2, 4).reshape(RT * 16, KT * 4, 16)
    codes = torch.stack([body & 15, body >> 4], -1).view(RT * 16, KT * 4 * BLOCK)
    scales = tail.view(RT, KS, 4, 16, 4).permute(0, 3, 1, 4, 2).reshape(RT * 16, KS * 16)
    return codes[:N, : Kb * BLOCK], scales[:N, :Kb], codes, scales


def rmsnorm1p(x, delta, w, eps):
    """(bf16(x + delta), the norm of it in 64 bits)."""
    if delta is not None:
        x = (x.float() + delta.float()).to(torch.bfloat16)
    y = x.to(F64)
    return x, y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * (1 + w.to(F64))


def swiglu(gu):
    g, u = gu.to(F64).chunk(2, -1)
    return g / (1 + torch.exp(-g)) * u


def product(x: torch.Tensor, w: torch.Tensor):
    """(x w^T, |x| |w|^T) in 64 bits: the result, and the size of what is summed."""
    return x @ w.T.contiguous(), x.abs() @ w.abs().T.contiguous()
