"""4-bit weights on the GPU against the oracle: codes, scales and their places bit for bit (the quantisation is exact
arithmetic), values read back, odd sizes and strides, extremes, untouched surroundings."""
import pytest
import torch

import mx_cases as C
from oracle import mx_oracle as M

pytestmark = pytest.mark.gpu
BF, U8, DEV = C.BF, C.U8, C.DEV


@pytest.mark.parametrize("N,K,pad,offset", [
    (16, 512, 0, 0), (1, 1, 0, 0), (1, 32, 0, 0), (17, 40, 0, 0), (33, 129, 0, 0), (5, 1000, 24, 8), (31, 520, 8, 0),
    (3, 2049, 3, 1), (64, 640, 1, 0), (15, 8, 0, 0), (200, 2600, 0, 0), (2, 96, 0, 3),
])
def test_quant_and_back(native, N, K, pad, offset):
    g = C.gen(N * 10007 + K)
    w = C.spread(g, N, max(K, 64))[:, :K].contiguous()
    nb = native.mx4_bytes(N, K)
    buf = torch.full((nb + 256,), 0x55, dtype=U8, device=DEV)
    native.mx4_quant(C.strided(w, pad, offset), buf[:nb])
    codes, scales = M.quant4(w)
    got, sc, all_codes, all_scales = M.unpack4(buf[:nb], N, K)
    assert torch.equal(sc, scales) and torch.equal(got, codes)
    Kb = codes.shape[1]
    assert (all_codes[N:] == 0).all() and (all_codes[:, Kb:] == 0).all()  # padding
    assert (all_scales[N:] == 0).all() and (all_scales[:, Kb // 32:] == 0).all()
    assert (buf[nb:] == 0x55).all()
    big = torch.full((N + 1, K + pad + offset), 7.0, dtype=BF, device=DEV)
    native.mx4_dequant(buf[:nb], big[:N, offset: offset + K])
    want = M.values4(codes, scales)[:, :K].to(BF)
    assert torch.equal(big[:N, offset: offset + K].cpu().view(torch.int16), want.view(torch.int16))
    assert (big[N] == 7).all() and (big[:, :offset] == 7).all() and (big[:, offset + K:] == 7).all()


def test_every_magnitude_and_tie(native):
    """All 32,768 bf16 magnitudes with both signs, each in a block of its own and in one beside 1.0: rounding, ties,
    the scale's borders, subnormals, infinities and NaN."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    x = bits.view(BF)
    w = torch.zeros(65536, 64, dtype=BF)
    w[:, 5] = x
    w[:, 32] = 1.0
    w[:, 50] = x
    w = w.to(DEV)
    wq = torch.empty(native.mx4_bytes(65536, 64), dtype=U8, device=DEV)
    native.mx4_quant(w, wq)
    codes, scales = M.quant4(w.cpu())
    got, sc, _, _ = M.unpack4(wq, 65536, 64)
    assert torch.equal(sc, scales)
    assert torch.equal(got, codes)
    out = torch.empty_like(w)
    native.mx4_dequant(wq, out)
    want = M.values4(codes, scales).to(BF)
    out = out.cpu()
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(out), torch.nan_to_num(want))


def test_large_weight_offsets(native):
    """A weight whose source passes 2^32 bytes: its last rows."""
    N, K = 140000, 16384
    w = torch.zeros(N, K, dtype=BF, device=DEV)
    g = C.gen(3)
    tail = C.randn(g, 3, K)
    w[-3:].copy_(tail)
    wq = torch.empty(native.mx4_bytes(N, K), dtype=U8, device=DEV)
    native.mx4_quant(w, wq)
    w.fill_(1.0)
    native.mx4_dequant(wq, w)
    assert torch.equal(w[-3:].cpu(), M.values4(*M.quant4(tail)).to(BF))
    assert (w[: N - 3] == 0).all()
