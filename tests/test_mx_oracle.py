"""CPU self-tests of the microscaled formats' oracle: torch's own E4M3 conversion, the formats' value lists, ties,
and that a scale is the smallest at which nothing rounds past the end."""
import torch

from oracle import mx_oracle as M

F64 = torch.float64


def test_grid8_is_torch_e4m3():
    codes = torch.arange(127, dtype=torch.uint8)
    assert torch.equal(codes.view(torch.float8_e4m3fn).to(F64), M.GRID8)
    x = torch.cat([M.GRID8, (M.GRID8[1:] + M.GRID8[:-1]) / 2, torch.rand(4096, dtype=F64) * 448]).float()
    assert torch.equal(M.nearest(x.to(F64), M.GRID8), x.to(torch.float8_e4m3fn).view(torch.uint8).long())


def test_ties_go_to_the_even_code():
    middle = (M.GRID4[1:] + M.GRID4[:-1]) / 2
    assert M.nearest(middle, M.GRID4).tolist() == [0, 2, 2, 4, 4, 6, 6]


def test_scales_are_the_smallest_that_fit():
    for grid, last, past in ((M.GRID4, 6.0, 7.0), (M.GRID8, 448.0, 464.0)):
        below = torch.nextafter(torch.tensor(past, dtype=F64), torch.tensor(0.0, dtype=F64))
        above = torch.nextafter(torch.tensor(past, dtype=F64), torch.tensor(1e9, dtype=F64))
        for top, want in ((last, 127), (float(below), 127), (float(above), 128), (last / 2, 126), (past, None)):
            x = torch.zeros(1, 1, 32, dtype=F64)
            x[0, 0, 5] = -top
            got = int(M.scale_codes(x, grid))
            assert got == (want if want is not None else (128 if last == 6.0 else 127)), (top, got)


def test_extremes():
    x = torch.zeros(5, 32)
    x[1, 3], x[2, 4], x[3, 5], x[4, 0] = float("inf"), float("nan"), 2.0 ** -149, 3.0e38
    for quant, values in ((M.quant8, M.values8), (M.quant4, M.values4)):
        q, s = quant(x)
        assert s.view(-1)[:4].tolist() == [0, 255, 255, 0]
        v = values(q, s)
        assert torch.isnan(v[1:3]).all() and torch.isfinite(v[[0, 3, 4]]).all()
        assert (v[[0, 3]].abs() <= 2.0 ** -127).all()


def test_layout_round_trip():
    N, K = 19, 600
    RT, KT, KS = 2, 5, 2
    g = torch.Generator().manual_seed(0)
    wq = torch.randint(0, 256, (RT * KT * 1024 + RT * KS * 256,), generator=g).to(torch.uint8)
    codes, scales, _, _ = M.unpack4(wq, N, K)
    assert codes.shape == (19, 608) and scales.shape == (19, 19)
    for row, k in ((0, 0), (3, 31), (15, 128), (16, 599), (18, 300)):
        rt, r, kt, b = row // 16, row % 16, k // 128, k % 128 // 32
        lane = r + 16 * b
        byte = int(wq[(rt * KT + kt) * 1024 + lane * 16 + k % 32 // 2])
        assert int(codes[row, k]) == (byte >> 4 if k % 2 else byte & 15)
        assert int(scales[row, k // 32]) == int(wq[RT * KT * 1024 + (rt * KS + kt // 4) * 256 + lane * 4 + kt % 4])


def test_product_of_codes_is_close_to_the_values():
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(5, 100, generator=g), torch.randn(7, 100, generator=g)
    a, b = M.values8(*M.quant8(x)), M.values4(*M.quant4(w))
    # half a step: 2^-4 and 2^-2 of a value, or of the least normal one under the scale
    assert ((a[:, :100] - x.to(F64)).abs() <= 2.0 ** -4 * x.abs() + 2.0 ** -10 * x.abs().amax()).all()
    assert ((b[:, :100] - w.to(F64)).abs() <= 0.25 * w.abs() + w.abs().amax() / 14).all()
    got, size = M.product(a, b)
    assert ((got - x.to(F64) @ w.to(F64).T).abs() <= 0.5 * size + 1).all()
