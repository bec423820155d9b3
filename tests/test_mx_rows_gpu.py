"""8-bit rows on the GPU against the 64-bit oracle: plain rows bit for bit, SwiGLU and the norm within their fp32
arithmetic, odd widths, strides and alignments, rows that hold infinities or NaN, untouched surroundings, rows
that do not depend on the others."""
import pytest
import torch

import mx_cases as C
from oracle import mx_oracle as M

pytestmark = pytest.mark.gpu
BF, F64, U8, DEV = C.BF, C.F64, C.U8, C.DEV

# (rows, width, pad of the source's rows, its offset, pad of the code rows, of the scale rows)
SHAPES = [(1, 32, 0, 0, 0, 0), (3, 1, 0, 0, 0, 0), (2, 33, 0, 0, 0, 0), (5, 5120, 0, 0, 0, 0), (4, 40, 8, 8, 16, 3),
          (7, 1000, 0, 0, 32, 0), (2, 1001, 6, 1, 0, 1), (3, 2056, 5, 0, 0, 0), (2, 8200, 0, 0, 0, 0),
          (1, 17408, 8, 0, 0, 0), (2, 40000, 0, 0, 0, 0), (300, 96, 0, 0, 0, 0), (2, 32776, 0, 0, 0, 0)]


def around(q_all, s_all, q, s):
    """The bytes beside the rows are as they were."""
    assert (q_all[:, q.shape[1]:] == 0x55).all() and (s_all[:, s.shape[1]:] == 0x55).all()


@pytest.mark.parametrize("n,K,pad,offset,padq,pads", SHAPES)
def test_plain_rows(native, n, K, pad, offset, padq, pads):
    x = C.spread(C.gen(K + n), n, max(K, 64))[:, :K].contiguous()
    qa, sa, q, s = C.out8(n, K, padq, pads)
    native.quant_mx8(C.strided(x, pad, offset), q, s)
    want_q, want_s = M.quant8(x)
    assert torch.equal(s.cpu(), want_s) and torch.equal(q.cpu(), want_q)
    around(qa, sa, q, s)


def test_every_magnitude_and_tie(native):
    """All bf16 values, each in a block of its own and beside 1.0."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF)
    rows = torch.zeros(65536, 64, dtype=BF)
    rows[:, 5], rows[:, 32], rows[:, 50] = x, 1.0, x
    _, _, q, s = C.out8(65536, 64)
    native.quant_mx8(rows.to(DEV), q, s)
    want_q, want_s = M.quant8(rows)
    assert torch.equal(s.cpu(), want_s)
    assert torch.equal(q.cpu(), want_q)


@pytest.mark.parametrize("n,K,pad,offset,padq,pads", SHAPES)
def test_swiglu(native, n, K, pad, offset, padq, pads):
    g = C.gen(K * 3 + n)
    gu = C.randn(g, n, 2 * K, scale=3.0)
    qa, sa, q, s = C.out8(n, K, padq, pads)
    native.swiglu_mx8(C.strided(gu, pad, offset), q, s)
    # the exponential's argument is rounded twice (2^-23 of |log2(e) g|, times ln 2), the instruction and the
    # reciprocal are off by 1 ulp each, and there are a sum and two products
    y = M.swiglu(gu)
    delta = float(gu[:, :K].float().abs().max()) * 2.0 ** -23 + 8 * 2.0 ** -23
    C.check_rows(q, s, y, delta)
    around(qa, sa, q, s)


@pytest.mark.parametrize("how", ["alone", "delta", "sum"])
@pytest.mark.parametrize("n,K,pad,offset,padq,pads", SHAPES)
def test_norm(native, n, K, pad, offset, padq, pads, how):
    g = C.gen(K * 7 + n)
    x, d, w = C.randn(g, n, K, scale=3.0), C.randn(g, n, K), C.randn(g, K, scale=0.3)
    xd = C.strided(x, pad, offset)
    before = xd.clone()
    dd = C.strided(d, pad, offset) if how != "alone" else None
    total = C.strided(torch.zeros_like(x), pad, offset) if how == "sum" else None
    qa, sa, q, s = C.out8(n, K, padq, pads)
    native.rmsnorm1p_mx8(xd, dd, w.to(DEV), q, s, 1e-6, total)
    want, y = M.rmsnorm1p(x, d if how != "alone" else None, w, 1e-6)
    got = total if how == "sum" else xd
    assert torch.equal(got.cpu(), want)
    if how != "delta":
        assert torch.equal(xd, before)
    # the sum of squares: no value passes through more than 40 additions and a product (relative 2^-24 each, all
    # positive), half of that in the root; then a quotient, two roots' roundings, 1 + w and two products
    C.check_rows(q, s, y, (41 / 2 + 8) * 2.0 ** -24)
    around(qa, sa, q, s)


def test_norm_sum_may_be_delta(native):
    g = C.gen(5)
    x, d, w = C.randn(g, 3, 1000), C.randn(g, 3, 1000), C.randn(g, 1000)
    for width in (1000, 997):  # both kernels
        dd = d.to(DEV)[:, :width]
        _, _, q, s = C.out8(3, width)
        native.rmsnorm1p_mx8(x.to(DEV)[:, :width], dd, w.to(DEV)[:width].clone(), q, s, 1e-6, dd)
        want, y = M.rmsnorm1p(x[:, :width], d[:, :width], w[:width], 1e-6)
        assert torch.equal(dd.cpu(), want)
        C.check_rows(q, s, y, 29 * 2.0 ** -24)


@pytest.mark.parametrize("K", [512, 501])
def test_non_finite_rows(native, K):
    """A block with an infinity or NaN is NaN, and no other block or row; a norm's row is NaN with it."""
    g = C.gen(K)
    x = C.randn(g, 4, K)
    x[1, 40], x[2, 100] = float("inf"), float("nan")
    _, _, q, s = C.out8(4, K)
    native.quant_mx8(x.to(DEV), q, s)
    want_q, want_s = M.quant8(x)
    assert torch.equal(s.cpu(), want_s) and torch.equal(q.cpu(), want_q) and int((s == 255).sum()) == 2
    gu = torch.cat([x, C.randn(g, 4, K)], 1)
    native.swiglu_mx8(gu.to(DEV), q, s)
    want = (~torch.isfinite(M.blocks(M.swiglu(gu)))).any(-1)
    assert torch.equal(s.cpu() == 255, want)
    native.rmsnorm1p_mx8(x.to(DEV), None, torch.zeros(K, dtype=BF, device=DEV), q, s, 1e-6)
    # an infinity's row: inf * 0 is NaN at its place, zeros elsewhere
    bad = s.cpu() == 255
    assert not bad[0].any() and not bad[3].any() and bad[2].all() and bad[1].nonzero().view(-1).tolist() == [1]


@pytest.mark.parametrize("K", [5120, 1003])
def test_rows_do_not_depend_on_others(native, K):
    g = C.gen(K + 1)
    x, d, w = (C.randn(g, 6, K).to(DEV), C.randn(g, 6, K).to(DEV), C.randn(g, K).to(DEV))
    for op in ("quant", "glu", "norm"):
        def run(a, b):
            _, _, q, s = C.out8(len(a), K)
            if op == "quant":
                native.quant_mx8(a, q, s)
            elif op == "glu":
                native.swiglu_mx8(torch.cat([a, b], 1), q, s)
            else:
                native.rmsnorm1p_mx8(a.clone(), b, w, q, s, 1e-6)
            return q, s
        q, s = run(x, d)
        for r in (0, 3, 5):
            q1, s1 = run(x[r: r + 1], d[r: r + 1])
            assert torch.equal(q[r], q1[0]) and torch.equal(s[r], s1[0])


def test_more_rows_than_a_launch_has(native):
    """Rows past 2^21 equal the same rows in a call of their own."""
    n, K = (1 << 21) + 5, 32
    g = C.gen(4)
    tail = torch.randn(9, 2 * K, generator=g).to(BF).to(DEV)
    x = torch.zeros(n, 2 * K, dtype=BF, device=DEV)
    x[-9:] = tail
    w, d = torch.randn(K, generator=g).to(BF).to(DEV), torch.randn(9, K, generator=g).to(BF).to(DEV)
    big, small = (tuple(torch.full((m, k), 0x55, dtype=U8, device=DEV) for k in (K, 1)) for m in (n, 9))
    native.swiglu_mx8(x, *big)
    native.swiglu_mx8(tail, *small)
    assert torch.equal(big[0][-9:], small[0]) and torch.equal(big[1][-9:], small[1]) and not big[0][:-9].any()
    native.quant_mx8(x[:, :K], *big)
    native.quant_mx8(tail[:, :K], *small)
    assert torch.equal(big[0][-9:], small[0]) and torch.equal(big[1][-9:], small[1])
    delta = torch.zeros(n, K, dtype=BF, device=DEV)
    delta[-9:] = d
    sums = torch.empty(n, K, dtype=BF, device=DEV), torch.empty(9, K, dtype=BF, device=DEV)
    native.rmsnorm1p_mx8(x[:, :K], delta, w, *big, 1e-6, sums[0])
    native.rmsnorm1p_mx8(tail[:, :K], d, w, *small, 1e-6, sums[1])
    assert torch.equal(big[0][-9:], small[0]) and torch.equal(big[1][-9:], small[1])
    assert torch.equal(sums[0][-9:], sums[1]) and not sums[0][:-9].any()


@pytest.mark.parametrize("K", [4096, 4091])
def test_swiglu_far_gates(native, K):
    """Gates down to -180, where e^g leaves fp32's range and silu(g) * u need not, and the largest ones; the block's
    values are all of one gate's size, or beside ordinary ones."""
    g = C.gen(K)
    gate = torch.linspace(-180.0, -50.0, K).repeat(8, 1)  # a block's gates are within 1.1 of each other
    up = torch.tensor([1.0, -3e2, 1e4, -1e10, 1e20, -1e30, 1.5e38, 1e-3])[:, None]
    up = up * (1 + 0.1 * torch.rand(8, K, generator=g))
    gate += 0.25 * torch.arange(8)[:, None]
    gate[::2, 7::640], gate[1::2, 7::640] = 2.0, -3.3e38
    gu = torch.cat([gate, up], 1).to(BF)
    _, _, q, s = C.out8(8, K)
    native.swiglu_mx8(gu.to(DEV), q, s)
    q, s = q.cpu(), s.cpu()
    y = M.blocks(M.swiglu(gu))
    # relative: as in test_swiglu; past fp32's normal range u e^g is off by half of 2^-149, |g| times that in the end
    d, a = (180 + 8) * 2.0 ** -23, 256 * 2.0 ** -150
    lo, hi = M.scale_codes((y.abs() * (1 - d) - a).clamp(min=0), M.GRID8), M.scale_codes(y.abs() * (1 + d) + a, M.GRID8)
    got = s.long()
    assert ((got >= lo) & (got <= hi)).all()
    scale = M.scale_values(got)[..., None]
    v = y / scale
    have = M.values8(q, torch.full_like(s, 127)).view(v.shape)
    off = (have - v).abs() - (M.GRID8[M.nearest(v, M.GRID8)] - v.abs()).abs()
    assert (off <= 2 * (d * v.abs() + a / scale)).all(), float((off / (d * v.abs() + a / scale)).max())
    assert torch.equal(torch.signbit(have), torch.signbit(v))


def test_swiglu_largest_gates(native):
    """Infinities, and gates as large as bf16 has: -inf makes its block NaN, as silu(-inf) = -inf * 0 is; the largest
    negative one is 0, with the sign of -u."""
    g = torch.full((3, 64), -100.0)
    g[0, 3], g[1, 40], g[2, 9] = -float("inf"), -3.38e38, float("inf")
    u = torch.full((3, 64), 2.0)
    u[1, 40] = -3e38
    _, _, q, s = C.out8(3, 64)
    native.swiglu_mx8(torch.cat([g, u], 1).to(BF).to(DEV), q, s)
    assert (s.cpu() == 255).tolist() == [[True, False], [False, False], [True, False]]
    assert int(q[1, 40]) == 0 and (q[1, :32] == 0x81).all()  # -200 e^-100 is 0.65 of the least code
