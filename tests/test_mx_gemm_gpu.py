"""The product of 8-bit rows and a 4-bit weight on the GPU against the 64-bit product of the values that the codes
stand for: row counts from one to a prompt's, odd sizes, strides, NaN, rows that keep their bits, untouched
surroundings, captures."""
import pytest
import torch

import mx_cases as C
from oracle import mx_oracle as M

pytestmark = pytest.mark.gpu
BF, F64, U8, DEV = C.BF, C.F64, C.U8, C.DEV


def rows8(g, n, K):
    """8-bit rows with a few large channels, their scales far apart."""
    x = torch.randn(n, K, generator=g) * torch.exp(1.5 * torch.randn(1, K, generator=g).clamp(0))
    return M.quant8(x * torch.exp2(torch.randint(-6, 6, (n, 1), generator=g).float()))


def case(native, g, n, N, K):
    q, s = rows8(g, n, K)
    w = (torch.randn(N, K, generator=g) * K ** -0.5).to(BF)
    wq, wv = C.weight(native, w)
    return q, s, wq, M.values8(q, s), wv


SHAPES = [(1, 16, 32), (1, 1, 32), (1, 5120, 544), (3, 17, 96), (8, 40, 1056), (16, 100, 512), (17, 33, 640),
          (5, 264, 4128), (31, 129, 224), (32, 257, 128), (33, 64, 2048), (64, 300, 160), (65, 500, 1152),
          (77, 129, 800), (96, 1000, 288), (127, 77, 416), (128, 512, 1024), (129, 255, 96), (200, 640, 1568),
          (255, 513, 544), (256, 256, 256), (257, 300, 2080), (300, 1025, 512), (511, 100, 192), (512, 768, 768),
          (700, 333, 1312), (1030, 300, 352), (2048, 520, 256)]


@pytest.mark.parametrize("n,N,K", SHAPES)
def test_product(native, n, N, K):
    import qengine_amd as qa
    g = C.gen(n * 31 + N * 7 + K)
    q, s, wq, xv, wv = case(native, g, n, N, K)
    for pads in (0, 1):
        if pads:  # rows of wider buffers; the scales' rows start at odd bytes
            qd = torch.full((n, K + 48), 0x7F, dtype=U8, device=DEV)[:, 16: 16 + K]
            sd = torch.full((n, K // 32 + 3), 0xFF, dtype=U8, device=DEV)[:, 1: 1 + K // 32]
            big = torch.full((n + 1, N + 5), 7.0, dtype=BF, device=DEV)
            out = big[:n, 3: 3 + N]
        else:
            qd, sd = torch.empty(n, K, dtype=U8, device=DEV), torch.empty(n, K // 32, dtype=U8, device=DEV)
            out = torch.full((n, N), float("nan"), dtype=BF, device=DEV)
        qd.copy_(q)
        sd.copy_(s)
        ws = qa.alloc_mx4_ws(n, N, K)
        native.gemm_mx4(wq, qd, sd, out, ws.fill_(0xFF))
        C.check_product(out, xv, wv, K)
        if pads:
            assert (big[n] == 7).all() and (big[:, :3] == 7).all() and (big[:, 3 + N:] == 7).all()
        first = out.clone()
        native.gemm_mx4(wq, qd, sd, out, ws)  # the same bits again
        assert torch.equal(first, out)
        native.gemm_mx4(wq, qd, sd, out)      # and without a workspace the same values
        C.check_product(out, xv, wv, K)


@pytest.mark.parametrize("n,N", [(40, 3000), (100, 1100), (300, 4200), (500, 2300)])
def test_every_remainder_of_k(native, n, N):
    """Parts of K that begin and end anywhere: in groups of waves, in workgroups (with a workspace), in steps."""
    import qengine_amd as qa
    for blocks in (*range(4, 37), 70, 75, 131, 134, 193, 258, 261, 266, 330):
        K = 32 * blocks
        g = C.gen(n + K)
        q, s, wq, xv, wv = case(native, g, n, N, K)
        out = torch.full((n, N), float("nan"), dtype=BF, device=DEV)
        ws = qa.alloc_mx4_ws(n, N, K).fill_(0xFF)
        q, s = q.to(DEV), s.to(DEV)
        native.gemm_mx4(wq, q, s, out, ws)
        C.check_product(out, xv, wv, K)
        first = out.clone()
        for _ in range(3):
            native.gemm_mx4(wq, q, s, out, ws)
            assert torch.equal(first, out), K


# weight rows past the last whole turn of the CUs go to another kernel: odd ends, strides, a workspace for them alone
@pytest.mark.parametrize("n,N,K", [(500, 33003, 2080), (64, 33001, 4096), (70, 16901, 8192), (1000, 17000, 2048),
                                   (32, 34815, 5120)])
def test_wide_products(native, n, N, K):
    import qengine_amd as qa
    g = C.gen(N)
    q, s, wq, xv, wv = case(native, g, n, N, K)
    big = torch.full((n, N + 6), 7.0, dtype=BF, device=DEV)
    for out in (big[:, 5: 5 + N], torch.empty(n, N, dtype=BF, device=DEV)):
        native.gemm_mx4(wq, q.to(DEV), s.to(DEV), out, qa.alloc_mx4_ws(n, N, K).fill_(0xFF))
        C.check_product(out, xv, wv, K)
    assert (big[:, :5] == 7).all() and (big[:, 5 + N:] == 7).all()


@pytest.mark.parametrize("n,N,K", [(1, 200, 96), (9, 200, 1056), (40, 200, 1056), (150, 200, 480), (600, 300, 480)])
def test_nan_stays_in_its_row_and_column(native, n, N, K):
    g = C.gen(n)
    q, s, wq, xv, _ = case(native, g, n, N, K)
    r, j = n // 2, N - 3
    s2, q2 = s.clone(), q.clone()
    s2[r, K // 32 - 1] = 255
    w = (torch.randn(N, K, generator=g) * K ** -0.5).to(BF)
    w[j, 7] = float("inf")
    wq, wv = C.weight(native, w)
    q2[0, 3] = 0x7F  # a NaN code under an ordinary scale
    out = torch.empty(n, N, dtype=BF, device=DEV)
    native.gemm_mx4(wq, q2.to(DEV), s2.to(DEV), out)
    got = torch.isnan(out.cpu())
    want = torch.zeros(n, N, dtype=torch.bool)
    want[r], want[0], want[:, j] = True, True, True
    assert torch.equal(got, want)
    keep = torch.ones(N, dtype=torch.bool)
    keep[j] = False
    rows = torch.ones(n, dtype=torch.bool)
    rows[r] = rows[0] = False
    if rows.any():
        C.check_product(out.cpu()[rows][:, keep], xv[rows], wv[keep], K)


def test_extreme_scales(native):
    """Scales at both ends: sums that leave fp32's range upwards are infinite, downwards zero, and a tiny scale times
    a large one is an ordinary value."""
    n, N, K = 2, 16, 64
    q = torch.full((n, K), 0x38, dtype=U8, device=DEV)  # 1.0
    w = torch.ones(N, K, dtype=BF)
    wq, _ = C.weight(native, w * 2.0 ** 100)
    out = torch.empty(n, N, dtype=BF, device=DEV)
    for code, want in ((254, float("inf")), (0, 64 * 2.0 ** -27), (27, 64.0)):
        s = torch.full((n, K // 32), code, dtype=U8, device=DEV)
        native.gemm_mx4(wq, q, s, out)
        assert (out == want).all(), (code, out)


@pytest.mark.parametrize("N,K", [(320, 5120), (1000, 992), (5120, 544)])
def test_decode_rows_keep_their_bits(native, N, K):
    """Row r of a call of up to 16 rows has the bits of a call on that row alone: a verify pass is plain decoding."""
    import qengine_amd as qa
    g = C.gen(N + K)
    q, s, wq, _, _ = case(native, g, 16, N, K)
    q, s = q.to(DEV), s.to(DEV)
    alone = torch.empty(16, N, dtype=BF, device=DEV)
    for r in range(16):
        native.gemm_mx4(wq, q[r: r + 1], s[r: r + 1], alone[r: r + 1], qa.alloc_mx4_ws(1, N, K))
    for n in range(2, 17):
        out = torch.empty(n, N, dtype=BF, device=DEV)
        native.gemm_mx4(wq, q[:n], s[:n], out, qa.alloc_mx4_ws(n, N, K))
        assert torch.equal(out, alone[:n]), n


@pytest.mark.parametrize("n", [1, 40, 300])
def test_captured_and_on_other_streams(native, n):
    """Replays of a graph on changed inputs equal the eager call, with eager work between them; two calls on two
    streams, each with its workspace, too."""
    import qengine_amd as qa
    N, K = 700, 1504
    g = C.gen(n)
    q, s, wq, _, _ = case(native, g, n, N, K)
    q, s = q.to(DEV), s.to(DEV)
    ws, out, ref = qa.alloc_mx4_ws(n, N, K), *(torch.empty(n, N, dtype=BF, device=DEV) for _ in range(2))
    native.gemm_mx4(wq, q, s, out, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        native.gemm_mx4(wq, q, s, out, ws)
    ws2 = qa.alloc_mx4_ws(n, N, K)
    for k in range(4):
        a, b = rows8(g, n, K)
        q.copy_(a)
        s.copy_(b)
        out.fill_(float("nan"))
        graph.replay()
        native.gemm_mx4(wq, q, s, ref, ws2)
        torch.cuda.synchronize()
        assert torch.equal(out, ref), k
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [torch.empty_like(out) for _ in range(6)]
    for k in range(6):
        with torch.cuda.stream(side if k % 2 else torch.cuda.current_stream()):
            native.gemm_mx4(wq, q, s, outs[k], ws if k % 2 else ws2)
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs)


def test_offsets_past_32_bits(native):
    """Codes of rows, and outputs, that lie past 2^32 bytes: the last rows of a tall call."""
    n, N, K = 66000, 33000, 64
    g = C.gen(9)
    q, s = rows8(g, 5, K)
    wide = torch.zeros(n, 1 << 16, dtype=U8, device=DEV)  # 4.3 GB: rows 65,536 bytes apart
    qd, sd = wide[:, 128: 128 + K], torch.full((n, 2), 127, dtype=U8, device=DEV)
    qd[-5:].copy_(q)
    sd[-5:].copy_(s)
    w = (torch.randn(N, K, generator=g)).to(BF)
    wq, wv = C.weight(native, w)
    out = torch.empty(n, N, dtype=BF, device=DEV)
    native.gemm_mx4(wq, qd, sd, out)
    C.check_product(out[-5:], M.values8(q, s), wv, K)
    assert (out[: n - 5] == 0).all()


@pytest.mark.parametrize("n,N,K", [(100, 513, 17408), (40, 100, 9376)])
def test_workspaces_of_any_size(native, n, N, K):
    """A workspace that is too small for a split is used for a smaller one, or not at all; no byte past it is written."""
    import qengine_amd as qa
    g = C.gen(n)
    q, s, wq, xv, wv = case(native, g, n, N, K)
    need = qa.mx4_ws_bytes(n, N, K)
    assert need > 0
    out = torch.empty(n, N, dtype=BF, device=DEV)
    for size in (need + 4096, need, need - 16, need // 2, need // 4 // 16 * 16, 16, 0):
        big = torch.full((size + 65536,), 0x55, dtype=U8, device=DEV)
        out.fill_(float("nan"))
        native.gemm_mx4(wq, q.to(DEV), s.to(DEV), out, big[:size])
        C.check_product(out, xv, wv, K)
        assert (big[max(size, 0):] == 0x55).all(), size


def test_weights_past_32_bits(native):
    """Codes of a weight that lie past 2^32 bytes: quantised, read back, and multiplied by one row and by many."""
    import qengine_amd as qa
    N, K, m = 270016, 32768, 40
    w = torch.zeros(N, K, dtype=BF, device=DEV)  # 17.7 GB, 4.4 GB of codes
    g = C.gen(3)
    tail = (torch.randn(m, K, generator=g) * K ** -0.5).to(BF)
    w[-m:].copy_(tail)
    wq = qa.alloc_mx4(N, K, DEV)
    native.mx4_quant(w, wq)
    native.mx4_dequant(wq, w.fill_(1.0))
    want = M.values4(*M.quant4(tail))
    assert torch.equal(w[-m:].cpu().to(F64), want.to(F64)) and not w[:-m:4096].any()
    del w
    for n in (1, 20, 300):
        q, s = rows8(g, n, K)
        out = torch.empty(n, N, dtype=BF, device=DEV)
        native.gemm_mx4(wq, q.to(DEV), s.to(DEV), out)
        C.check_product(out[:, -m:].contiguous(), M.values8(q, s), want, K)
        assert not out[:, :-m].any(), n
