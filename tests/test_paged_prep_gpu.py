"""attn_prep_paged / attn_prep_paged_fp8 against the fp64 model: q rows, the written cache rows, and every
other cache row untouched."""
import numpy as np
import pytest
import torch

from oracle import kv8_oracle, paged_oracle
from paged_cases import BF, D, FP8, KV_SCALE, gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
# fp32 in units of the row's (pair's) magnitude: the sum of squares (8 terms and 5 levels), quotient, root,
# three products, cos and sin rounded to fp32, two products and their sum: fewer than 32 roundings of 2^-24.
# Then one rounding to bf16.
FP32 = 32 * 2.0 ** -24
EPS = 1e-6


def _case(seed, pos, R, hq, hkv, P, M, rd=64, pad=8, shift=0, kv="bf16"):
    g = gen(seed)
    B = len(pos)
    rows = B * R
    w = (hq * 2 + 2 * hkv) * D
    proj = torch.zeros(rows, w + pad + shift, dtype=BF)
    proj[:, shift:shift + w] = (torch.randn(rows, w, generator=g) * 3).to(BF)
    N = B * M + 3
    table = torch.randperm(N, generator=g)[:B * M].int().view(B, M)
    pool = torch.randn(N, hkv, P, D, generator=g)
    pool = pool.to(BF) if kv == "bf16" else pool.to(FP8)
    nw = [(torch.randn(D, generator=g) * 0.3).to(BF) for _ in range(2)]
    freq = (1.0 / (1e7 ** (torch.arange(0, rd, 2, dtype=torch.float32) / rd)))
    return dict(proj=proj.to(DEV), shift=shift, w=w, table=table.to(DEV), kp=pool.to(DEV),
                vp=pool.clone().to(DEV), qnw=nw[0].to(DEV), knw=nw[1].to(DEV), freq=freq.to(DEV), pos=pos, R=R,
                hq=hq, hkv=hkv, P=P, M=M, N=N, kv=kv, rows=rows)


def _run(native, c, q=None):
    a = c["shift"]
    b, d = a + c["hq"] * 2 * D, a + (c["hq"] * 2 + c["hkv"]) * D
    pr = c["proj"]
    q = torch.full((c["rows"], c["hq"] * D), 9.0, dtype=BF, device=DEV) if q is None else q
    pos = torch.tensor(c["pos"], dtype=torch.int32, device=DEV)
    args = (pr[:, a:b], pr[:, b:d], pr[:, d:a + c["w"]], c["qnw"], c["knw"], c["freq"], pos, q, c["kp"],
            c["vp"], c["table"], EPS)
    if c["kv"] == "fp8":
        native.attn_prep_paged_fp8(*args, KV_SCALE, 2 * KV_SCALE)
    else:
        native.attn_prep_paged(*args)
    return q, args


def _check(native, c):
    k0, v0 = c["kp"].clone(), c["vp"].clone()
    q, args = _run(native, c)
    hq, hkv, R, P, M, N = c["hq"], c["hkv"], c["R"], c["P"], c["M"], c["N"]
    f = lambda x: x.float().cpu().numpy()  # noqa: E731
    wq, wk, wv, qm, km = paged_oracle.prep(f(args[0]), f(args[1]), f(args[2]), f(c["qnw"]), f(c["knw"]),
                                           c["freq"].cpu().numpy(), c["pos"], R, hq, hkv, EPS)
    got = f(q).reshape(-1, hq, D)
    kp, vp = k0.view(torch.uint8).cpu().clone(), v0.view(torch.uint8).cpu().clone()
    gk, gv = c["kp"].view(torch.uint8).cpu(), c["vp"].view(torch.uint8).cpu()
    table = c["table"].cpu().numpy()
    for i in range(c["rows"]):
        b, t = divmod(i, R)
        if c["pos"][b] < 0:
            assert (got[i] == 9.0).all()
            continue
        assert (np.abs(got[i] - wq[i]) <= FP32 * qm[i] + 2.0 ** -8 * np.abs(wq[i])).all(), i
        p = c["pos"][b] + t
        page = table[b, p // P] if p < M * P else -1
        if not 0 <= page < N:
            continue
        # these rows were written: check them, then take them over, so that the rest must be untouched
        rk, rv = c["kp"][page, :, p % P], c["vp"][page, :, p % P]
        if c["kv"] == "bf16":
            assert (np.abs(f(rk) - wk[i]) <= FP32 * km[i] + 2.0 ** -8 * np.abs(wk[i])).all(), i
            assert (f(rv) == wv[i]).all(), i
        else:
            x = wk[i] / KV_SCALE
            y = kv8_oracle.decode(rk).reshape(x.shape)
            xc = np.clip(x, -448, 448)
            # half a step of E4M3: 2^-4 of the value, 2^-10 below the least normal 2^-6
            assert (np.abs(y - xc) <= 2.0 ** -4 * np.abs(xc) + 2.0 ** -10 + FP32 * km[i] / KV_SCALE).all(), i
            code = kv8_oracle.encode(wv[i].astype(np.float32), 2 * KV_SCALE)
            assert (rv.view(torch.uint8).cpu().numpy() == code).all(), i
        kp[page, :, p % P] = gk[page, :, p % P]
        vp[page, :, p % P] = gv[page, :, p % P]
    assert torch.equal(kp, gk) and torch.equal(vp, gv)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("hq,hkv,R,P", [(24, 4, 1, 64), (24, 4, 4, 16), (16, 2, 8, 32), (1, 1, 3, 16),
                                        (5, 5, 2, 128)])
def test_rows_and_pages(native, hq, hkv, R, P, kv):
    _check(native, _case(hq + R, [0, P - 1, 2 * P - 2, -1, 3 * P - 1], R, hq, hkv, P, 4, kv=kv))


@pytest.mark.parametrize("rd", [2, 6, 34, 64, 128, 256])
def test_rotary_widths(native, rd):
    _check(native, _case(rd, [3, 40], 2, 3, 1, 16, 4, rd=rd))


@pytest.mark.parametrize("shift,pad", [(0, 8), (1, 3), (8, 0), (4, 4)])
def test_alignment(native, shift, pad):
    _check(native, _case(9, [3, 40], 2, 3, 2, 16, 4, shift=shift, pad=pad))


def test_far_positions(native):
    """The angle is not rounded to fp32 (at 500,000 its last place is 0.03 rad)."""
    c = _case(4, [500000, 131071], 3, 2, 1, 32768, 16)
    _check(native, c)


def test_rows_without_a_page(native):
    c = _case(5, [15, 30, 62, 200, 2 ** 31 - 3], 4, 2, 1, 16, 4)
    c["table"][0, 1] = -1
    c["table"][1, 1] = c["N"]
    c["table"][2, 3] = 2 ** 31 - 1
    _check(native, c)


def test_a_prompt_of_many_rows(native):
    _check(native, _case(6, [5], 700, 4, 2, 64, 12))


def test_capture(native):
    c = _case(7, [5, 20], 2, 4, 2, 16, 4)
    q, args = _run(native, c)
    want = q.clone(), c["kp"].clone(), c["vp"].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        native.attn_prep_paged(*args)
    for _ in range(3):
        q.zero_(), c["kp"].view(torch.uint8).zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, want[0])
        for b, p in ((0, 5), (0, 6), (1, 20), (1, 21)):
            page = int(c["table"][b, p // 16])
            assert torch.equal(c["kp"][page, :, p % 16], want[1][page, :, p % 16])
