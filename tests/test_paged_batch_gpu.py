"""The paged decode's batch form (persistent waves that take equal parts of a batch's items), over the cases that
test_paged_decode_gpu.py has for small calls: windows, poisoned rows, NaN, unmapped pages, rows whose slice size
changes inside a call, more sequences than lanes. Each test asserts that its sizes take that form."""
import numpy as np
import pytest
import torch

import paged_exact
from paged_cases import D
from paged_exact import Big
from test_paged_decode_gpu import DEV, Call

pytestmark = pytest.mark.gpu


def is_batch(native, c, ns):
    return native._attn_decode_paged_form(c.B, c.hkv, c.M * c.P, ns, c.window, c.sinks)[2]


def check(native, c, ns=16):
    """One call in the batch form against float64."""
    assert is_batch(native, c, ns)
    k = Call(c, ns)
    out = k.run(native).double().view(-1, c.hq, D)
    want, tol = paged_exact.decode(c, k.kp, k.vp, k.table, k.q, k.qg)
    idle = want.isnan().all(-1).all(-1)
    assert (out[idle] == 7.0).all()
    d = (out - want).abs()[~idle]
    assert (d <= tol[~idle]).all(), (float((d / tol[~idle]).max()), float(d.max()))
    return k


def lens_of(seed, n, lo, hi):
    return [int(x) for x in np.random.default_rng(seed).integers(lo, hi, n)]


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("P", [16, 32, 128])
@pytest.mark.parametrize("hq,hkv,R", [(24, 4, 1), (16, 2, 3), (16, 2, 4), (24, 4, 8), (8, 8, 2), (40, 1, 2)])
def test_lengths_heads_and_rows(native, hq, hkv, R, P, kv):
    n = 64 if hkv == 8 else 72 if hkv == 4 else 110 if hkv == 2 else 200
    c = Big(P + R, lens_of(P, n - 4, 400, 1800) + [0, 31, -1, 1900], R=R, hq=hq, hkv=hkv, P=P, kv=kv)
    check(native, c)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("window,sinks", [(900, 0), (900, 5), (1024, 33), (700, 300), (3000, 4)])
@pytest.mark.parametrize("hq,hkv,R,P", [(24, 4, 1, 16), (16, 2, 4, 32), (12, 4, 8, 64)])
def test_windows_and_first_tokens(native, hq, hkv, R, P, window, sinks, kv):
    """Rows that nobody attends hold NaN."""
    lens = lens_of(window, 84, 10, 6000) + [0, 1, window - 1, window, window + sinks, -5]
    c = Big(window + sinks + R, lens * (1 if hkv == 4 else 2), R=R, hq=hq, hkv=hkv, P=P, kv=kv, window=window,
              sinks=sinks)
    c.poison()
    check(native, c)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_rows_outside_hold_anything(native, bad, kv):
    lens = lens_of(3, 80, 300, 1500)
    lens[0] = lens[17] = lens[18] = lens[79] = -1
    c = Big(5, lens, R=3, hq=12, hkv=4, P=64, kv=kv)
    c.poison(bad)
    check(native, c)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("window", [0, 800])
def test_unmapped_and_foreign_pages(native, kv, window):
    c = Big(11, lens_of(4, 90, 600, 1600), R=2, hq=16, hkv=4, P=16, kv=kv, window=window, sinks=9 if window else 0,
              trim=False)
    rng = np.random.default_rng(9)
    hole = torch.from_numpy(rng.random((c.B, c.M)) < 0.3)
    bad = torch.from_numpy(rng.choice([-1, c.N, 2 ** 31 - 1, -2 ** 31], (c.B, c.M)).astype(np.int32))
    c.table = torch.where(hole, bad, c.table)
    c.table[5] = -1
    c.table[6, : c.M // 2] = c.N + 3
    check(native, c)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("ns", [4, 5])
def test_rows_whose_slice_size_changes_inside_a_call(native, ns, kv):
    """Slices above the call's least grow by 128 positions where the length passes a multiple of 128 NS: rows of one
    sequence on both sides, each with the bits of a call of its own."""
    R, edges = 8, [128 * ns * i for i in (1, 2, 3) if 128 * ns * i < 1500] + [300]
    lens = [edges[i % len(edges)] - 1 - i % 7 for i in range(70)]
    c = Big(ns, lens, R=R, hq=16, hkv=4, P=16, kv=kv, extra_m=3)
    k = check(native, c, ns)
    whole = k.out.view(c.B, R, -1).clone()
    q, qg = c.q.view(c.B, R, -1), c.qg.view(c.B, R, -1)
    for t in range(R):
        k.c.R, k.c.pos = 1, [n + t for n in lens]
        one = Call(k.c, ns)
        one.q, one.qg = q[:, t].contiguous().to(DEV), qg[:, t].contiguous().to(DEV)
        n = c.B
        one.po, one.pml, one.out = one.po[:n], one.pml[:n], one.out[:n]
        assert torch.equal(one.run(native), whole[:, t]), t


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (900, 20)])
@pytest.mark.parametrize("hq,hkv", [(24, 4), (16, 2)])
def test_row_bits_do_not_depend_on_other_rows_or_sequences(native, kv, window, sinks, hq, hkv):
    R, n = 8, 72 if hkv == 4 else 130
    lens = lens_of(6, n, 200, 1900)
    args = dict(hq=hq, hkv=hkv, P=32, kv=kv, window=window, sinks=sinks, trim=False)
    c = Big(20, lens, R=R, **args)
    assert is_batch(native, c, 16)
    k = Call(c)
    whole = k.run(native).view(n, R, -1).clone()
    q, qg = k.q.view(n, R, -1), k.qg.view(n, R, -1)
    rng = np.random.default_rng(1)
    for t in (0, 3, 7):
        k.q, k.qg, k.out = q[:, t].contiguous(), qg[:, t].contiguous(), torch.zeros_like(whole[:, 0])
        k.pos.copy_(torch.tensor([m + t for m in lens]))
        assert torch.equal(k.run(native), whole[:, t]), t
        # others idle or elsewhere: the items fall to other waves
        mine = rng.random(n) < 0.4
        other = rng.integers(-400, 1500, n)
        k.pos.copy_(torch.tensor([m + t if x else int(o) for m, x, o in zip(lens, mine, other)]))
        assert torch.equal(k.run(native)[torch.from_numpy(mine)], whole[:, t][torch.from_numpy(mine)]), t


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_nan_is_not_lost(native, kv):
    """A NaN query, and a sequence whose keys all are NaN (no slice has a maximum then): those rows are NaN, no other
    row of the call changes."""
    c = Big(31, lens_of(8, 90, 300, 1700), R=2, hq=8, hkv=4, P=16, kv=kv)
    assert is_batch(native, c, 16)
    want = Call(c).run(native).view(-1, c.hq, D).clone()
    c.q.view(-1, c.hq, D)[5, 3, 17] = float("nan")       # row 1 of sequence 2
    for page in c.table[40].tolist():
        if page >= 0:
            c.kp.view(torch.uint8)[page] = 0xff
    got = Call(c).run(native).view(-1, c.hq, D)
    assert got[80:82].isnan().all() and got[5, 3].isnan().all()
    rest = torch.ones(got.shape[:2], dtype=torch.bool, device=DEV)
    rest[80:82], rest[5, 3] = False, False
    assert torch.equal(got[rest], want[rest])


def test_capture_and_two_calls_at_once(native):
    a, b = (Call(Big(s, lens_of(s, 80, 300, 1500), R=2, hq=12, hkv=4, P=16)) for s in (80, 81))
    assert is_batch(native, a.c, 16) and is_batch(native, b.c, 16)
    want = a.run(native).clone(), b.run(native).clone()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        a.run(native)
    for _ in range(4):
        for k in (a, b):
            k.out.zero_(), k.po.fill_(float("nan")), k.pml.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            graph.replay()
        with torch.cuda.stream(streams[1]):
            b.run(native)
        torch.cuda.synchronize()
        assert torch.equal(a.out, want[0]) and torch.equal(b.out, want[1])
