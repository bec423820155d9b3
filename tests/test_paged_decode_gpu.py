"""attn_decode_paged / attn_decode_paged_fp8 against the fp64 model (oracle/paged_oracle.py, whose bound
counts the roundings of a correct fp32 evaluation), over lengths, page sizes, head groupings, windows,
unmapped pages, poisoned cache rows, strides, streams and captures."""
import numpy as np
import pytest
import torch

from paged_cases import BF, D, KV_SCALE, Batch, gen

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Call:
    """A Batch on the GPU with its scratch; run() returns out as float32 on the host."""

    def __init__(self, c, ns=16):
        self.c, self.ns = c, ns
        self.kp, self.vp, self.table = c.kp.to(DEV), c.vp.to(DEV), c.table.to(DEV)
        self.q, self.qg = c.q.to(DEV), c.qg.to(DEV)
        self.pos = torch.tensor(c.pos, dtype=torch.int32, device=DEV)
        n = c.B * c.R
        self.po = torch.full((n, c.hq, ns, D), float("nan"), device=DEV)
        self.pml = torch.full((n, c.hq, ns, 2), float("nan"), device=DEV)
        self.out = torch.full((n, c.hq * D), 7.0, dtype=BF, device=DEV)

    def run(self, native):
        c = self.c
        if c.kv == "fp8":
            native.attn_decode_paged_fp8(self.q, self.kp, self.vp, self.table, self.pos, self.qg, self.po,
                                         self.pml, self.out, KV_SCALE, KV_SCALE, c.window, c.sinks)
        else:
            native.attn_decode_paged(self.q, self.kp, self.vp, self.table, self.pos, self.qg, self.po,
                                     self.pml, self.out, c.window, c.sinks)
        return self.out

    def check(self, native):
        out = self.run(native).float().cpu().numpy().reshape(-1, self.c.hq, D)
        want, tol = self.c.exact()
        for b, p in enumerate(self.c.pos):
            for t in range(self.c.R):
                i = b * self.c.R + t
                if p < 0:
                    assert (out[i] == 7.0).all(), ("idle row written", b, t)
                    continue
                d = np.abs(out[i] - want[i])
                assert (d <= tol[i]).all(), (b, t, p, float((d / tol[i]).max()), float(d.max()))


EDGES = [0, 1, 14, 15, 16, 30, 31, 32, 62, 63, 64, 127, 128, 129, 255, 300, 511, 512, 513, 1025]


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("P", [16, 32, 64, 256])
def test_lengths_at_the_edges(native, P, kv):
    Call(Batch(P, EDGES, hq=6, hkv=1, P=P, kv=kv)).check(native)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("hq,hkv,R", [(1, 1, 1), (2, 2, 8), (24, 4, 2), (24, 4, 3), (24, 4, 5), (24, 4, 8),
                                      (16, 2, 4), (16, 2, 8), (32, 8, 5), (40, 1, 1), (40, 1, 3), (64, 1, 2),
                                      (34, 2, 7)])
def test_head_groupings_and_rows(native, hq, hkv, R, kv):
    Call(Batch(hq + R, [0, 61, 250, 126], R=R, hq=hq, hkv=hkv, P=32, kv=kv)).check(native)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (16, 16), (31, 4), (32, 0), (33, 40), (64, 1),
                                          (100, 100), (257, 4), (4000, 4), (4000, 0)])
@pytest.mark.parametrize("R", [1, 4])
def test_windows_and_first_tokens(native, window, sinks, R, kv):
    c = Batch(window + sinks + R, [0, 3, 31, 64, 97, 255, 256, 700, 1501], R=R, hq=6, hkv=2, P=16, kv=kv,
              window=window, sinks=sinks)
    c.poison()
    Call(c).check(native)


@pytest.mark.parametrize("ns,window", [(1, 0), (2, 0), (3, 0), (4, 0), (7, 0), (64, 0), (200, 0), (4, 90),
                                       (5, 90), (7, 90), (64, 90), (200, 90)])
def test_split_counts(native, ns, window):
    Call(Batch(ns, [10, 700, 2111], R=3, hq=6, hkv=1, P=16, window=window, sinks=5 if window else 0),
         ns=ns).check(native)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_rows_outside_hold_anything(native, bad, kv):
    """Cache rows that nobody attends, scratch and the rows of idle sequences may hold anything."""
    c = Batch(5, [0, -1, 45, 200, -7, 333], R=3, hq=12, hkv=2, P=64, kv=kv)
    c.poison(bad)
    Call(c).check(native)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("hq", [2, 6])
@pytest.mark.parametrize("window", [0, 40])
def test_a_later_rows_values_do_not_reach_an_earlier_row(native, kv, hq, window):
    """K and V of row t at infinity or NaN: rows before t stay finite and keep their values, rows from t on
    show it."""
    R = 4
    for t, bad in ((1, float("inf")), (2, float("nan")), (3, float("-inf"))):
        c = Batch(9, [37, 61, 64], R=R, hq=hq, hkv=1, P=16, kv=kv, window=window)
        clean = Call(c).run(native).clone()
        for b in range(c.B):
            p = c.pos[b] + t
            page = int(c.table[b, p // c.P])
            for x, d in ((c.vp, slice(3, 9)), (c.kp, slice(0, 1))):
                if x is c.kp and bad != bad:
                    continue
                y = x.float()
                y[page, :, p % c.P, d] = bad if x is c.vp else 1.0
                x.copy_(y.to(x.dtype))
        k = Call(c)
        out = k.run(native).float().view(c.B, R, hq, D)
        # row t's key changed: only rows < t keep the clean bits
        assert torch.equal(out[:, :t], clean.float().view(c.B, R, hq, D)[:, :t]), (t, bad)
        want = torch.from_numpy(c.exact()[0]).view(c.B, R, hq, D)
        nan = bad != bad or kv == "fp8"  # (E4M3FN has no infinity: inf becomes NaN)
        seen = out[:, t:, :, 3:9].cpu()
        assert (torch.isnan(seen) if nan else seen == want[:, t:, :, 3:9].float()).all(), (t, bad)
        assert torch.isfinite(out[:, t:, :, 9:]).all() and torch.isfinite(out[:, t:, :, :3]).all()


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("lens", [[0, 40, 700], [0, 3, 700, 1500] + [200] * 30])
def test_nan_is_not_lost(native, lens, kv):
    """A row whose query is NaN, or whose attended keys all are, is NaN (no score is a maximum then), and no other
    row of the call changes."""
    c = Batch(31, lens, R=2, hq=8, hkv=2, kv=kv)
    want = Call(c).run(native).view(-1, c.hq, D).clone()
    c.q.view(-1, c.hq, D)[5, 3, 17] = float("nan")                # row 1 of sequence 2
    c.kp.view(torch.uint8)[int(c.table[0, 0])] = 0xff             # every key that sequence 0 attends
    got = Call(c).run(native).view(-1, c.hq, D)
    assert got[:2].isnan().all() and got[5, 3].isnan().all()
    rest = torch.ones(got.shape[:2], dtype=torch.bool, device=DEV)
    rest[:2], rest[5, 3] = False, False
    assert torch.equal(got[rest], want[rest])


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_unmapped_and_foreign_pages_are_not_attended(native, kv):
    c = Batch(11, [50, 200, 64, 33], R=2, hq=6, hkv=1, P=16, kv=kv)
    c.table[0, 1] = -1
    c.table[1, 0] = c.N
    c.table[1, 12] = 2 ** 31 - 1
    c.table[2, :] = -5          # a row that attends nothing: 0
    c.table[3, 2] = -2 ** 31
    Call(c).check(native)


def test_positions_past_the_table(native):
    c = Batch(12, [40, 40, 40, 40], R=2, hq=6, hkv=1, P=16, extra_m=0)
    c.pos = [47, 300, 2 ** 31 - 1, 46]  # table rows hold 48 positions
    Call(c).check(native)
    c.window, c.sinks = 20, 3
    c.pos = [47, 66, 67, 2 ** 31 - 1]
    Call(c).check(native)
    c.sinks = 0                 # a window past the table: nothing to attend
    Call(c).check(native)


def _bits(c, native, ns=16):
    return Call(c, ns).run(native).clone()


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 3), (600, 20)])
@pytest.mark.parametrize("hq,hkv", [(24, 4), (16, 2)])
def test_row_bits_do_not_depend_on_other_rows_or_sequences(native, kv, window, sinks, hq, hkv):
    R, lens = 8, [1020, 30, 505, 91]
    c = Batch(20, lens, R=R, hq=hq, hkv=hkv, P=16, kv=kv, window=window, sinks=sinks, trim=False)
    whole = _bits(c, native).view(4, R, -1)
    q, qg = c.q.view(4, R, -1), c.qg.view(4, R, -1)
    for t in range(R):
        one = Batch(20, lens, R=R, hq=hq, hkv=hkv, P=16, kv=kv, window=window, sinks=sinks, trim=False)
        one.R, one.q, one.qg = 1, q[:, t].contiguous(), qg[:, t].contiguous()
        one.pos = [n + t for n in lens]
        assert torch.equal(_bits(one, native), whole[:, t]), t
        one.pos = [-1, lens[1] + t, -1, 0]  # the others idle or elsewhere
        assert torch.equal(_bits(one, native)[1], whole[1, t]), t


def test_rows_whose_slice_size_changes_inside_a_call(native):
    """Slices grow by 32 positions where the length passes a multiple of 32 NS: rows on both sides."""
    ns, R = 5, 8
    for n in (32 * ns * 3 - 4, 32 * ns * 8 - 7, 32 * ns - 1):
        c = Batch(n, [n, 7], R=R, hq=6, hkv=1, P=16)
        Call(c, ns).check(native)
        whole = _bits(c, native, ns).view(2, R, -1)
        one = Batch(n, [n, 7], R=R, hq=6, hkv=1, P=16)
        for t in range(R):
            one.R, one.q, one.qg = 1, c.q.view(2, R, -1)[:, t].contiguous(), c.qg.view(2, R, -1)[:, t].contiguous()
            one.pos = [n + t, 7 + t]
            assert torch.equal(_bits(one, native, ns), whole[:, t]), (n, t)


def test_large_batches_and_many_items(native):
    """More sequences than lanes, more items than workgroups."""
    g = np.random.default_rng(0)
    lens = [int(x) for x in g.integers(0, 120, 150)]
    lens[17] = -1
    Call(Batch(30, lens, hq=2, hkv=1, P=16), ns=4).check(native)
    lens = [int(x) for x in g.integers(0, 40, 1024)]
    Call(Batch(31, lens, hq=1, hkv=1, P=16), ns=2).check(native)
    lens = [int(x) for x in g.integers(400, 2000, 24)]
    Call(Batch(32, lens, R=2, hq=8, hkv=8, P=32), ns=64).check(native)


def test_tables_and_rows_with_strides(native):
    c = Batch(40, [33, 90, 128], R=2, hq=6, hkv=2, P=32)
    want = _bits(c, native)
    k = Call(c)
    wide = torch.full((c.B, c.M + 5), 3, dtype=torch.int32, device=DEV)
    wide[:, :c.M] = k.table
    k.table = wide[:, :c.M]
    pad = torch.zeros(c.B * c.R, c.hq * 2 * D + 40, dtype=BF, device=DEV)
    pad[:, 3:3 + c.hq * 2 * D] = k.qg
    k.qg = pad[:, 3:3 + c.hq * 2 * D]       # odd alignment
    o = torch.full((c.B * c.R, c.hq * D + 9), 5.0, dtype=BF, device=DEV)
    k.out = o[:, 1:1 + c.hq * D]
    assert torch.equal(k.run(native), want)
    assert (o[:, 0] == 5).all() and (o[:, 1 + c.hq * D:] == 5).all()


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_pools_past_32_bit_offsets(native, kv):
    """Page ids whose byte offset passes 2^32 (and 2^31 elements)."""
    P, hkv = 64, 4
    elem = 1 if kv == "fp8" else 2
    N = (1 << 32) // (hkv * P * D * elem) + 40
    c = Batch(50, [100, 300], R=2, hq=24, hkv=hkv, P=P, kv=kv)
    k = Call(c)
    for name in ("kp", "vp"):
        small = getattr(k, name)
        big = torch.empty(N, hkv, P, D, dtype=small.dtype, device=DEV)
        big.view(torch.uint8)[N - c.N:] = small.view(torch.uint8)
        setattr(k, name, big)
    k.table = torch.where(k.table >= 0, k.table + (N - c.N), k.table)
    k.check(native)


def test_long_cache(native):
    """130,000 positions (slices of many tiles; pages shared between them, to keep the pool small), against
    float64 on the GPU."""
    P, L, hq, hkv, R = 64, 130001, 6, 1, 2
    g = gen(60)
    N = 40
    kp = torch.randn(N, hkv, P, D, generator=g).to(BF).to(DEV)
    vp = torch.randn(N, hkv, P, D, generator=g).to(BF).to(DEV)
    M = L // P + 2
    table = torch.randint(0, N, (1, M), generator=g).int().to(DEV)
    q = torch.randn(R, hq * D, generator=g).to(BF).to(DEV)
    qg = torch.randn(R, hq * 2 * D, generator=g).to(BF).to(DEV)
    for ns in (3, 64):
        po, pml = torch.empty(R, hq, ns, D, device=DEV), torch.empty(R, hq, ns, 2, device=DEV)
        out = torch.empty(R, hq * D, dtype=BF, device=DEV)
        pos = torch.tensor([L - R], dtype=torch.int32, device=DEV)
        native.attn_decode_paged(q, kp, vp, table, pos, qg, po, pml, out)
        for t in range(R):
            n = L - R + t + 1
            K = kp[table[0].long(), 0].reshape(-1, D)[:n].double()
            V = vp[table[0].long(), 0].reshape(-1, D)[:n].double()
            s = q[t].view(hq, D).double() @ K.T.contiguous() / 16
            w = torch.softmax(s, -1)
            gate = torch.sigmoid(qg[t].view(hq, 2 * D)[:, D:].double())
            want = (w @ V) * gate
            A = (q[t].view(hq, D).double().abs() @ K.abs().T.contiguous()).max(-1, keepdim=True)[0] / 16
            eps = 2 * 262 * 2.0 ** -24 * A + 2.0 ** -15 + 2 * (n + 64) * 2.0 ** -24
            tol = eps * (w @ V.abs()) * gate + 2.0 ** -8 * want.abs()
            assert ((out[t].view(hq, D).double() - want).abs() <= tol).all(), (ns, t)


def test_other_stream_and_capture(native):
    c = Batch(70, [100, 37, -1], R=2, hq=6, hkv=2, P=16, window=50, sinks=4, trim=False)
    k = Call(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        k.check(native)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k.run(native)
    e = Call(c)
    for pos in ([0, 5, 9], [101, -1, 40], [64, 30, 31], [77, 12, -1]):
        for call in (k, e):
            call.pos.copy_(torch.tensor(pos, dtype=torch.int32))
            call.out.fill_(3.0)
        graph.replay()
        e.run(native)
        torch.cuda.synchronize()
        assert torch.equal(k.out, e.out), pos


def test_two_calls_at_once(native):
    a, b = Call(Batch(80, [900, 800], R=2)), Call(Batch(81, [700, 950], R=2))
    want = a.run(native).clone(), b.run(native).clone()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        a.out.zero_(), b.out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            a.run(native)
        with torch.cuda.stream(s2):
            b.run(native)
        torch.cuda.synchronize()
        assert torch.equal(a.out, want[0]) and torch.equal(b.out, want[1])


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (20, 0), (20, 5), (200, 3)])
@pytest.mark.parametrize("hq,hkv,R,P,M", [(24, 4, 1, 16, 1), (24, 4, 6, 32, 1), (16, 2, 8, 64, 2), (40, 1, 3, 16, 16),
                                          (6, 3, 2, 128, 2)])
def test_short_tables(native, hq, hkv, R, P, M, window, sinks, kv):
    """Short tables, whose rows are one or a few slices, and rows past their end; the same bits where the output's rows
    are not aligned to 16 bytes."""
    cap = P * M
    lens = sorted({0, 1, 7, cap // 2, cap - 1, cap + 3, -1, max(cap - R, 0), cap + 500, 3 * cap})
    c = Batch(77, [min(n, cap - 1) for n in lens], R=R, hq=hq, hkv=hkv, P=P, kv=kv, window=window, sinks=sinks,
              trim=False, extra_m=0)
    c.table, c.M = c.table[:, :M].contiguous(), M
    c.pos = lens
    call = Call(c)
    call.check(native)
    first = call.out.clone()
    call.po.fill_(float("nan"))
    wide = torch.full((c.B * R, hq * D + 8), 7.0, dtype=BF, device=DEV)
    call.out = wide[:, 4:4 + hq * D]
    call.run(native)
    assert torch.equal(call.out, first)
    assert (wide[:, :4] == 7).all() and (wide[:, 4 + hq * D:] == 7).all()
