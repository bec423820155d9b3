"""The operations on pages against the CPU model (oracle/paged_oracle.py): table, ref, missing and every
byte of the pools are equal."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as po
from paged_cases import BF, D, FP8, gen, tables_ok

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = torch.int32
MAX = 2 ** 31 - 1


def ints(x):
    return torch.tensor(np.asarray(x), dtype=I32, device=DEV)


class Pages:
    """An allocation on the GPU and its twin in numpy."""

    def __init__(self, B, M, N, P=16, hkv=1, layers=2, kv="bf16", seed=0, stride=3):
        self.P, self.N, self.B, self.M = P, N, B, M
        self.t, self.r = np.full((B, M), -1, np.int32), np.zeros(N, np.int32)
        self.wide = torch.full((B, M + stride), 77, dtype=I32, device=DEV)
        self.wide[:, :M] = -1
        self.table, self.ref = self.wide[:, :M], torch.zeros(N, dtype=I32, device=DEV)
        g = gen(seed)
        shape = (layers, N, hkv, P, D)
        pool = [torch.randint(0, 127, shape, generator=g, dtype=torch.uint8).to(DEV) for _ in range(2)]
        if kv == "fp8":
            self.kp, self.vp = (x.view(FP8) for x in pool)
        else:
            self.kp, self.vp = (x.to(BF) for x in pool)
        self.k, self.v = self.bytes(self.kp), self.bytes(self.vp)
        self.missing = torch.full((1,), 99, dtype=I32, device=DEV)
        self.ws = torch.full((2 * N + 8,), -9, dtype=I32, device=DEV)

    @staticmethod
    def bytes(x):
        return x.view(torch.uint8).cpu().numpy().copy()

    def same(self, pools=True):
        assert np.array_equal(self.table.cpu().numpy(), self.t)
        assert np.array_equal(self.ref.cpu().numpy(), self.r)
        assert (self.wide[:, self.M:] == 77).all()
        if pools:
            assert np.array_equal(self.bytes(self.kp), self.k) and np.array_equal(self.bytes(self.vp), self.v)

    def move(self, pairs):
        for x in (self.k, self.v):
            if pairs:
                a, b = np.array(pairs).T
                x[:, b] = x[:, a]

    def extend(self, C, pos, count):
        C.kv_pages_extend(self.table, self.ref, ints(pos), ints(count), self.P, self.missing)
        want = po.extend(self.t, self.r, pos, count, self.P)
        assert int(self.missing) == want
        return want

    def free(self, C, first, last):
        C.kv_pages_free(self.table, self.ref, ints(first), ints(last), self.P)
        po.free(self.t, self.r, first, last, self.P)

    def fork(self, C, src, dst, length):
        C.kv_pages_fork(self.table, self.ref, ints(src), ints(dst), ints(length), self.kp, self.vp,
                        self.missing, self.ws)
        want, moves = po.fork(self.t, self.r, src, dst, length, self.P)
        assert int(self.missing) == want
        self.move(moves)
        return want

    def compact(self, C):
        C.kv_pages_compact(self.table, self.ref, self.kp, self.vp, self.ws)
        self.move(po.compact(self.t, self.r))


def test_extend_gives_the_lowest_free_pages_in_order(native):
    p = Pages(5, 6, 20)
    p.extend(native, [0, 10, -1, 95, 3], [1, 30, 50, 1, 0])
    p.same()
    p.free(native, [0, 16, 0, 0, 0], [0, 32, 0, MAX, 0])
    p.same()
    p.extend(native, [0, 10, 4, 90, 16], [96, 30, 1, 40, 80])   # more than are free, and past the table
    p.same()
    assert int(p.missing) > 0
    p.extend(native, [-5, MAX, 200, MAX, -2 ** 31], [MAX, MAX, 1, 1, MAX])
    p.same()


@pytest.mark.parametrize("N", [1, 2, 63, 64, 65, 1000, 16384, 16385, 40000])
def test_extend_over_pool_sizes(native, N):
    """One workgroup scans up to 16,384 ids a step; 1,024 candidates at a time."""
    B, M = 37, 130
    p = Pages(B, M, N, hkv=1, layers=1) if N <= 1000 else None
    if p is None:  # no pools needed
        p = Pages(B, M, 4, layers=1)
        p.N, p.r, p.ref = N, np.zeros(N, np.int32), torch.zeros(N, dtype=I32, device=DEV)
    rng = np.random.default_rng(N)
    busy = rng.random(N) < 0.5
    p.r[busy] = 1
    p.ref.copy_(ints(p.r))
    for _ in range(3):
        p.extend(native, rng.integers(-3, M * 16, B), rng.integers(0, 1500, B))
        p.same(pools=False)


def test_free_ranges(native):
    p = Pages(4, 40, 200, P=32)
    p.extend(native, [0] * 4, [40 * 32] * 4)
    p.free(native, [5, 64, 1279, -2 ** 31], [1000, 96, MAX, 31])
    p.same()
    p.free(native, [0, 33, 0, 0], [0, 63, -1, 32])
    p.same()
    p.free(native, [-1, 5, MAX, -2 ** 31], [MAX, 4, MAX, MAX])
    p.same()
    assert tables_ok(p.t, p.r)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_fork_shares_whole_pages_and_copies_the_last(native, kv):
    p = Pages(8, 5, 30, hkv=3, kv=kv)
    p.extend(native, [0] * 4 + [-1] * 4, [80, 33, 16, 1, 0, 0, 0, 0])
    assert p.fork(native, [0, 0, 1, 2], [4, 5, 6, 7], [37, 48, 33, 0]) == 0
    p.same()
    p.free(native, [0] * 8, [MAX, 0, 0, 0, 0, 0, 0, 0])   # the parent ends, its children keep the pages
    p.same()
    # a child that held pages becomes another's copy; lengths past the source and past the table
    p.fork(native, [4, 1], [5, 3], [38, 79])
    p.same()
    p.fork(native, [6, 6], [0, 2], [MAX, -4])
    p.same()
    assert tables_ok(p.t, p.r)


def test_fork_refuses_and_runs_short(native):
    p = Pages(6, 4, 7)
    p.extend(native, [0, 0, -1, -1, -1, 0], [30, 20, 0, 0, 0, 5])
    # dst twice; src == dst; dst that is a source; outside the table
    assert p.fork(native, [0, 0, 1, 1, 6, 0, -1], [3, 3, 1, 0, 4, -1, 4], [20] * 7) == 7
    p.same()
    assert p.fork(native, [0, 0, 1], [2, 3, 4], [20, 17, 3]) == 1   # two pages are free for three
    p.same()
    assert p.fork(native, [0, 7], [2, 3], [20, 17]) == 1
    p.same()
    assert tables_ok(p.t, p.r)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("N,hkv,layers", [(1, 1, 1), (2, 1, 1), (7, 2, 3), (64, 1, 1), (300, 1, 2)])
def test_compact(native, N, hkv, layers, kv):
    rng = np.random.default_rng(N)
    B, M = 5, max(1, N // 4)
    p = Pages(B, M, N, hkv=hkv, layers=layers, kv=kv)
    for _ in range(4):
        p.extend(native, rng.integers(0, M * 16, B), rng.integers(0, M * 16, B))
        f = rng.integers(0, M * 16, B)
        p.free(native, f, f + rng.integers(0, M * 8, B))
        p.fork(native, [0], [1], [int(rng.integers(0, M * 16))])
        p.compact(native)
        p.same()
        p.compact(native)    # nothing left to move
        p.same()
    assert tables_ok(p.t, p.r)


def test_compact_large_allocation(native):
    """More ids than one scan step; sequences share pages."""
    N, B, M = 40001, 64, 400
    p = Pages(B, M, 4, layers=1, P=16)
    p.N = N
    rng = np.random.default_rng(1)
    ids = rng.permutation(N)[:20000]
    flat = np.full(B * M, -1, np.int32)
    flat[rng.permutation(B * M)[:22000]] = np.concatenate([ids, ids[:2000]])
    p.t = flat.reshape(B, M)
    p.r = np.bincount(flat[flat >= 0], minlength=N).astype(np.int32)
    p.table.copy_(ints(p.t))
    p.ref = ints(p.r)
    p.vp = (torch.arange(N, device=DEV) % 256).to(torch.uint8).view(N, 1, 1, 1).expand(N, 1, 16, D).contiguous()
    p.kp = (torch.arange(N, device=DEV) // 256).to(torch.uint8).view(N, 1, 1, 1).expand(N, 1, 16, D).contiguous()
    p.k, p.v = p.bytes(p.kp)[None], p.bytes(p.vp)[None]
    p.ws = torch.empty(2 * N + 8, dtype=I32, device=DEV)
    p.compact(native)
    p.k, p.v = p.k[0], p.v[0]
    p.same()


@pytest.mark.parametrize("hkv,P,layers", [(1, 16, 1), (4, 64, 3), (3, 32, 2)])
@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_copy(native, hkv, P, layers, kv):
    p = Pages(1, 1, 40, hkv=hkv, P=P, layers=layers, kv=kv)
    #      plain    same   twice         chain (5 is a source)   outside
    src = [0, 1, 2, 3, 4, 4, 5, 6, -1, 7, 40, 8, 2 ** 31 - 1]
    dst = [20, 21, 2, 22, 23, 22, 24, 5, 25, -1, 26, 40, 27]
    native.kv_pages_copy(p.kp, p.vp, ints(src), ints(dst))
    p.move(po.copy_pairs(src, dst, 40))
    p.same()
    four = p.kp[0], p.vp[0]     # pools of one layer, [N, Hkv, P, 256]
    native.kv_pages_copy(*four, ints([20]), ints([30]))
    p.k[0][30], p.v[0][30] = p.k[0][20], p.v[0][20]
    p.same()


def test_copy_many_pairs_past_32_bits(native):
    N = 9000
    kp = torch.zeros(N, 4, 128, D, dtype=BF, device=DEV)   # 2.36 GB
    kp.view(N, -1)[:, 0] = torch.arange(N, device=DEV).to(BF)
    kp.view(N, -1)[:, -1] = 1.0
    vp = torch.zeros_like(kp)
    vp.view(N, -1)[:, 5] = 2.0
    src = torch.arange(0, 3000, dtype=I32, device=DEV)
    want = kp.clone()
    want[6000:9000] = kp[:3000]
    native.kv_pages_copy(kp, vp, src, src + 6000)
    assert torch.equal(kp, want)


def test_a_life_of_an_allocation(native):
    """Random operations one after another, each against the model."""
    rng = np.random.default_rng(7)
    p = Pages(9, 7, 45, hkv=2, layers=2)
    for step in range(120):
        op = rng.integers(5)
        if op <= 1:
            p.extend(native, rng.integers(-20, 7 * 16, 9), rng.integers(0, 40, 9))
        elif op == 2:
            f = rng.integers(0, 7 * 16, 9)
            p.free(native, f, f + rng.integers(0, 70, 9))
        elif op == 3:
            p.fork(native, rng.integers(-1, 10, 3).tolist(), rng.integers(0, 9, 3).tolist(),
                   rng.integers(0, 7 * 16 + 9, 3))
        else:
            p.compact(native)
        p.same(pools=step % 10 == 9)
        assert tables_ok(p.t, p.r), (step, op)


def test_capture(native):
    """Free, extend, fork and compact in one graph; every replay against the model."""
    rng = np.random.default_rng(8)
    p = Pages(6, 5, 40)
    first, last, pos, count = (torch.zeros(6, dtype=I32, device=DEV) for _ in range(4))
    src, dst, length = (torch.zeros(2, dtype=I32, device=DEV) for _ in range(3))

    def step():
        native.kv_pages_free(p.table, p.ref, first, last, p.P)
        native.kv_pages_extend(p.table, p.ref, pos, count, p.P, p.missing)
        native.kv_pages_fork(p.table, p.ref, src, dst, length, p.kp, p.vp, p.missing, p.ws)
        native.kv_pages_compact(p.table, p.ref, p.kp, p.vp, p.ws)

    src.fill_(-1)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(6):
        a = [rng.integers(0, 80, 6) for _ in range(3)]
        for x, y in ((first, a[0]), (last, a[0] + a[1]), (pos, a[2]), (count, a[1] // 2)):
            x.copy_(ints(y))
        s, d, n = rng.integers(0, 6, 2), rng.integers(0, 6, 2), rng.integers(0, 80, 2)
        src.copy_(ints(s)), dst.copy_(ints(d)), length.copy_(ints(n))
        graph.replay()
        po.free(p.t, p.r, a[0], a[0] + a[1], p.P)
        po.extend(p.t, p.r, a[2], a[1] // 2, p.P)
        want, moves = po.fork(p.t, p.r, s.tolist(), d.tolist(), n, p.P)
        p.move(moves)
        p.move(po.compact(p.t, p.r))
        assert int(p.missing) == want
        p.same()
