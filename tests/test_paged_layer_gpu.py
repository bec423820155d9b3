"""The paged operators as a decode loop uses them together (PagedCache, PagedGatedAttention): extend, norm + RoPE
into pages and decode in every pass, forks, freed windows, ended sequences and compaction between passes.
The same passes over a table that maps everything once, and never changes, give the same bits."""
import pytest
import torch

from attn_cases import norm_weights
from paged_cases import BF, D, KV_SCALE, gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
MAX = 2 ** 31 - 1


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Loop:
    """`layers` layers and the passes' inputs. fixed: every sequence owns its pages from the start."""

    B, M = 6, 8

    def __init__(self, fixed, P=16, hq=8, hkv=2, layers=2, kv="bf16", window=0, sinks=0, n_max=8, seed=5):
        from qengine_amd.layer import PagedCache, PagedGatedAttention
        self.fixed, self.P, self.hq, self.window, self.sinks = fixed, P, hq, window, sinks
        s = KV_SCALE if kv == "fp8" else 1.0
        self.cache = PagedCache(hkv, self.M * P, self.B, self.B * self.M if fixed else self.B * self.M // 2 + 4, P,
                                layers, kv == "fp8", s, s)
        if fixed:
            self.cache.table.copy_(torch.arange(self.B * self.M).view(self.B, self.M))
            self.cache.ref.fill_(1)
        g = gen(seed)
        self.layers = []
        for i in range(layers):
            qnw, knw = norm_weights(g)
            self.layers.append(PagedGatedAttention(self.cache, i, hq, qnw, knw, n_max=n_max, window=window,
                                                   sinks=sinks, share=self.layers[0] if i else None))
        self.g = g

    def rows(self, R):
        return [torch.randn(self.B * R, l.width, generator=self.g).to(BF).to(DEV) for l in self.layers]

    def step(self, pos, R, proj, out):
        """One pass: pos int32 [B] on the device, proj and out per layer."""
        if not self.fixed:
            self.cache.extend(pos, torch.full_like(pos, R))
        for l, p, o in zip(self.layers, proj, out):
            l(p, pos, o)

    def fork(self, src, dst, length):
        if not self.fixed:
            self.cache.fork(ints([src]), ints([dst]), ints([length]))
            return
        for x in (self.cache.kp, self.cache.vp):
            x = x.view(torch.uint8)
            x[:, dst * self.M:(dst + 1) * self.M] = x[:, src * self.M:(src + 1) * self.M]

    def end(self, b):
        if not self.fixed:
            self.cache.free(ints([0 if i == b else MAX for i in range(self.B)]), ints([MAX] * self.B))

    def tidy(self, pos):
        """Frees what lies behind the windows, then compacts."""
        if self.fixed:
            return
        if self.window:
            self.cache.free(ints([self.sinks] * self.B), ints([max(p + 1 - self.window, 0) for p in pos]))
        self.cache.compact()


def script(loop):
    """Passes of 1..8 rows over sequences that start, fork and end; (outputs, pages in use) of each."""
    pos, res = [0, 0, 0, -1, -1, -1], []
    for i, R in enumerate([8, 5, 1, 8, 8, 1, 2, 8, 8, 3, 1, 1, 8, 8, 4, 1]):
        if i == 3:      # three that go on from two shared beginnings
            for src, dst in ((0, 3), (0, 4), (1, 5)):
                loop.fork(src, dst, pos[src])
                pos[dst] = pos[src]
        if i == 8:
            loop.end(1)
            pos[1] = -1
        if i == 11:     # the ended one's place is taken by a shorter beginning of another
            loop.fork(4, 1, 21)
            pos[1] = 21
        out = [torch.full((loop.B * R, loop.hq * D), 7.0, dtype=BF, device=DEV) for _ in loop.layers]
        loop.step(ints(pos), R, loop.rows(R), out)
        for b, p in enumerate(pos):
            if p < 0:
                assert all((o[b * R:(b + 1) * R] == 7).all() for o in out)
            else:
                assert all(o[b * R:(b + 1) * R].isfinite().all() for o in out)
        pos = [p + R if p >= 0 else p for p in pos]
        loop.tidy(pos)
        if not loop.fixed:
            assert int(loop.cache.missing) == 0
        res.append((out, int((loop.cache.ref > 0).sum())))
    return res


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("P", [16, 32])
@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 3)])
def test_a_moving_table_changes_no_bit(native, P, kv, window, sinks):
    got = script(Loop(False, P=P, kv=kv, window=window, sinks=sinks))
    want = script(Loop(True, P=P, kv=kv, window=window, sinks=sinks))
    for (a, _), (b, _) in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    if window and P == 16:  # a sequence holds its first page and those its window touches
        assert got[-1][1] <= Loop.B * (1 + 3)


def test_against_the_contiguous_layer(native):
    """The same rows through GatedAttention, which rounds q and k after every op of norm and RoPE (at most four
    further roundings each) and the output three times instead of once. A rounding's error is at most 2^-8
    of a value, 2^-8 / sqrt(3) in the mean of squares: eight of them in a product of 256 terms of that size
    move a score by about 0.0064 sqrt(256) / 16, an output by as much of its size, and two roundings of its
    own by 0.0032: 0.7% together. Four times that is allowed, in the mean of squares of a row."""
    from qengine_amd.layer import GatedAttention
    hq, hkv, T = 24, 4, 100
    loop = Loop(False, hq=hq, hkv=hkv, layers=1)
    lay = loop.layers[0]
    ref = GatedAttention(hq, hkv, T, lay.q_norm, lay.k_norm)
    pos = 0
    for R in [8, 8, 1, 5, 8, 8, 8, 8, 2, 8, 8, 8, 1, 1]:
        proj = loop.rows(R)
        out = torch.empty(loop.B * R, hq * D, dtype=BF, device=DEV)
        loop.step(ints([-1, -1, pos, -1, -1, -1]), R, proj, [out])
        want = torch.empty(R, hq * D, dtype=BF, device=DEV)
        ref(proj[0][2 * R:3 * R], ints([pos]), want)
        a, b = out[2 * R:3 * R].double(), want.double()
        err = ((a - b).square().mean(1) / b.square().mean(1)).sqrt().max()
        assert err < 4 * 0.007, (pos, R, float(err))
        pos += R


def test_a_captured_pass(native):
    """A pass with its extend, the release of what lies behind the window and the advance of the positions as one
    graph, replayed with eager work between, against the same passes run eagerly."""
    steps, R, window, sinks = 12, 3, 20, 4

    def setup():
        loop = Loop(False, window=window, sinks=sinks, n_max=R)
        pos = ints([0, 5, -1, 30, 0, 63])
        proj = [torch.zeros(loop.B * R, l.width, dtype=BF, device=DEV) for l in loop.layers]
        out = [torch.full((loop.B * R, loop.hq * D), 7.0, dtype=BF, device=DEV) for _ in loop.layers]
        first = ints([sinks] * loop.B)

        def body():
            loop.step(pos, R, proj, out)
            pos.add_(R * (pos >= 0).to(torch.int32))
            loop.cache.free(first, pos + (1 - window))

        return loop, pos, proj, out, body

    def feed(loop, proj):
        for p, x in zip(proj, loop.rows(R)):
            p.copy_(x)

    want = []
    loop, pos, proj, out, body = setup()
    for _ in range(steps):
        feed(loop, proj)
        body()
        want.append([o.clone() for o in out] + [loop.cache.table.clone(), pos.clone()])

    loop, pos, proj, out, body = setup()
    start = [x.clone() for x in (pos, loop.cache.table, loop.cache.ref, *out)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        body()  # warm-up
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        body()
    for x, s in zip((pos, loop.cache.table, loop.cache.ref, *out), start):
        x.copy_(s)
    for i in range(steps):
        feed(loop, proj)
        graph.replay()
        torch.cuda.synchronize()
        got = [*out, loop.cache.table, pos]
        assert all(torch.equal(a, b) for a, b in zip(got, want[i])), i
        torch.randn(1000, device=DEV).sum()
