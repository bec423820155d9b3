"""Infinities and NaN among the cache values that rows of the paged decode attend. A dim of V in which a row attends
+inf is +inf, -inf is -inf, both or a NaN is NaN, wherever the value lies (a tile that every row attends whole, the
rows' last tile, a window's edge) and whatever the call's form and number of rows are. Every other value of the
output keeps its bits."""
import numpy as np
import pytest
import torch

import paged_exact
from paged_cases import BF, D
from paged_exact import Big
from test_paged_decode_gpu import DEV, Call

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")

# (sequences, lengths from, to, hq, hkv, R, P, window, sinks): slices of 32; of more, four waves each; persistent waves
FORMS = {"short": (3, 30, 200, 6, 1, 4, 16, 0, 0), "short_8_rows": (3, 40, 200, 12, 2, 8, 32, 0, 0),
         "waves": (24, 150, 500, 12, 4, 4, 32, 0, 0), "waves_two_tiles": (24, 150, 500, 32, 4, 4, 16, 0, 0),
         "waves_window": (24, 150, 900, 12, 4, 4, 16, 200, 40), "batch": (72, 300, 1900, 8, 4, 4, 16, 0, 0),
         "batch_two_tiles": (72, 300, 1900, 32, 4, 4, 64, 0, 0),
         "batch_window": (90, 300, 3000, 12, 4, 8, 16, 900, 70)}


def make(form, kv, seed=1):
    n, lo, hi, hq, hkv, R, P, window, sinks = FORMS[form]
    lens = [int(x) for x in np.random.default_rng(seed).integers(lo, hi, n)]
    return Big(seed, lens, R=R, hq=hq, hkv=hkv, P=P, kv=kv, window=window, sinks=sinks, trim=False)


def attends(c, p, j):
    return j <= p and (not c.window or j < c.sinks or j >= p + 1 - c.window)


def same(x, y):
    """Equal bits, NaN of any payload."""
    return torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(7.0, INF, -INF), y.nan_to_num(7.0, INF, -INF))


def places(c, b):
    """Positions of sequence b: tiles that its rows attend whole, the last tile, what only some rows attend."""
    n, R = c.pos[b], c.R
    at = [0, 5, 33, n // 2, n - 40, n - 1, n, n + 1, n + R - 1]
    if c.window:
        at += [max(n + 1 - c.window, 0), max(n + 2 - c.window, 0), max(n + 40 - c.window, 0), c.sinks - 1]
    return at


def put(c, b, j, dims, value):
    x = c.vp.view(torch.uint8) if c.kv == "fp8" else c.vp
    bad = 0x7f if c.kv == "fp8" else value          # (E4M3FN: one NaN, no infinity)
    x[int(c.table[b, j // c.P]), :, j % c.P, dims] = bad


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("form", list(FORMS))
def test_attended_values_that_are_not_finite(native, form, kv):
    c = make(form, kv)
    k = Call(c)
    want = k.run(native).view(c.B, c.R, c.hq, D).clone()
    kinds = torch.zeros(c.B, c.R, D, dtype=torch.int32)
    for b in range(c.B):
        at = places(c, b)
        for i, value in enumerate((INF, -INF, NAN, INF, -INF)):
            dims = slice(12 * i, 12 * i + 9) if i < 4 else slice(20 + 10 * (b % 3), 50)  # the last meets others
            put(c, b, at[(b + 2 * i) % len(at)], dims, value)
        for j in sorted(set(at)):
            row = c.vp[int(c.table[b, j // c.P]), 0, j % c.P].float().cpu()
            kind = torch.where(row.isnan(), 4, torch.where(row == INF, 1, torch.where(row == -INF, 2, 0))).int()
            for t in range(c.R):
                if attends(c, c.pos[b] + t, j):
                    kinds[b, t] |= kind
    value = torch.tensor([0.0, INF, -INF] + [NAN] * 5, dtype=BF)[kinds.long()].to(DEV)[:, :, None].expand_as(want)
    want = torch.where((kinds > 0).to(DEV)[:, :, None], value, want)
    got = Call(c).run(native).view_as(want)
    for b in range(c.B):
        for t in range(c.R):
            assert same(got[b, t], want[b, t]), (b, t, c.pos[b])
    # the same rows in calls of one row each
    q, qg = c.q.view(c.B, c.R, -1), c.qg.view(c.B, c.R, -1)
    R, lens = c.R, c.pos
    for t in range(R):
        c.R, c.q, c.qg, c.pos = 1, q[:, t].contiguous(), qg[:, t].contiguous(), [n + t for n in lens]
        assert same(Call(c).run(native).view(c.B, c.hq, D), want[:, t]), t


@pytest.mark.parametrize("form", list(FORMS))
def test_scores_of_minus_infinity(native, form):
    """A row whose attended scores all are -inf has no softmax: NaN, not the 0 of a row that attends nothing. Beside finite
    scores they weigh nothing. One score of +inf: NaN."""
    c = make(form, "bf16")
    c.q.view(-1, c.hq, D)[..., 0].abs_().clamp_(min=0.25)
    clean = Call(c).run(native).view(c.B, c.R, c.hq, D).clone()
    for b, n in enumerate(c.pos):
        # every third sequence: all keys up to row 0's, every second one of them, none; the next: no page at all
        for j in range(0, n + 1, 1 + b % 3) if b % 3 < 2 else ():
            c.kp[int(c.table[b, j // c.P]), :, j % c.P, 0] = -INF
    if c.B > 5:
        c.table[5] = -1
        c.kp[int(c.table[8, c.pos[8] // c.P]), :, c.pos[8] % c.P, 0] = INF
    k = Call(c)
    got = k.run(native).view_as(clean)
    want, _ = paged_exact.decode(c, k.kp, k.vp, k.table, k.q, k.qg)
    want = want.view_as(clean)
    for b, n in enumerate(c.pos):
        for t in range(c.R):
            if c.B > 5 and b == 5:
                assert (got[b, t] == 0).all()
            elif c.B > 5 and b == 8:
                assert got[b, t].isnan().all()
            elif b % 3 == 2:
                assert same(got[b, t], clean[b, t]), (b, t)
            elif all(j <= n for j in range(n + t + 1) if attends(c, n + t, j)) and b % 3 == 0:
                assert got[b, t].isnan().all(), (b, t)
            else:
                # sum |q k| / 16 of a finite score is below 20 (256 products of unit normals: 163 / 16 on average, its
                # deviation 0.8), so weights are off by 2 * 262 * 2^-24 * 20 + 2^-15 < 2^-10, times |V| < 6; then one rounding
                tol = 6 * 2.0 ** -10 + 2.0 ** -8 * want[b, t].abs()
                assert ((got[b, t].double() - want[b, t]).abs() <= tol).all(), (b, t)
