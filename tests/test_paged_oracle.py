"""The CPU model of the paged cache (oracle/paged_oracle.py) against the contiguous oracle's independent
fp64 loops on a gathered cache, and the page model's invariants."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as po
from paged_cases import Batch, D, tables_ok
from refmath import attention_fp64, sigmoid64


@pytest.mark.parametrize("P,lens,R", [(16, [0, 5, 40], 1), (32, [31, 33], 3)])
def test_decode_equals_contiguous_attention(P, lens, R):
    c = Batch(1, lens, R=R, hq=4, hkv=2, P=P)
    out, tol = c.exact()
    for b, n in enumerate(lens):
        for t in range(R):
            L = n + t + 1
            pages = c.table[b].long()
            K = c.kp[pages[:-1]].permute(1, 0, 2, 3).reshape(2, -1, D)[:, :L].float().numpy()
            V = c.vp[pages[:-1]].permute(1, 0, 2, 3).reshape(2, -1, D)[:, :L].float().numpy()
            i = b * R + t
            want = attention_fp64(c.q[i].view(4, D).float().numpy(), K, V, 2, L, 1 / 16)
            want = want * sigmoid64(c.qg[i].view(4, 2 * D)[:, D:].float().numpy())
            assert np.abs(out[i] - want).max() < 1e-12
            assert (tol[i] > 0).all()


def test_attended():
    row = [3, -1, 0, 9]
    assert po.attended(20, 4, 8, 4, row) == list(range(8)) + list(range(16, 21))
    assert po.attended(20, 4, 8, 4, row, window=3, sinks=2) == [0, 1, 18, 19, 20]
    assert po.attended(100, 4, 8, 4, row, window=5) == []          # past the table
    assert po.attended(30, 4, 8, 4, row, window=100, sinks=0) == po.attended(30, 4, 8, 4, row)


def test_prep_rotation_keeps_pairs():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 2 * D, generator=g)
    k = torch.randn(2, D, generator=g)
    f = 1.0 / 1e4 ** (np.arange(4) / 4)
    q, kk, v, qm, km = po.prep(x, k, k, np.zeros(D), np.zeros(D), f, [7], 2, 1, 1, 0.0)
    n = x[:, :D].numpy() / np.sqrt((x[:, :D].numpy() ** 2).mean(-1, keepdims=True))
    assert np.allclose(np.hypot(q[:, 0, :4], q[:, 0, 4:8]), np.hypot(n[:, :4], n[:, 4:8]), atol=1e-6)
    assert np.allclose(q[:, 0, 8:], n[:, 8:], atol=1e-6)
    z = po.prep(x, k, k, np.zeros(D), np.zeros(D), f, [0, 0], 1, 1, 1, 0.0)[0]
    assert np.allclose(z[0, 0], n[0], atol=1e-6)  # position 0: no rotation


def test_page_model_keeps_counts():
    rng = np.random.default_rng(3)
    B, M, N, P = 6, 5, 20, 16
    table, ref = np.full((B, M), -1, np.int32), np.zeros(N, np.int32)
    for step in range(200):
        op = rng.integers(4)
        if op == 0:
            po.extend(table, ref, rng.integers(-1, M * P, B), rng.integers(0, 40, B), P)
        elif op == 1:
            f = rng.integers(0, M * P, B)
            po.free(table, ref, f, f + rng.integers(0, 60, B), P)
        elif op == 2:
            s, d = rng.integers(-1, B + 1, 3), rng.integers(0, B, 3)
            po.fork(table, ref, s.tolist(), d.tolist(), rng.integers(0, M * P + 9, 3), P)
        else:
            po.compact(table, ref)
            U = int((ref > 0).sum())
            assert (ref[:U] > 0).all() and (ref[U:] == 0).all()
        assert tables_ok(table, ref), (step, op)
