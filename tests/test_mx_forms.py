"""CPU tests of how the product on 4-bit weights chooses its kernels: what holds for every call whatever the choice's
constants are, and the refusals of the call of a given kernel. No kernel runs here."""
import random

import pytest
import torch

BF, U8 = torch.bfloat16, torch.uint8
FP8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
ROWS, KERNELS = -1, range(-1, 7)
COLS = (256, 256, 160, 128, 256, 128, 64)  # weight rows of a tile, kernels 0 .. 6


def calls(count=400):
    rng = random.Random(5)
    lg = lambda lo, hi: round(lo * (hi / lo) ** rng.random())  # noqa: E731
    return [(lg(1, 4096), lg(1, 40000), 32 * lg(1, 700)) for _ in range(count)]


def test_up_to_16_rows_stream_the_weight(native):
    """Or a row's bits would depend on the others."""
    for n, N, K in calls(100) + [(16, 2 ** 24, 32), (16, 34816, 2 ** 20), (16, 1, 2 ** 20)]:
        for ws in (0, 1 << 40):
            assert native._gemm_mx4_form(min(n, 16), N, K, ws)[:3] == (ROWS, 1, N)
        assert native.mx4_ws_bytes(min(n, 16), N, K) == 0


def test_cuts_and_workspaces(native):
    """A cut leaves whole tiles to the first kernel and at least a weight row to the second; a split's partial sums fit
    the workspace, and the one that is asked for gives the choice that any larger one would."""
    cut_calls = split_calls = 0
    for n, N, K in calls() + [(128, 5120, 17408), (32, 34815, 5120), (2048, 34816, 5120)]:
        need = native.mx4_ws_bytes(n, N, K)
        free = native._gemm_mx4_form(n, N, K, 1 << 40)
        assert native._gemm_mx4_form(n, N, K, need) == free
        for ws in (0, need // 2, need):
            kernel, splits, cut, rest, rest_splits = native._gemm_mx4_form(n, N, K, ws)
            assert kernel in KERNELS and 0 < cut <= N
            parts = [(splits, cut)]
            if cut < N:
                cut_calls += 1
                assert cut % COLS[kernel] == 0 and cut % 16 == 0 and splits == 1 and rest in KERNELS
                parts = [(rest_splits, N - cut)]
            for s, rows in parts:
                split_calls += s > 1
                assert s >= 1 and (s == 1 or s * n * (-(-rows // 16) * 16) * 4 <= ws)
    assert cut_calls and split_calls


def test_every_kernel_is_some_calls(native):
    """None of them is there for nothing, and both parts of K that a workspace holds occur."""
    seen, split = set(), set()
    for n, N, K in calls(2000):
        k, s, cut, k2, s2 = native._gemm_mx4_form(n, N, K, 1 << 40)
        seen |= {k} if cut == N else {k, k2}
        split |= {s} if cut == N else {s, s2}
    assert seen == set(KERNELS) and split >= {1, 2, 4}


def test_a_given_kernel_refuses(native):
    def z(*s, dt=BF):
        return torch.zeros(*s, dtype=dt)
    n, N, K = 20, 40, 1024
    args = dict(wq=z(native.mx4_bytes(N, K), dt=U8), xq=z(n, K, dt=FP8), xs=z(n, K // 32, dt=E8), out=z(n, N),
                ws=z(2 * n * 48 * 4, dt=U8))

    def call(kernel, splits, **k):
        native._gemm_mx4_as(kernel, splits, *{**args, **k}.values())
    for kernel, splits in ((-2, 1), (7, 1), (0, 2), (-1, 2), (3, 0), (3, 3), (3, 4), (3, 16), (6, 3), (2 ** 40, 1)):
        with pytest.raises(RuntimeError, match="does not take"):
            call(kernel, splits)  # 8 tiles of K are no 16 parts, nor 3 times 4; 3 or 4 need a larger workspace
    for ws in (None, args["ws"][:-16]):
        with pytest.raises(RuntimeError, match="does not take"):
            call(3, 2, ws=ws)
    with pytest.raises(RuntimeError, match="20 rows"):
        call(0, 1, out=z(19, N))
    for kernel, splits in ((-1, 1), (0, 1), (3, 2), (5, 2), (6, 1)):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            call(kernel, splits)
