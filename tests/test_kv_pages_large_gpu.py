"""The operations on pages at sizes where they take other paths than in test_kv_pages_gpu.py: forks of more than 8,192
table entries (the entries are shared by a launch of their own), copies whose every byte tells its place."""
import numpy as np
import pytest
import torch

from paged_cases import D, tables_ok
from test_kv_pages_gpu import DEV, Pages, ints

pytestmark = pytest.mark.gpu
I32 = torch.int32


def held(p, native, lens):
    """Positions [0, lens[b]) of every sequence mapped."""
    assert p.extend(native, [0] * p.B, lens) == 0


@pytest.mark.parametrize("m,M", [(64, 128), (60, 200), (100, 82), (1, 9000)])
@pytest.mark.parametrize("spare", [0, 30, 200])
def test_forks_on_both_sides_of_8192_entries(native, m, M, spare):
    """Pairs that are refused, dst sequences that hold pages (some shared with their new source), lengths past the source
    and past the table, too few free pages for the partial ones."""
    rng = np.random.default_rng(m + spare)
    B = 2 * m + 3
    lens = [int(x) for x in rng.integers(1, 16 * min(M, 60), B)]
    for b in range(m, 2 * m, 3):
        lens[b] = 0
    N = sum(-(-n // 16) for n in lens) + spare
    p = Pages(B, M, N, layers=1)
    held(p, native, lens)
    p.same(pools=False)
    src, dst = rng.integers(0, m, m), m + rng.permutation(m)
    length = np.array([max(1, lens[s] + int(x)) for s, x in zip(src, rng.integers(-40, 20, m))])
    if m > 8:
        src[3], dst[5], dst[7], src[9] = B, -1, dst[8], 2 ** 31 - 1  # outside, outside, twice a dst, outside
        dst[11] = src[12]                                            # a source
        length[13], length[14], length[15] = 2 ** 31 - 1, 0, -5
    else:
        length[0] = 16 * M
    bad = p.fork(native, src.tolist(), dst.tolist(), length)
    assert bad >= (6 if m > 8 else 0)
    p.same()
    assert tables_ok(p.t, p.r)
    # once more onto the same places: their pages are shared ones now
    p.fork(native, src.tolist(), dst[::-1].tolist(), length // 2 + 3)
    p.same()
    assert tables_ok(p.t, p.r)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_every_byte_of_a_copy(native, kv):
    """Pools past 2^32 bytes whose 4-byte words all differ: pages of four 32 KB pieces, of one and a half, of less than
    one, in every layer."""
    dtype = torch.bfloat16 if kv == "bf16" else torch.uint8
    width = 2 if kv == "bf16" else 1
    for layers, N, hkv, P in ((1, 34000, 4, 128 // width), (3, 500, 3, 64 // width), (2, 900, 1, 16)):
        words = layers * N * hkv * P * D * width // 4
        pools = []
        for k in range(2):
            w = torch.arange(words, dtype=I32, device=DEV)
            pools.append((w if k == 0 else ~w).view(dtype).view(layers, N, hkv, P, D))
        rng = np.random.default_rng(layers)
        ids = rng.permutation(N)
        m = N * 2 // 5
        src, dst = ids[:m], ids[m:2 * m]
        page = hkv * P * D * width // 4
        want = []
        for x in pools:
            y = x.view(I32).view(layers, N, page).clone()
            y[:, torch.from_numpy(dst).to(DEV)] = y[:, torch.from_numpy(src).to(DEV)]
            want.append(y)
        native.kv_pages_copy(*pools, ints(src), ints(dst))
        for x, y in zip(pools, want):
            assert torch.equal(x.view(I32).view(layers, N, page), y), (layers, N)
        del pools, want, x, y, w
        torch.cuda.empty_cache()
