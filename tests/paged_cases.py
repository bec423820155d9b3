"""Seeded inputs for the tests of the paged KV cache (CPU tensors; the GPU tests move them)."""
from __future__ import annotations

import numpy as np
import torch

BF = torch.bfloat16
FP8 = torch.float8_e4m3fn
D = 256
KV_SCALE = 1.0 / 16


def gen(seed):
    return torch.Generator().manual_seed(seed)


class Batch:
    """Random pools, a table that maps the pages that ``spans`` of positions need in random order, q and gate
    rows. lens[b]: position of sequence b's first row (< 0: idle). Every value of a page is random, also
    those past a sequence's end; unmapped entries are -1."""

    def __init__(self, seed, lens, R=1, hq=24, hkv=4, P=16, kv="bf16", window=0, sinks=0, spare=2, extra_m=1,
                 trim=True, scale=1.0):
        g = gen(seed)
        self.R, self.hq, self.hkv, self.P, self.kv = R, hq, hkv, P, kv
        self.window, self.sinks, self.pos = window, sinks, list(lens)
        B = len(lens)
        need = []
        for n in lens:
            last = (n + R - 1) // P
            lo = max(0, n + 1 - window) // P if window and trim else 0
            need.append([j for j in range(last + 1) if n >= 0 and (j >= lo or j * P < sinks)])
        M = max(max(s, default=0) for s in need) + 1 + extra_m
        N = sum(map(len, need)) + spare
        ids = torch.randperm(N, generator=g).tolist()
        self.table = torch.full((B, M), -1, dtype=torch.int32)
        for b, s in enumerate(need):
            for j in s:
                self.table[b, j] = ids.pop()
        self.N, self.M, self.B = N, M, B
        k, v = torch.randn(N, hkv, P, D, generator=g), torch.randn(N, hkv, P, D, generator=g)
        if kv == "fp8":
            self.kp, self.vp = ((x / KV_SCALE).clamp(-448, 448).to(FP8) for x in (k, v))
        else:
            self.kp, self.vp = k.to(BF), v.to(BF)
        self.q = (torch.randn(B * R, hq * D, generator=g) * scale).to(BF)
        self.qg = torch.randn(B * R, hq * 2 * D, generator=g).to(BF)

    @property
    def scale(self):
        return KV_SCALE if self.kv == "fp8" else 1.0

    def exact(self):
        from oracle import paged_oracle as po
        return po.decode(self.q.float().numpy(), self.kp.float().numpy(), self.vp.float().numpy(),
                         self.table.numpy(), self.pos, self.qg.float().numpy(), self.R, self.window,
                         self.sinks, self.scale, self.scale)

    def poison(self, bad=float("nan")):
        """Puts `bad` into every row of both pools that no row of the batch attends."""
        from oracle import paged_oracle as po
        keep = np.zeros((self.N, self.P), bool)
        for b, p0 in enumerate(self.pos):
            for t in range(self.R if p0 >= 0 else 0):
                for j in po.attended(p0 + t, self.M, self.P, self.N, self.table[b], self.window, self.sinks):
                    keep[self.table[b, j // self.P], j % self.P] = True
        for x in (self.kp, self.vp):
            y = x.float().permute(0, 2, 1, 3).contiguous()
            y[~torch.from_numpy(keep)] = bad
            x.copy_(y.permute(0, 2, 1, 3).to(x.dtype))


def tables_ok(table, ref):
    """ref[i] is the number of entries that name page i."""
    t, r = np.asarray(table), np.asarray(ref)
    named = t[(t >= 0) & (t < len(r))]
    return np.array_equal(np.bincount(named, minlength=len(r)), r)
