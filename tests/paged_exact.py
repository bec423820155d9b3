"""Large batches for the tests of the paged decode, made on the GPU, and the definition in float64 there, for what the
loops of oracle/paged_oracle.py take too long: row by row over the attended positions, written apart from both the
kernels and that model."""
import numpy as np
import torch

from paged_cases import BF, D, FP8, KV_SCALE, Batch


class Big(Batch):
    """A Batch (paged_cases.py) whose tensors are on the GPU."""

    def __init__(self, seed, lens, R=1, hq=24, hkv=4, P=16, kv="bf16", window=0, sinks=0, spare=2, extra_m=1,
                 trim=True):
        self.R, self.hq, self.hkv, self.P, self.kv = R, hq, hkv, P, kv
        self.window, self.sinks, self.pos = window, sinks, list(lens)
        B, rng = len(lens), np.random.default_rng(seed)
        M = max((n + R - 1) // P for n in lens) + 1 + extra_m
        last = (np.array(lens)[:, None] + R - 1) // P
        j, lo = np.arange(M)[None], np.maximum(np.array(lens)[:, None] + 1 - window, 0) // P
        need = (j <= last) & (np.array(lens)[:, None] >= 0)
        if window and trim:
            need &= (j >= lo) | (j * P < sinks)
        N = int(need.sum()) + spare
        table = np.full((B, M), -1, np.int32)
        table[need] = rng.permutation(N)[: need.sum()]
        self.table, self.N, self.M, self.B = torch.from_numpy(table), N, M, B
        g = torch.Generator(device="cuda").manual_seed(seed)
        k, v = (torch.randn(N, hkv, P, D, generator=g, device="cuda") for _ in range(2))
        if kv == "fp8":
            self.kp, self.vp = ((x / KV_SCALE).clamp(-448, 448).to(FP8) for x in (k, v))
        else:
            self.kp, self.vp = k.to(BF), v.to(BF)
        self.q = torch.randn(B * R, hq * D, generator=g, device="cuda").to(BF)
        self.qg = torch.randn(B * R, hq * 2 * D, generator=g, device="cuda").to(BF)

    def poison(self, bad=float("nan")):
        """Puts `bad` into every row of both pools that no row of the batch attends."""
        keep = np.zeros((self.N, self.P), bool)
        j = np.arange(self.M * self.P)
        for b, p0 in enumerate(self.pos):
            for t in range(self.R if p0 >= 0 else 0):
                p, page = p0 + t, self.table[b].numpy()[j // self.P]
                on = (j <= p) & (page >= 0) & (page < self.N)
                if self.window:
                    on &= (j < self.sinks) | (j >= p + 1 - self.window)
                keep[page[on], j[on] % self.P] = True
        off = torch.from_numpy(~keep).to(self.kp.device)
        for x in (self.kp, self.vp):
            y = x.float().permute(0, 2, 1, 3).contiguous()
            y[off] = bad
            x.copy_(y.permute(0, 2, 1, 3).to(x.dtype))


def decode(c, kp, vp, table, q, qg):
    """(out, bound) [B*R, Hq, 256] of a Batch (paged_cases.py) whose tensors are on the GPU; NaN for idle rows. The
    bound counts the roundings of a correct fp32 evaluation, as oracle/paged_oracle.py:decode lists them."""
    dev, G, scale = q.device, c.hq // c.hkv, c.scale
    cap = c.M * c.P
    out = torch.full((c.B * c.R, c.hq, D), float("nan"), dtype=torch.float64, device=dev)
    tol = torch.zeros_like(out)
    kp, vp = (x.float() if x.dtype == torch.bfloat16 else x for x in (kp, vp))
    k8 = kp.dtype == torch.float8_e4m3fn
    for b, p0 in enumerate(c.pos):
        for t in range(c.R if p0 >= 0 else 0):
            i, p = b * c.R + t, p0 + t
            j = torch.arange(min(p + 1, cap), device=dev)
            page = table[b].long()[j // c.P]
            keep = (page >= 0) & (page < c.N)
            if c.window:
                keep &= (j < c.sinks) | (j >= p + 1 - c.window)
            j, page = j[keep], page[keep]
            if j.numel() == 0:
                out[i] = 0
                continue
            if k8:
                K, V = (x.view(torch.uint8)[page, :, j % c.P].view(x.dtype).double() for x in (kp, vp))
            else:
                K, V = (x[page, :, j % c.P].double() for x in (kp, vp))
            K, V = (x.permute(1, 0, 2).contiguous() * scale for x in (K, V))           # [hkv, n, 256]
            x = q[i].view(c.hkv, G, D).double()
            KT = K.transpose(1, 2).contiguous()
            w = torch.softmax(x @ KT / 16, -1)
            gate = torch.sigmoid(qg[i].view(c.hkv, G, 2 * D)[..., D:].double())
            o = (w @ V) * gate
            A = (x.abs() @ KT.abs()).amax(-1, keepdim=True) / 16
            eps = 2 * 262 * 2.0 ** -24 * A + 2.0 ** -22 + 2.0 ** -16 + 2 * (j.numel() + 64) * 2.0 ** -24 + 2.0 ** -20
            out[i] = o.reshape(c.hq, D)
            tol[i] = (eps * (w @ V.abs()) * gate + 2.0 ** -8 * o.abs() + 1e-37).reshape(c.hq, D)
    return out, tol
