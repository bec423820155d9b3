"""Host-side mirror of the reference decode loop's gated-attention branch on the gfx950 ops.

The reference runs, per full-attention layer and pass of n rows (python/qengine/engine.py:448-458):
  pr  = fused projection rows [qg (Hq*2*256) | k (Hkv*256) | v (Hkv*256)]
  attn_prep(pr[:, :q0], pr[:, q0:k1], pr[:, k1:], q_norm, k_norm, inv_freq, pos, q, kc, vc, eps)
  attn_decode(q, kc, vc, pos, pr[:, :q0], part_o, part_ml, out)
with inv_freq built on the CPU in fp32 and moved (engine.py:409-410), per-layer kc/vc
[Hkv, max_len, 256] (engine.py:419) and a shared q / part_o / part_ml scratch (engine.py:405-408).
GatedAttention owns the same buffers and issues the same work, by default as the reference's two
calls; fused=True issues the fused attn_prep_decode instead (two launches instead of three,
bit-identical results; on gfx950 up to 0.7 us faster per layer-call for one row on caches up to
8k positions, up to 1.2 us slower for two rows and at 16k, where the fused kernel's single-slot
KV tile loop costs more than the launch it saves). It allocates only at construction, so a pass
can be captured in a hipGraph.

PagedCache and PagedGatedAttention are the same for a batch of sequences over one paged cache: a pass
extends the tables once, then every layer issues attn_prep_paged and attn_decode_paged. The reference
serves one sequence and has no counterpart.

MX4Linear and MX4MLP are linear layers on 4-bit weights (microscaled E2M1 codes, where the reference's W4Linear has
integers: python/qengine/engine.py:74-186) for decode rows and prompt chunks alike: MX4MLP is the second half of
Engine._layer (engine.py:460-466), norm with the residual's addition, gate and up, SwiGLU, down, in four calls.
"""
from __future__ import annotations

import torch

from . import (_C, alloc_mx4, alloc_mx8, alloc_pages_ws, alloc_partials, default_paged_splits, default_splits)

HEAD_DIM = 256


def rope_inv_freq(theta: float, rotary_dim: int, device="cuda") -> torch.Tensor:
    """fp32 RoPE inverse frequencies, computed on the CPU and then moved, like the reference
    (engine.py:409-410)."""
    expo = torch.arange(0, rotary_dim, 2, dtype=torch.float32) / rotary_dim
    return (1.0 / (theta ** expo)).to(device)


class GatedAttention:
    """One gated full-attention layer's KV cache plus the decode-path calls for n <= n_max rows."""

    def __init__(self, hq: int, hkv: int, max_len: int, q_norm: torch.Tensor, k_norm: torch.Tensor,
                 rope_theta: float = 1e7, rotary_dim: int = 64, eps: float = 1e-6, n_max: int = 8,
                 splits: int | None = None, fused: bool = False, device="cuda"):
        d = HEAD_DIM
        self.hq, self.hkv, self.max_len, self.eps, self.fused = hq, hkv, max_len, eps, fused
        self.q_norm, self.k_norm = q_norm.to(device), k_norm.to(device)
        self.inv_freq = rope_inv_freq(rope_theta, rotary_dim, device)
        self.kc = torch.zeros(hkv, max_len, d, dtype=torch.bfloat16, device=device)
        self.vc = torch.zeros_like(self.kc)
        self.q = torch.zeros(n_max, hq * d, dtype=torch.bfloat16, device=device)
        self.splits = splits or default_splits(max_len, hkv)
        self.part_o, self.part_ml = alloc_partials(n_max, hq, self.splits, device)
        self.q0 = hq * 2 * d
        self.k1 = self.q0 + hkv * d
        self.width = self.k1 + hkv * d

    def __call__(self, proj: torch.Tensor, pos: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
        """proj: [n, >= width] bf16 projection rows (any row stride); pos: int32 device tensor,
        element 0 = position of row 0; out: [n, Hq*256] bf16 rows. Writes K/V of the n rows at
        pos..pos+n-1 and the gated attention output of each row into out."""
        n = proj.shape[0]
        pr = proj[:, : self.width]
        qg = pr[:, : self.q0]
        q = self.q[:n]
        prep = (qg, pr[:, self.q0: self.k1], pr[:, self.k1:], self.q_norm, self.k_norm,
                self.inv_freq, pos, q, self.kc, self.vc, self.eps)
        if self.fused:
            _C.attn_prep_decode(*prep, self.part_o, self.part_ml, out)
        else:
            _C.attn_prep(*prep)
            _C.attn_decode(q, self.kc, self.vc, pos, qg, self.part_o, self.part_ml, out)
        return out


class PagedCache:
    """The paged KV cache of `layers` layers for up to `sequences` sequences of up to `max_len` positions: pools
    kp / vp [layers, pages, Hkv, page_size, 256] (bf16, or E4M3FN codes with kv8), one table and its page counts
    for all layers. What `extend`, `free`, `fork` and `compact` change is device memory of fixed addresses, so a
    pass that calls them can be captured. Their arguments are int32 device tensors; none allocates or syncs."""

    def __init__(self, hkv: int, max_len: int, sequences: int, pages: int, page_size: int = 64, layers: int = 1,
                 kv8: bool = False, k_scale: float = 1.0, v_scale: float = 1.0, device="cuda"):
        if page_size < 16 or page_size > 32768 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two, 16..32768")
        self.hkv, self.page_size, self.sequences, self.layers = hkv, page_size, sequences, layers
        self.kv8, self.k_scale, self.v_scale = kv8, k_scale, v_scale
        width = -(-max_len // page_size)  # entries of a sequence
        self.max_len = width * page_size
        dtype = torch.float8_e4m3fn if kv8 else torch.bfloat16
        shape = (layers, pages, hkv, page_size, HEAD_DIM)
        self.kp, self.vp = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        self.table = torch.full((sequences, width), -1, dtype=torch.int32, device=device)
        self.ref = torch.zeros(pages, dtype=torch.int32, device=device)
        # of the last extend or fork: pages that it could not give
        self.missing = torch.zeros(1, dtype=torch.int32, device=device)
        self.ws = alloc_pages_ws(pages, device)

    def extend(self, pos: torch.Tensor, count: torch.Tensor) -> None:
        """Maps the pages of positions [pos[b], pos[b] + count[b]) of every sequence b with pos[b] >= 0."""
        _C.kv_pages_extend(self.table, self.ref, pos, count, self.page_size, self.missing)

    def free(self, first: torch.Tensor, last: torch.Tensor) -> None:
        """Releases the pages wholly inside [first[b], last[b]) of every sequence b."""
        _C.kv_pages_free(self.table, self.ref, first, last, self.page_size)

    def fork(self, src: torch.Tensor, dst: torch.Tensor, length: torch.Tensor) -> None:
        """Sequence dst[i] becomes a copy of the first length[i] positions of src[i]: whole pages are shared, the
        last partial one is copied. Both go on at `length` or behind it, where neither writes into a
        shared page; to go back further, fork to the earlier length."""
        _C.kv_pages_fork(self.table, self.ref, src, dst, length, self.kp, self.vp, self.missing, self.ws)

    def compact(self) -> None:
        """Moves the pages in use to the pools' front."""
        _C.kv_pages_compact(self.table, self.ref, self.kp, self.vp, self.ws)


class PagedGatedAttention:
    """One gated full-attention layer over a PagedCache: the decode-path calls for up to n_max rows per sequence,
    optionally with a sliding window and first tokens that stay visible. `share`: another layer of the same
    sizes whose scratch (q, part_o, part_ml) this one uses too, for layers that run one after another."""

    def __init__(self, cache: PagedCache, layer: int, hq: int, q_norm: torch.Tensor, k_norm: torch.Tensor,
                 rope_theta: float = 1e7, rotary_dim: int = 64, eps: float = 1e-6, n_max: int = 1,
                 window: int = 0, sinks: int = 0, splits: int | None = None,
                 share: "PagedGatedAttention | None" = None):
        d, dev = HEAD_DIM, cache.kp.device
        self.cache, self.kp, self.vp = cache, cache.kp[layer], cache.vp[layer]
        self.hq, self.hkv, self.eps, self.window, self.sinks = hq, cache.hkv, eps, window, sinks
        self.q_norm, self.k_norm = q_norm.to(dev), k_norm.to(dev)
        self.inv_freq = rope_inv_freq(rope_theta, rotary_dim, dev)
        if share is not None:
            self.q, self.part_o, self.part_ml = share.q, share.part_o, share.part_ml
        else:
            rows = cache.sequences * n_max
            self.q = torch.zeros(rows, hq * d, dtype=torch.bfloat16, device=dev)
            ns = splits or default_paged_splits(cache.max_len, cache.hkv)
            self.part_o, self.part_ml = alloc_partials(rows, hq, ns, dev)
        self.q0 = hq * 2 * d
        self.k1 = self.q0 + cache.hkv * d
        self.width = self.k1 + cache.hkv * d

    def __call__(self, proj: torch.Tensor, pos: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
        """proj: [sequences * R, >= width] bf16 projection rows (any row stride), R per sequence; pos: int32
        [sequences], the position of each sequence's first row, negative for an idle one; out: [sequences * R,
        Hq*256] bf16 rows. Writes K/V of the rows into their pages (mapped by cache.extend) and the gated
        attention output of each row into out; an idle sequence's rows are left as they are."""
        pr = proj[:, : self.width]
        qg, k, v = pr[:, : self.q0], pr[:, self.q0: self.k1], pr[:, self.k1:]
        q, c = self.q[: proj.shape[0]], self.cache
        prep = (qg, k, v, self.q_norm, self.k_norm, self.inv_freq, pos, q, self.kp, self.vp, c.table, self.eps)
        decode = (q, self.kp, self.vp, c.table, pos, qg, self.part_o, self.part_ml, out)
        if c.kv8:
            _C.attn_prep_paged_fp8(*prep, c.k_scale, c.v_scale)
            _C.attn_decode_paged_fp8(*decode, c.k_scale, c.v_scale, self.window, self.sinks)
        else:
            _C.attn_prep_paged(*prep)
            _C.attn_decode_paged(*decode, self.window, self.sinks)
        return out


class MX4Linear:
    """y = x W^T with the weight [N, K] held as 4-bit codes with scales, for up to `rows` 8-bit rows. Owns the codes
    and the product's workspace, both made at construction, so calls can be captured. Calls of one layer, or of
    layers that `share` a workspace, follow one another."""

    def __init__(self, weight: torch.Tensor, rows: int = 8, share: "MX4Linear | None" = None):
        self.n_out, self.width, self.rows = weight.shape[0], weight.shape[1], rows
        dev = weight.device
        self.wq = alloc_mx4(self.n_out, self.width, dev)
        _C.mx4_quant(weight, self.wq)
        need = max(_C.mx4_ws_bytes(n, self.n_out, self.width) for n in range(1, rows + 1))
        if share is not None and share.ws.numel() >= need:
            self.ws = share.ws
        else:
            self.ws = torch.empty(need, dtype=torch.uint8, device=dev)

    def __call__(self, q: torch.Tensor, s: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
        """q, s: 8-bit rows as `rmsnorm1p_mx8`, `swiglu_mx8` or `quant_mx8` write them; out: [n, N] bf16 rows."""
        _C.gemm_mx4(self.wq, q, s, out, self.ws)
        return out


class MX4MLP:
    """One layer's MLP on 4-bit weights for up to `rows` rows: h = bf16(h + delta), then
    down(silu(gate(x)) * up(x)) of its norm x. gate_up: [2 I, H] (gate rows first), down: [H, I], both bf16. Calls of
    one layer follow one another. `share`: another layer of the same sizes whose scratch (the 8-bit rows, gate and up,
    the workspaces) this one uses too, for layers that run one after another (2048 rows of 5120 / 17408: 190 MB)."""

    def __init__(self, norm: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor, eps: float = 1e-6,
                 rows: int = 8, share: "MX4MLP | None" = None):
        dev, H, I = norm.device, down.shape[0], down.shape[1]
        self.norm, self.eps = norm, eps
        self.gate_up = MX4Linear(gate_up, rows, share=share.gate_up if share is not None else None)
        self.down = MX4Linear(down, rows, share=share.down if share is not None else self.gate_up)
        if share is not None:
            self.x, self.act, self.gu = share.x, share.act, share.gu
        else:
            self.x, self.act = alloc_mx8(rows, H, dev), alloc_mx8(rows, I, dev)
            self.gu = torch.empty(rows, 2 * I, dtype=torch.bfloat16, device=dev)

    def __call__(self, h: torch.Tensor, delta: torch.Tensor | None, out: torch.Tensor) -> torch.Tensor:
        """h: [n, H] bf16 residual rows, updated in place where there is a delta [n, H]; out: [n, H] bf16 rows
        (delta itself is fine: it is read before)."""
        n = h.shape[0]
        xq, xs, aq, as_, gu = *(t[:n] for t in self.x), *(t[:n] for t in self.act), self.gu[:n]
        _C.rmsnorm1p_mx8(h, delta, self.norm, xq, xs, self.eps)
        self.gate_up(xq, xs, gu)
        _C.swiglu_mx8(gu, aq, as_)
        return self.down(aq, as_, out)
