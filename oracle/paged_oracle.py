"""CPU model of the paged KV cache, its attention and the operations on pages, in 64 bits.
TEST INFRASTRUCTURE ONLY: only ``tests/`` may import this module, as the checker. The reference has one
contiguous cache (python/qengine/engine.py:419) and no counterpart: parity unpinned; pinned by brute force,
by the contiguous oracle on a gathered cache and by invariants in ``tests/test_paged_oracle.py``.

A pool [N, Hkv, P, 256] holds pages, a table [B, M] names the page of positions [jP, (j+1)P) of sequence b
(an id outside [0, N): none), ref[i] counts the entries that name page i. Row b*R + t is the token of
sequence b at position pos[b] + t; pos[b] < 0: the sequence is idle.
"""
from __future__ import annotations

import numpy as np

D = 256


def attended(p: int, M: int, P: int, N: int, row, window: int = 0, sinks: int = 0) -> list[int]:
    """Positions that a row at position p attends."""
    out = []
    for j in range(min(p + 1, M * P)):
        if not 0 <= int(row[j // P]) < N:
            continue
        if window == 0 or j < sinks or j >= p + 1 - window:
            out.append(j)
    return out


def decode(q, kp, vp, table, pos, qg, R, window=0, sinks=0, k_scale=1.0, v_scale=1.0):
    """(out, bound) of every row, float64 [B*R, Hq, 256]; rows of idle sequences are NaN. bound is what a
    correct fp32 evaluation rounded once to bf16 may be off by:

      scores       s = q.k / 16: 256 products and sums, the scale, log2(e) and the subtraction of the
                   maximum, each within 2^-24 of sum |q k| / 16 =: A  ->  2 * 262 * 2^-24 * A on a weight
                   relative to the row's sum of weights
      weights      the hardware exponential (2^-22) and two bf16 terms (2^-16) for the product with V
      sums         n terms, at most 2 (n + 64) 2^-24
      gate, quotient and the products: 2^-20
      all relative to sum w |v| / sum w (times the gate); then one bf16 rounding: 2^-8 of the value.
    """
    q, qg = np.asarray(q, np.float64), np.asarray(qg, np.float64)
    kp, vp = np.asarray(kp, np.float64), np.asarray(vp, np.float64)
    B, M = table.shape
    N, hkv, P, _ = kp.shape
    hq = q.shape[1] // D
    G = hq // hkv
    out = np.full((B * R, hq, D), np.nan)
    tol = np.zeros((B * R, hq, D))
    for b in range(B):
        if pos[b] < 0:
            continue
        for t in range(R):
            i, p = b * R + t, int(pos[b]) + t
            js = np.array(attended(p, M, P, N, table[b], window, sinks), dtype=np.int64)
            if js.size == 0:
                out[i] = 0
                continue
            pages = np.asarray(table[b])[js // P].astype(np.int64)
            for g in range(hkv):
                K = kp[pages, g, js % P] * k_scale
                V = vp[pages, g, js % P] * v_scale
                for h in range(g * G, g * G + G):
                    x = q[i, h * D:(h + 1) * D]
                    with np.errstate(all="ignore"):
                        s = K @ x / 16
                        w = np.exp(s - s.max())
                        w = w / w.sum()
                        gate = 1 / (1 + np.exp(-qg[i, h * 2 * D + D:(h + 1) * 2 * D]))
                        out[i, h] = (w @ V) * gate
                        A = (np.abs(K) @ np.abs(x)).max() / 16
                        eps = 2 * 262 * 2.0 ** -24 * A + 2.0 ** -22 + 2.0 ** -16 + \
                            2 * (js.size + 64) * 2.0 ** -24 + 2.0 ** -20
                        tol[i, h] = eps * (w @ np.abs(V)) * gate + 2.0 ** -8 * np.abs(out[i, h]) + 1e-37
    return out, tol


def prep(qg, k, v, qnw, knw, inv_freq, pos, R, hq, hkv, eps):
    """(q [rows, Hq, 256], k [rows, Hkv, 256], v, magnitudes of q and k) in float64: RMSNorm1p, then
    rotate-half RoPE at angle pos * inv_freq. The magnitude of a rotated value is that of its pair."""
    qg, k, v = (np.asarray(x, np.float64) for x in (qg, k, v))
    rows = qg.shape[0]
    f = np.asarray(inv_freq, np.float64)
    half = f.size
    p = np.array([int(pos[i // R]) + i % R for i in range(rows)], np.float64)
    ang = p[:, None] * f

    def one(x, w):
        n = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1 + np.asarray(w, np.float64))
        y, m = n.copy(), np.abs(n)
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
        a, b = n[..., :half], n[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = a * c - b * s, b * c + a * s
        m[..., :half] = m[..., half:2 * half] = np.hypot(a, b)
        return y, m

    q, qm = one(qg.reshape(rows, hq, 2 * D)[..., :D], qnw)
    kk, km = one(k.reshape(rows, hkv, D), knw)
    return q, kk, v.reshape(rows, hkv, D), qm, km


# ---------------------------------------------------------------------------------- pages
def _lowest_free(ref, n):
    return [i for i in range(len(ref)) if ref[i] == 0][:n]


def free(table, ref, first, last, P):
    for b in range(table.shape[0]):
        for j in range(table.shape[1]):
            if j * P >= first[b] and (j + 1) * P <= last[b]:
                if 0 <= table[b, j] < len(ref):
                    ref[table[b, j]] -= 1
                table[b, j] = -1


def extend(table, ref, pos, count, P):
    """Returns the pages that were missing."""
    M, missing = table.shape[1], 0
    for b in range(table.shape[0]):
        if pos[b] < 0 or count[b] <= 0:
            continue
        for j in range(int(pos[b]) // P, (int(pos[b]) + int(count[b]) - 1) // P + 1):
            if j < M and 0 <= table[b, j] < len(ref):
                continue
            new = _lowest_free(ref, 1) if j < M else []
            if not new:
                missing += 1
                continue
            table[b, j] = new[0]
            ref[new[0]] = 1
    return missing


def fork(table, ref, src, dst, length, P):
    """(missing, [(from page, to page)])."""
    B, M = table.shape
    N, bad, moves = len(ref), 0, []
    ok = []
    for i, (a, b) in enumerate(zip(src, dst)):
        if not (0 <= a < B and 0 <= b < B) or b in [s for s in src if 0 <= s < B] or \
                sum(1 for d in dst if d == b) > 1:
            bad += 1
        else:
            ok.append(i)
    for i in ok:
        for j in range(M):
            if 0 <= table[dst[i], j] < N:
                ref[table[dst[i], j]] -= 1
            table[dst[i], j] = -1
    for i in ok:
        for j in range(min(max(int(length[i]), 0) // P, M)):
            page = table[src[i], j]
            if 0 <= page < N:
                table[dst[i], j] = page
                ref[page] += 1
    for i in ok:
        n = max(int(length[i]), 0)
        j = n // P
        if n % P and j < M and 0 <= table[src[i], j] < N:
            new = _lowest_free(ref, 1)
            if not new:
                bad += 1
                continue
            table[dst[i], j] = new[0]
            ref[new[0]] = 1
            moves.append((int(table[src[i], j]), new[0]))
    return bad, moves


def compact(table, ref):
    """[(from page, to page)]."""
    U = sum(1 for r in ref if r > 0)
    used = [i for i in range(len(ref)) if ref[i] > 0 and i >= U]
    into = [i for i in range(len(ref)) if ref[i] == 0 and i < U]
    to = dict(zip(used, into))
    for b in range(table.shape[0]):
        for j in range(table.shape[1]):
            table[b, j] = to.get(int(table[b, j]), table[b, j])
    for a, b in to.items():
        ref[b], ref[a] = ref[a], 0
    return list(to.items())


def copy_pairs(src, dst, N):
    """The pairs that kv_pages_copy copies."""
    out = []
    for i, (a, b) in enumerate(zip(src, dst)):
        if not (0 <= a < N and 0 <= b < N) or a == b or b in dst[i + 1:] or b in src:
            continue
        out.append((a, b))
    return out
