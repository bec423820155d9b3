"""Performance cases of the paged key-value cache: the decode attention that reads it (dense, and with a
sliding window and first tokens that stay visible), the norm + RoPE that writes it, and the operations on
its pages.

A pool holds pages of P positions, [N, Hkv, P, 256] for K and for V; a table [B, M] names the page of
every P positions of a sequence (-1: none), ``ref`` counts a page's table entries. Row b * R + t of a
call is the token of sequence b at position pos[b] + t.

Heads and head dim are those of the repository's benchmark and tests: 24 query heads over 4 KV heads
of 256 dims, also 16 / 2 and 32 / 8. Each call is one layer's.
"""
from __future__ import annotations

import math

import torch

own = False

BF, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
FP8 = torch.float8_e4m3fn
DEV = "cuda"
D = 256
EPS = 1e-6
THETA, ROTARY = 1e7, 64
KV_SCALE = 1.0 / 16  # fp8 cache: one scale for unit-scale K and V
SPLITS = 64          # slots of the caller's partials


def listed():
    return [
        # one token of one short conversation: latency and launches count
        dict(name="decode_1x1k", kind="decode", batch=1, rows=1, hq=24, hkv=4, page=64, least=1000,
             most=1000, kv="bf16", window=0, sinks=0),
        # a few conversations of very different lengths
        dict(name="decode_7_ragged", kind="decode", batch=7, rows=1, hq=24, hkv=4, page=64, least=300,
             most=24011, kv="bf16", window=0, sinks=0),
        # a full batch of ordinary conversations: the large, bandwidth-bound call
        dict(name="decode_64_ragged", kind="decode", batch=64, rows=1, hq=24, hkv=4, page=64, least=500,
             most=8000, kv="bf16", window=0, sinks=0),
        # one very long document on the half-size cache
        dict(name="decode_1x128k_fp8", kind="decode", batch=1, rows=1, hq=24, hkv=4, page=128,
             least=131000, most=131000, kv="fp8", window=0, sinks=0),
        # speculative verify of three drafts for a batch, small pages, the other head grouping
        dict(name="verify_16x4_fp8", kind="decode", batch=16, rows=4, hq=16, hkv=2, page=16, least=200,
             most=6000, kv="fp8", window=0, sinks=0),
        # endless conversations in a bounded cache: far positions, a window, four first tokens
        dict(name="window_32x4096", kind="decode", batch=32, rows=1, hq=24, hkv=4, page=64, least=3000,
             most=120000, kv="bf16", window=4096, sinks=4),
        # a short window of a few sequences, two rows each
        dict(name="window_3x500_rows2", kind="decode", batch=3, rows=2, hq=32, hkv=8, page=32, least=100,
             most=30000, kv="bf16", window=500, sinks=16),
        # the new rows of one sequence, and of a verify pass of a batch, into their pages
        dict(name="prep_1", kind="prep", batch=1, rows=1, hq=24, hkv=4, page=64, least=1000, most=1000,
             kv="bf16"),
        dict(name="prep_64x4_fp8", kind="prep", batch=64, rows=4, hq=24, hkv=4, page=64, least=10,
             most=131000, kv="fp8"),
        # eight sequences forked (parallel samples of their prompts), 8 layers' pools
        dict(name="fork_8", kind="fork", batch=32, pairs=8, hkv=4, page=64, least=100, most=4000, layers=8,
             kv="bf16"),
        # a pool after many requests came and went, packed: 500 pages of two layers move
        dict(name="compact_500", kind="compact", batch=48, hkv=4, page=64, used=1200, moves=500, free=800,
             layers=2, kv="bf16"),
        # between two steps of a large batch: finished sequences and pages behind the window are freed,
        # the others get pages for their next tokens
        dict(name="turnover_200", kind="turnover", batch=200, hkv=4, page=16, least=1, most=9000,
             window=2048, sinks=4, rows=4),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["decode"] * 6 + ["window"] * 3 + ["prep", "fork", "compact", "turnover"])
    hq, hkv = rng.choice([(24, 4), (24, 4), (24, 4), (16, 2), (32, 8)])
    page = rng.choice([16, 32, 64, 64, 128])
    kv = rng.choice(["bf16", "bf16", "fp8"])
    if kind in ("decode", "window"):
        batch = _log(rng, 1, 64)
        # no more than the largest listed call: 64 sequences of up to 8,000 positions on 4 heads
        most = max(2, min(131000, 64 * 8000 * 4 // (batch * hkv)))
        top = _log(rng, 1, most)
        least = _log(rng, 1, top)
        window = _log(rng, 64, 8192) if kind == "window" else 0
        sinks = rng.choice([0, 1, 4, 16, 100]) if window else 0
        return dict(kind="decode", batch=batch, rows=rng.choice([1, 1, 1, rng.randint(2, 8)]), hq=hq,
                    hkv=hkv, page=page, least=least, most=top, kv=kv, window=window, sinks=sinks)
    if kind == "prep":
        batch = _log(rng, 1, 100)
        return dict(kind="prep", batch=batch, rows=rng.randint(1, 8), hq=hq, hkv=hkv, page=page, least=1,
                    most=_log(rng, 2, 131000), kv=kv)
    if kind == "fork":
        batch = rng.randint(4, 64)
        return dict(kind="fork", batch=batch, pairs=rng.randint(1, batch // 2), hkv=hkv, page=page,
                    least=1, most=_log(rng, 10, 4000), layers=rng.randint(1, 8), kv=kv)
    if kind == "compact":
        used = rng.randint(20, 1200)
        moves = rng.randint(0, used // 2)
        return dict(kind="compact", batch=rng.randint(1, 64), hkv=hkv, page=page, used=used, moves=moves,
                    free=moves + rng.randint(1, 300), layers=rng.randint(1, 2), kv=kv)
    return dict(kind="turnover", batch=_log(rng, 1, 256), hkv=4, page=page, least=1,
                most=_log(rng, 2, 9000), window=_log(rng, 64, 4096), sinks=rng.choice([0, 4, 20]),
                rows=rng.randint(1, 8))


# ---------------------------------------------------------------------------------- inputs
def _lengths(case):
    """The sequences' lengths before the call (so the positions of their first new rows): spread over
    the logarithm of [least, most], in no order. They are part of the case, not of the seed."""
    n, lo, hi = case["batch"], case["least"], case["most"]
    if n == 1:
        return [hi]
    x = [round(lo * (hi / lo) ** (i / (n - 1))) for i in range(n)]
    return [x[i * 37 % n] if n % 37 else x[i] for i in range(n)]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, scale=1.0, dtype=BF):
    x = torch.empty(shape, dtype=dtype, device=DEV).normal_(generator=g)
    return x if scale == 1.0 else x.mul_(scale)


def _pool(g, kv, *shape):
    x = _randn(g, *shape)
    return (x.float() / KV_SCALE).clamp(-448, 448).to(FP8) if kv == "fp8" else x


def _ints(x):
    return torch.tensor(x, dtype=I32, device=DEV)


def _span(case, length):
    """Page indices that hold what a sequence of `length` positions and `rows` new ones reads or writes."""
    P, last = case["page"], (length + case["rows"] - 1) // case["page"]
    lo = max(0, length + 1 - case["window"]) // P if case.get("window") else 0
    first = -(-min(case.get("sinks", 0), length + case["rows"]) // P) if lo else 0
    if case["kind"] == "prep":
        return [j for j in range(length // P, last + 1)]
    return [j for j in range(last + 1) if j < first or j >= lo]


def _mapped(case, g, spans, spare):
    """A table that maps the given page indices to pages in random order, and the pool's size."""
    need = sum(len(s) for s in spans)
    N = need + spare
    ids = torch.randperm(N, generator=g, device=DEV)[:need].tolist()
    M = max(max(s, default=0) for s in spans) + 1
    table = [[-1] * M for _ in spans]
    for row, s in zip(table, spans):
        for j in s:
            row[j] = ids.pop()
    return _ints(table), N


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    return {"decode": _prepare_decode, "prep": _prepare_prep, "fork": _prepare_fork,
            "compact": _prepare_compact, "turnover": _prepare_turnover}[kind](case, g)


def _prepare_decode(case, g):
    B, R, hq, hkv = case["batch"], case["rows"], case["hq"], case["hkv"]
    lens = _lengths(case)
    table, N = _mapped(case, g, [_span(case, n) for n in lens], 3)
    return dict(case=case, table=table, pos=_ints(lens), q=_randn(g, B * R, hq * D, scale=1.5),
                qg=_randn(g, B * R, hq * 2 * D), kp=_pool(g, case["kv"], N, hkv, case["page"], D),
                vp=_pool(g, case["kv"], N, hkv, case["page"], D),
                part_o=torch.empty(B * R, hq, SPLITS, D, dtype=F32, device=DEV),
                part_ml=torch.empty(B * R, hq, SPLITS, 2, dtype=F32, device=DEV),
                out=torch.zeros(B * R, hq * D, dtype=BF, device=DEV))


def _prepare_prep(case, g):
    B, R, hq, hkv = case["batch"], case["rows"], case["hq"], case["hkv"]
    lens = _lengths(case)
    table, N = _mapped(case, g, [_span(case, n) for n in lens], 3)
    expo = torch.arange(0, ROTARY, 2, dtype=F32) / ROTARY
    return dict(case=case, table=table, pos=_ints(lens),
                proj=_randn(g, B * R, (hq * 2 + 2 * hkv) * D, scale=3.0),
                qnw=_randn(g, D, scale=0.3), knw=_randn(g, D, scale=0.3),
                inv_freq=(1.0 / (THETA ** expo)).to(DEV),
                kp=_pool(g, case["kv"], N, hkv, case["page"], D),
                vp=_pool(g, case["kv"], N, hkv, case["page"], D),
                q=torch.zeros(B * R, hq * D, dtype=BF, device=DEV))


def _prepare_fork(case, g):
    """The first `pairs` sequences fork into as many empty ones, all but a few of their positions kept."""
    m, P = case["pairs"], case["page"]
    spans = [[] if m <= b < 2 * m else list(range(-(-n // P))) for b, n in enumerate(_lengths(case))]
    table, N = _mapped(case, g, spans, m + 5)
    src = list(range(m))
    length = [max(1, n - 3) for n in _lengths(case)[:m]]
    return dict(_pages(case, g, table, N), src=_ints(src), dst=_ints([m + i for i in src]),
                length=_ints(length))


def _prepare_compact(case, g):
    """`used` pages, `moves` of them with ids past `used`; a tenth as many entries share pages."""
    U, mv, N, B = case["used"], case["moves"], case["used"] + case["free"], case["batch"]
    low = torch.randperm(U, generator=g, device=DEV)[:U - mv]
    high = U + torch.randperm(N - U, generator=g, device=DEV)[:mv]
    ids = torch.cat([low, high])
    extra = ids[torch.randint(0, U, (U // 10,), generator=g, device=DEV)]
    ids = torch.cat([ids, extra])
    M = -(-ids.numel() // B)
    flat = torch.full((B * M,), -1, dtype=I32, device=DEV)
    at = torch.randperm(B * M, generator=g, device=DEV)[:ids.numel()]
    flat[at] = ids.to(I32)
    return _pages(case, g, flat.view(B, M), N)


def _prepare_turnover(case, g):
    lens = _lengths(case)
    P, R = case["page"], case["rows"]
    spans = [list(range(-(-n // P))) for n in lens]
    table, N = _mapped(case, g, spans, 2 * case["batch"])
    table = torch.nn.functional.pad(table, (0, 2), value=-1).contiguous()
    done = [i % 8 == 3 for i in range(case["batch"])]
    first = [0 if d else case["sinks"] for d in done]
    last = [2 ** 31 - 1 if d else max(0, n + 1 - case["window"]) for d, n in zip(done, lens)]
    st = _pages(dict(case, layers=0), g, table, N)
    return dict(st, first=_ints(first), last=_ints(last),
                pos=_ints([-1 if d else n for d, n in zip(done, lens)]),
                count=_ints([R] * case["batch"]))


def _pages(case, g, table, N):
    """Allocation state (kept a second time, since a pass starts from it again) and the layers' pools."""
    ref = torch.zeros(N, dtype=I32, device=DEV)
    named = table[table >= 0].long()
    ref.scatter_add_(0, named, torch.ones_like(named, dtype=I32))
    st = dict(case=case, table0=table, ref0=ref, table=table.clone(), ref=ref.clone(),
              missing=torch.zeros(1, dtype=I32, device=DEV),
              ws=torch.zeros(2 * N + 8, dtype=I32, device=DEV))
    if case["layers"]:
        shape = (case["layers"], N, case["hkv"], case["page"], D)
        st.update(kp=_pool(g, case["kv"], *shape), vp=_pool(g, case["kv"], *shape))
    return st


# ---------------------------------------------------------------------------------- a pass
def run(s):
    kind = s["case"]["kind"]
    return {"decode": _decode, "prep": _prep, "fork": _fork, "compact": _compact,
            "turnover": _turnover}[kind](s)


def _decode(s):
    c = s["case"]
    if own:
        from qengine_amd import _C
        if c["kv"] == "fp8":
            _C.attn_decode_paged_fp8(s["q"], s["kp"], s["vp"], s["table"], s["pos"], s["qg"],
                                     s["part_o"], s["part_ml"], s["out"], KV_SCALE, KV_SCALE,
                                     c["window"], c["sinks"])
        else:
            _C.attn_decode_paged(s["q"], s["kp"], s["vp"], s["table"], s["pos"], s["qg"], s["part_o"],
                                 s["part_ml"], s["out"], c["window"], c["sinks"])
        return {"out": s["out"]}
    B, R, hq, hkv = c["batch"], c["rows"], c["hq"], c["hkv"]
    at, seen = _places(s["table"], s["pos"], c)
    k, v = _rows_of(s["kp"], s["table"], at, c), _rows_of(s["vp"], s["table"], at, c)  # [B, hkv, L, D]
    G, L = hq // hkv, k.shape[2]
    q = s["q"].view(B, R, hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, hkv, R * G, D).float()
    x = (q @ k.transpose(2, 3)).view(B, hkv, R, G, L) / 16
    x = x.masked_fill(~seen.view(B, 1, R, 1, L), -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    o = (e.view(B, hkv, R * G, L) @ v).view(B, hkv, R, G, D) / e.sum(-1, keepdim=True)
    gate = s["qg"].view(B, R, hkv, G, 2 * D)[..., D:].permute(0, 2, 1, 3, 4).float()
    o = o / (1 + torch.exp(-gate))
    return {"out": o.permute(0, 2, 1, 3, 4).reshape(B * R, hq * D).to(BF)}


def _places(table, pos, c):
    """Positions that a sequence's rows may attend, [B, L] (None: all of the table's), and which row attends
    which, [B, R, L]."""
    B, R, W, S = c["batch"], c["rows"], c["window"], c["sinks"]
    p = pos.long().view(B, 1, 1) + torch.arange(R, device=DEV).view(1, R, 1)
    if not W:
        at = torch.arange(table.shape[1] * c["page"], device=DEV).view(1, 1, -1)
        return None, (at <= p) & (table >= 0).repeat_interleave(c["page"], 1).view(B, 1, -1)
    first = torch.arange(S, device=DEV).expand(B, S)
    near = pos.long().view(B, 1) + 1 - W + torch.arange(W + R - 1, device=DEV)
    at = torch.cat([first, near], 1)
    ok = torch.cat([first >= 0, near >= S], 1).view(B, 1, -1)
    a = at.view(B, 1, -1)
    return at.clamp(0, table.shape[1] * c["page"] - 1), ok & (a <= p) & ((a < S) | (a > p - W))


def _rows_of(pool, table, at, c):
    """A sequence's cache rows at the positions `at`, in 32 bits: [B, hkv, L, D]."""
    raw = _stored(pool, c)
    if at is None:
        x = raw[table.clamp(min=0).long()].permute(0, 2, 1, 3, 4)
        x = x.reshape(x.shape[0], x.shape[1], -1, x.shape[4])
    else:
        page = table.gather(1, at // c["page"]).clamp(min=0).long()
        x = raw[page, :, at % c["page"]].permute(0, 2, 1, 3).contiguous()
    return x.view(FP8).float() * KV_SCALE if c["kv"] == "fp8" else x.float()


def _prep(s):
    c = s["case"]
    B, R, hq, hkv = c["batch"], c["rows"], c["hq"], c["hkv"]
    a, b = hq * 2 * D, (hq * 2 + hkv) * D
    qg, k, v = s["proj"][:, :a], s["proj"][:, a:b], s["proj"][:, b:]
    if own:
        from qengine_amd import _C
        if c["kv"] == "fp8":
            _C.attn_prep_paged_fp8(qg, k, v, s["qnw"], s["knw"], s["inv_freq"], s["pos"], s["q"],
                                   s["kp"], s["vp"], s["table"], EPS, KV_SCALE, KV_SCALE)
        else:
            _C.attn_prep_paged(qg, k, v, s["qnw"], s["knw"], s["inv_freq"], s["pos"], s["q"], s["kp"],
                               s["vp"], s["table"], EPS)
        return {"q": s["q"], "kp": s["kp"], "vp": s["vp"]}
    p = (s["pos"].long().view(B, 1) + torch.arange(R, device=DEV)).view(-1)  # [B * R]
    ang = p.to(F64).view(-1, 1, 1) * s["inv_freq"].to(F64)
    cos, sin = torch.cos(ang).float(), torch.sin(ang).float()

    def normed(x, w):
        x = x.float()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * (1 + w.float())
        h = ROTARY // 2
        lo, hi = x[..., :h], x[..., h:ROTARY]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, x[..., ROTARY:]], -1)

    q = normed(qg.reshape(B * R, hq, 2 * D)[..., :D], s["qnw"])
    kn = normed(k.reshape(B * R, hkv, D), s["knw"])
    page = s["table"].long()[torch.arange(B, device=DEV).repeat_interleave(R), p // c["page"]]
    _stored(s["kp"], c)[page, :, p % c["page"]] = _codes(kn, c)
    _stored(s["vp"], c)[page, :, p % c["page"]] = _codes(v.reshape(B * R, hkv, D).float(), c)
    return {"q": q.reshape(B * R, hq * D).to(BF), "kp": s["kp"], "vp": s["vp"]}


def _stored(pool, c):
    return pool.view(torch.uint8) if c["kv"] == "fp8" else pool


def _codes(x, c):
    if c["kv"] == "fp8":
        return (x / KV_SCALE).clamp(-448, 448).to(FP8).view(torch.uint8)
    return x.to(BF)


def _fork(s):
    _again(s)
    if own:
        from qengine_amd import _C
        _C.kv_pages_fork(s["table"], s["ref"], s["src"], s["dst"], s["length"], s["kp"], s["vp"],
                         s["missing"], s["ws"])
    else:
        P, table, ref = s["case"]["page"], s["table"], s["ref"]
        src, dst, n = s["src"].long(), s["dst"].long(), s["length"].long()
        _release(table, ref, dst)
        j = torch.arange(table.shape[1], device=DEV)
        rows = table[src]
        whole = (j < (n // P).view(-1, 1)) & (rows >= 0)
        part = (j == (n // P).view(-1, 1)) & (n % P > 0).view(-1, 1) & (rows >= 0)
        ref.add_(torch.bincount(rows[whole], minlength=ref.numel()).to(I32))
        new, got, short = _lowest_free(ref, part)
        ref[new[got].long()] += 1
        table[dst] = torch.where(got, new, torch.where(whole, rows, -1))
        a, b = rows[got].long(), new[got].long()
        _move(s["kp"], s["case"], a, b)
        _move(s["vp"], s["case"], a, b)
        s["missing"].copy_(short)
    return {"table": s["table"], "ref": s["ref"], "kp": s["kp"], "vp": s["vp"], "missing": s["missing"]}


def _compact(s):
    _again(s)
    if own:
        from qengine_amd import _C
        _C.kv_pages_compact(s["table"], s["ref"], s["kp"], s["vp"], s["ws"])
    else:
        table, ref = s["table"], s["ref"]
        used, ids = ref > 0, torch.arange(ref.numel(), device=DEV)
        U = used.sum()
        a, b = ids[used & (ids >= U)], ids[~used & (ids < U)]
        b = b[:a.numel()]
        to = ids.clone()
        to[a] = b
        table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].to(I32), table))
        ref[b] = ref[a]
        ref[a] = 0
        _move(s["kp"], s["case"], a, b)
        _move(s["vp"], s["case"], a, b)
    return {"table": s["table"], "ref": s["ref"], "kp": s["kp"], "vp": s["vp"]}


def _turnover(s):
    _again(s)
    if own:
        from qengine_amd import _C
        _C.kv_pages_free(s["table"], s["ref"], s["first"], s["last"], s["case"]["page"])
        _C.kv_pages_extend(s["table"], s["ref"], s["pos"], s["count"], s["case"]["page"], s["missing"])
    else:
        P, table, ref = s["case"]["page"], s["table"], s["ref"]
        j = torch.arange(table.shape[1], device=DEV)
        gone = (j * P >= s["first"].view(-1, 1)) & ((j + 1) * P <= s["last"].view(-1, 1)) & (table >= 0)
        ref.sub_(torch.bincount(table[gone], minlength=ref.numel()).to(I32))
        table.masked_fill_(gone, -1)
        p, n = s["pos"].long().view(-1, 1), s["count"].long().view(-1, 1)
        need = (p >= 0) & (n > 0) & (j >= p // P) & (j <= (p + n - 1) // P) & (table < 0)
        new, got, short = _lowest_free(ref, need)
        ref[new[got].long()] += 1
        table.copy_(torch.where(got, new, table))
        s["missing"].copy_(short)
    return {"table": s["table"], "ref": s["ref"], "missing": s["missing"]}


def _again(s):
    """A pass starts from the same allocation, so that it can be called again on the same state."""
    s["table"].copy_(s["table0"])
    s["ref"].copy_(s["ref0"])


def _release(table, ref, rows):
    old = table[rows]
    ref.sub_(torch.bincount(old[old >= 0], minlength=ref.numel()).to(I32))
    table[rows] = -1


def _lowest_free(ref, need):
    """For the true places of `need`, in row-major order, the lowest free ids: (ids, places that got one,
    how many got none)."""
    rank = need.view(-1).long().cumsum(0) - 1
    order = torch.sort((ref > 0).to(I32), stable=True).indices
    got = need & (rank < (ref == 0).sum()).view(need.shape)
    new = order[rank.clamp(0, ref.numel() - 1)].view(need.shape).to(I32)
    return torch.where(got, new, 0), got, (need.sum() - got.sum()).view(1).to(I32)


def _move(pool, c, a, b):
    p = _stored(pool, c)
    p[:, b] = p[:, a]


# ---------------------------------------------------------------------------------- floors
def work(case):
    """Bytes and operations that a pass cannot do without: each position attended by a sequence's rows read
    once, each row's inputs and outputs once; each moved page read and written once."""
    kind, elem = case["kind"], 1 if case.get("kv") == "fp8" else 2
    if kind == "turnover":
        P, R = case["page"], case["rows"]
        lens = _lengths(case)
        M = -(-max(lens) // P) + 2
        N = sum(-(-n // P) for n in lens) + 2 * case["batch"]
        return {"bytes": 2 * 4 * case["batch"] * M + 2 * 4 * N + 16 * case["batch"], "flops": 0}
    hkv, P = case["hkv"], case["page"]
    if kind in ("fork", "compact"):
        if kind == "fork":
            lens = [max(1, n - 3) for n in _lengths(case)[:case["pairs"]]]
            pages, entries = sum(n % P > 0 for n in lens), sum(-(-n // P) for n in lens)
        else:
            pages, entries = case["moves"], case["used"]
        return {"bytes": case["layers"] * 2 * pages * 2 * hkv * P * D * elem + 16 * entries, "flops": 0}
    B, R, hq = case["batch"], case["rows"], case["hq"]
    if kind == "prep":
        return {"bytes": B * R * ((hq + 2 * hkv) * D * 2 + hq * D * 2 + 2 * hkv * D * elem),
                "flops": B * R * (hq + hkv) * D * 8}
    kept = reads = 0
    for n in _lengths(case):
        seen = [_seen(case, n + t) for t in range(R)]
        kept += sum(a + b - c for a, b, c in seen)
        # what any of the rows attends: the first tokens, and the first row's window to the last row
        a, b, c = seen[0]
        reads += min(n + R, max(a, min(case["sinks"], n + R)) + b - c + R - 1)
    return {"bytes": reads * 2 * hkv * D * elem + B * R * hq * D * 6, "flops": kept * hq * 4 * D}


def _seen(case, p):
    """Of the row at position p: first tokens, positions of the window, both."""
    if not case["window"]:
        return 0, p + 1, 0
    lo = max(0, p + 1 - case["window"])
    a = min(case["sinks"], p + 1)
    return a, p + 1 - lo, max(0, a - lo)


# ---------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The definition, row by row over the attended positions, in 64 bits."""
    if case["kind"] not in ("decode", "prep"):
        return None  # whole numbers and moved bytes
    s = prepare(case, seed)
    c, P, R = case, case["page"], case["rows"]
    G = c["hq"] // c["hkv"]
    scale = KV_SCALE if c["kv"] == "fp8" else 1.0
    pos = s["pos"].tolist()
    if c["kind"] == "decode":
        out = torch.zeros(len(pos) * R, c["hq"], D, dtype=F64, device=DEV)
        for b, p0 in enumerate(pos):
            for t in range(R):
                p = p0 + t
                keep = torch.arange(p + 1, device=DEV)
                if c["window"]:
                    keep = keep[(keep < c["sinks"]) | (keep >= p + 1 - c["window"])]
                page, off = s["table"][b, keep // P].long(), keep % P
                for g in range(c["hkv"]):
                    k = s["kp"].view(torch.uint8 if c["kv"] == "fp8" else BF)[page, g, off]
                    v = s["vp"].view(torch.uint8 if c["kv"] == "fp8" else BF)[page, g, off]
                    if c["kv"] == "fp8":
                        k, v = k.view(FP8), v.view(FP8)
                    h = slice(g * G, g * G + G)
                    q = s["q"][b * R + t].view(c["hq"], D)[h].to(F64)
                    w = torch.softmax(q @ k.to(F64).T.contiguous() * (scale / 16), -1)
                    gate = s["qg"][b * R + t].view(c["hq"], 2 * D)[h, D:].to(F64)
                    out[b * R + t, h] = (w @ v.to(F64)) * scale * torch.sigmoid(gate)
        return {"out": out.view(len(pos) * R, -1)}
    kp, vp = s["kp"].to(F64), s["vp"].to(F64)
    q = torch.zeros(len(pos) * R, c["hq"], D, dtype=F64, device=DEV)
    h = ROTARY // 2
    x = s["proj"].to(F64).view(len(pos) * R, -1, D)
    for b, p0 in enumerate(pos):
        for t in range(R):
            p, i = p0 + t, b * R + t
            a = p * s["inv_freq"].to(F64)
            turn = torch.polar(torch.ones_like(a), a)
            y = x[i].clone()
            for rows, w in ((slice(0, 2 * c["hq"], 2), s["qnw"]),
                            (slice(2 * c["hq"], 2 * c["hq"] + c["hkv"]), s["knw"])):
                z = y[rows] * torch.rsqrt(y[rows].square().mean(-1, keepdim=True) + EPS) * (1 + w.to(F64))
                pair = torch.complex(z[:, :h], z[:, h:ROTARY]) * turn
                z[:, :h], z[:, h:ROTARY] = pair.real, pair.imag
                y[rows] = z
            q[i] = y[0:2 * c["hq"]:2]
            page, off = int(s["table"][b, p // P]), p % P
            kp[page, :, off] = y[2 * c["hq"]: 2 * c["hq"] + c["hkv"]] / scale
            vp[page, :, off] = y[2 * c["hq"] + c["hkv"]:] / scale
    return {"q": q.view(len(pos) * R, -1), "kp": kp, "vp": vp}
