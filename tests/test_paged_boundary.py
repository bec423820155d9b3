"""CPU tests of the paged cache's contract: what the torch ops and the C ABI accept, and each refusal (raised
before any launch). No kernel runs here."""
import pytest
import torch

BF, F32, I32, U8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8
FP8 = torch.float8_e4m3fn
D = 256
INVALID = 1  # hipErrorInvalidValue
A = 1 << 20  # an aligned address; the C ABI validates before touching it


def z(*s, dt=BF):
    return torch.zeros(*s, dtype=dt)


def decode_args(B=3, R=2, hq=6, hkv=2, N=5, P=16, M=4, ns=4, kv=BF):
    n = B * R
    return dict(q=z(n, hq * D), kp=z(N, hkv, P, D, dt=kv), vp=z(N, hkv, P, D, dt=kv), table=z(B, M, dt=I32),
                pos=z(B, dt=I32), qg=z(n, hq * 2 * D), po=z(n, hq, ns, D, dt=F32),
                pml=z(n, hq, ns, 2, dt=F32), out=z(n, hq * D), window=0, sinks=0, kv8=kv != BF)


def check_decode(native, **kw):
    a = decode_args()
    a.update(kw)
    return native._check_attn_decode_paged(*a.values())


def test_decode_contract_accepts(native):
    assert check_decode(native) == [3, 2, 6, 2, 5, 16, 4, 4, 4, 6 * 512, 6 * D]
    for kv in (FP8, U8):
        native._check_attn_decode_paged(*decode_args(kv=kv).values())
    for kw in (dict(B=1, R=8), dict(B=1024, R=1, M=1, N=1, hq=1, hkv=1), dict(hq=1, hkv=1), dict(P=128)):
        native._check_attn_decode_paged(*decode_args(**kw).values())
    # row strides: tables, gates and outputs that are views; one row's stride is of no account
    got = check_decode(native, table=z(3, 9, dt=I32)[:, :4], qg=z(6, 6 * 512 + 8)[:, 3:-5],
                       out=z(6, 6 * D + 1)[:, 1:])
    assert got[-3:] == [9, 6 * 512 + 8, 6 * D + 1]
    a = decode_args(B=1, R=1)
    a["out"] = a["out"].as_strided((1, 6 * D), (1, 1))
    native._check_attn_decode_paged(*a.values())
    check_decode(native, window=2 ** 23 - 1, sinks=2 ** 40)


@pytest.mark.parametrize("kw,why", [
    (dict(q=z(7, 6 * D)), "1..8 rows"), (dict(q=z(0, 6 * D)), "1..8 rows"), (dict(q=z(27, 6 * D)), "1..8 rows"),
    (dict(q=z(6, 6 * D + 8)), "q rows must be contiguous"), (dict(q=z(6, 5 * D)), "Hq % Hkv"),
    (dict(q=z(6, 6 * D, dt=F32)), "dtype"), (dict(q=z(6, 6 * D + 1)[:, 1:]), "contiguous|aligned"),
    (dict(kp=z(5, 2, 16, 128)), "kp/vp"), (dict(kp=z(2, 16, D)), "kp/vp"),
    (dict(kp=z(6, 2, 16, D)), "kp/vp"), (dict(kp=z(1, 5, 2, 16, D), vp=z(1, 5, 2, 16, D)), "kp/vp"),
    (dict(kp=z(5, 2, 24, D), vp=z(5, 2, 24, D)), "power of two"),
    (dict(kp=z(5, 2, 8, D), vp=z(5, 2, 8, D)), "power of two"),
    (dict(kp=z(5, 2, 16, D, dt=U8)), "dtype"), (dict(kp=z(0, 2, 16, D), vp=z(0, 2, 16, D)), "pages"),
    (dict(kp=z(5, 2, 32, D)[:, :, ::2], vp=z(5, 2, 16, D)), "contiguous"),
    (dict(table=z(3, 4, dt=torch.int64)), "int32"), (dict(table=z(12, dt=I32)), "table must be"),
    (dict(table=z(4, 3, dt=I32).t()), "inner stride"), (dict(table=z(1, 4, dt=I32).expand(3, 4)), "overlap"),
    (dict(table=z(3, 0, dt=I32)), "table must be"), (dict(table=z(3, 1 << 19, dt=I32)), "positions"),
    (dict(pos=z(2, dt=I32)), "pos must have"), (dict(pos=z(3, dt=torch.int64)), "dtype"),
    (dict(pos=z(6, dt=I32)[::2]), "contiguous"),
    (dict(qg=z(6, 6 * 512 - 8)), "qg width"), (dict(qg=z(5, 6 * 512)), "q's rows"),
    (dict(qg=z(1, 6 * 512).expand(6, 6 * 512)), "overlap"),
    (dict(out=z(6, 5 * D)), "out width"), (dict(out=z(1, 6 * D).expand(6, 6 * D)), "overlap"),
    (dict(po=z(5, 6, 4, D, dt=F32)), "part_o"), (dict(po=z(6, 6, 4, D)), "dtype"),
    (dict(po=z(6, 5, 4, D, dt=F32)), "part_o"), (dict(po=z(6, 6, 0, D, dt=F32)), "part_o"),
    (dict(pml=z(6, 6, 4, dt=F32)), "part_ml"),
    (dict(window=-1), "window"), (dict(window=2 ** 23), "window"), (dict(sinks=-1), "window"),
    (dict(window=5, po=z(6, 6, 3, D, dt=F32), pml=z(6, 6, 3, 2, dt=F32)), "4 splits"),
])
def test_decode_contract_rejects(native, kw, why):
    with pytest.raises(RuntimeError, match=why):
        check_decode(native, **kw)


def test_too_many_sequences(native):
    with pytest.raises(RuntimeError, match="1..1024"):
        native._check_attn_decode_paged(*decode_args(B=1025, R=1, hq=1, hkv=1, M=1, ns=1).values())


def prep_args(B=3, R=2, hq=6, hkv=2, N=5, P=16, M=4, kv=BF, rd=64):
    n, w = B * R, (hq * 2 + 2 * hkv) * D
    pr = z(n, w)
    a, b = hq * 2 * D, (hq * 2 + hkv) * D
    return dict(qg=pr[:, :a], k=pr[:, a:b], v=pr[:, b:], qnw=z(D), knw=z(D), f=z(rd // 2, dt=F32),
                pos=z(B, dt=I32), q=z(n, hq * D), kp=z(N, hkv, P, D, dt=kv), vp=z(N, hkv, P, D, dt=kv),
                table=z(B, M, dt=I32), kv8=kv != BF)


def test_prep_contract_accepts(native):
    assert native._check_attn_prep_paged(*prep_args().values()) == [3, 2, 6, 2, 5, 16, 4, 64, 4, 16 * D]
    native._check_attn_prep_paged(*prep_args(B=1, R=500, kv=FP8, rd=256).values())


@pytest.mark.parametrize("kw,why", [
    (dict(k=z(6, 2 * D)), "row stride"), (dict(qg=z(5, 12 * D)), "row stride|rows"),
    (dict(qg=z(6, 16 * D)[:, :11 * D]), "widths"), (dict(q=z(5, 6 * D)), "rows"),
    (dict(q=z(6, 7 * D)[:, :6 * D]), "contiguous q_out"), (dict(q=z(6, 6 * D + 8)), "q_out width"),
    (dict(qnw=z(D, dt=F32)), "dtype"), (dict(knw=z(D - 1)), "256 elements"), (dict(f=z(129, dt=F32)), "rotary"),
    (dict(f=z(0, dt=F32)), "rotary"), (dict(f=z(32)), "dtype"), (dict(pos=z(1, dt=I32)), "pos must have"),
    (dict(kp=z(5, 3, 16, D), vp=z(5, 3, 16, D)), "widths"), (dict(table=z(2, 4, dt=I32)), "pos must have"),
    (dict(kp=z(5, 2, 16, D, dt=FP8)), "dtype"),
])
def test_prep_contract_rejects(native, kw, why):
    a = prep_args()
    a.update(kw)
    with pytest.raises(RuntimeError, match=why):
        native._check_attn_prep_paged(*a.values())


@pytest.mark.parametrize("k,v", [(0.0, 1.0), (1.0, -1.0), (float("inf"), 1.0), (1.0, float("nan")), (1e-40, 1.0)])
def test_fp8_scales(native, capi, k, v):
    with pytest.raises(RuntimeError, match="k_scale"):
        native._check_kv_scales(k, v)
    assert c_decode(capi, fp8=(k, v)) == INVALID
    assert c_prep(capi, fp8=(k, v)) == INVALID


T, R5, I3, ONE = z(3, 4, dt=I32), z(5, dt=I32), z(3, dt=I32), z(1, dt=I32)
KP, WS = z(2, 5, 2, 16, D), z(18, dt=I32)


def test_page_contracts_accept(native):
    native._check_kv_pages_free(T, R5, I3, I3, 16)
    native._check_kv_pages_extend(T, R5, I3, I3, 32768, ONE)
    native._check_kv_pages_fork(T, R5, ONE, ONE, ONE, KP, KP, ONE, WS)
    native._check_kv_pages_fork(T, R5, I3, I3, I3, KP[0], KP[0], ONE, z(50, dt=I32))
    native._check_kv_pages_compact(z(3, 9, dt=I32)[:, 2:5], R5, KP.to(FP8), KP.to(FP8), WS)
    native._check_kv_pages_copy(KP, KP, I3, I3)


@pytest.mark.parametrize("op,args,why", [
    ("free", (T, R5, I3, ONE, 16), "last"), ("free", (T, R5, I3, I3, 17), "power of two"),
    ("free", (T, R5, I3, I3, 8), "power of two"), ("free", (T, z(0, dt=I32), I3, I3, 16), "ref"),
    ("free", (T, z(5), I3, I3, 16), "dtype"), ("free", (T.long(), R5, I3, I3, 16), "int32"),
    ("free", (z(3, 1000, dt=I32), R5, I3, I3, 16384), "positions"),
    ("free", (ONE.view(1, 1).expand(3, 4), R5, I3, I3, 16), "inner stride|overlap"),
    ("extend", (T, R5, I3, I3, 16, I3), "missing"), ("extend", (T, R5, z(2, dt=I32), I3, 16, ONE), "pos"),
    ("extend", (z(1025, 1, dt=I32), R5, z(1025, dt=I32), z(1025, dt=I32), 16, ONE), "1..1024"),
    ("fork", (T, R5, z(0, dt=I32), z(0, dt=I32), z(0, dt=I32), KP, KP, ONE, WS), "pairs"),
    ("fork", (T, R5, z(1025, dt=I32), z(1025, dt=I32), z(1025, dt=I32), KP, KP, ONE, WS), "pairs"),
    ("fork", (T, R5, I3, ONE, I3, KP, KP, ONE, WS), "dst"), ("fork", (T, R5, I3, I3, ONE, KP, KP, ONE, WS), "length"),
    ("fork", (T, z(6, dt=I32), I3, I3, I3, KP, KP, ONE, WS), "per page"),
    ("fork", (T, R5, I3, I3, I3, KP, KP, ONE, z(17, dt=I32)), "ws"),
    ("fork", (T, R5, I3, I3, I3, KP, KP[:1], ONE, WS), "kp/vp"),
    ("compact", (T, R5, KP, KP, z(17, dt=I32)), "ws"), ("compact", (T, R5, KP, KP, z(18)), "dtype"),
    ("compact", (T, R5, KP.float(), KP.float(), WS), "float8"),
    ("compact", (T, R5, KP[:, :, ::2], KP[:, :, ::2], WS), "contiguous"),
    ("copy", (KP, KP, I3, ONE), "dst"), ("copy", (KP, KP, z(0, dt=I32), z(0, dt=I32)), "pairs"),
    ("copy", (KP, KP, z(65536, dt=I32), z(65536, dt=I32)), "pairs"), ("copy", (KP, KP, I3.long(), I3), "dtype"),
])
def test_page_contracts_reject(native, op, args, why):
    with pytest.raises(RuntimeError, match=why):
        getattr(native, f"_check_kv_pages_{op}")(*args)


def test_gpu_tensors_are_required(native):
    a = decode_args()
    kv8 = a.pop("kv8")
    assert not kv8
    with pytest.raises(RuntimeError, match="device|GPU"):
        native.attn_decode_paged(*a.values())
    with pytest.raises(RuntimeError, match="GPU"):
        native.kv_pages_free(T, R5, I3, I3, 16)


# ---------------------------------------------------------------------------------- the C ABI
def c_decode(capi, fp8=None, **kw):
    a = dict(q=A, kp=A, vp=A, table=A, ldt=4, pos=A, qg=A, ldp=6 * 512, po=A, pml=A, out=A, ldo=6 * D, B=3, R=2,
             hq=6, hkv=2, N=5, P=16, M=4, ns=4, window=0, sinks=0, scale=1 / 16)
    a.update(kw)
    if fp8:
        return capi.load().qe_attn_decode_paged_fp8(*a.values(), *fp8, None)
    return capi.load().qe_attn_decode_paged(*a.values(), None)


@pytest.mark.parametrize("kw", [
    dict(B=0), dict(B=1025), dict(R=0), dict(R=9), dict(hq=5), dict(hq=0), dict(hkv=0), dict(N=0), dict(P=8),
    dict(P=48), dict(P=65536), dict(M=0), dict(ldt=3), dict(M=1 << 19, ldt=1 << 19), dict(ns=0),
    dict(ns=3, window=4), dict(window=-1), dict(window=1 << 23), dict(sinks=-1), dict(ldp=6 * 512 - 1),
    dict(ldo=6 * D - 1), dict(q=A + 2), dict(kp=A + 8), dict(vp=A + 8), dict(po=A + 4), dict(pml=A + 4),
    dict(q=None), dict(kp=None), dict(vp=None), dict(table=None), dict(pos=None), dict(qg=None), dict(po=None),
    dict(pml=None), dict(out=None), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(B=1024, ns=1 << 20), dict(M=-1), dict(P=-16), dict(N=-5),
])
def test_capi_decode_rejects(capi, kw):
    assert c_decode(capi, **kw) == INVALID


def c_prep(capi, fp8=None, **kw):
    a = dict(qg=A, k=A, v=A, ldp=16 * D, qnw=A, knw=A, f=A, pos=A, q=A, kp=A, vp=A, table=A, ldt=4, B=3, R=2,
             hq=6, hkv=2, N=5, P=16, M=4, rd=64, eps=1e-6)
    a.update(kw)
    if fp8:
        return capi.load().qe_attn_prep_paged_fp8(*a.values(), *fp8, None)
    return capi.load().qe_attn_prep_paged(*a.values(), None)


@pytest.mark.parametrize("kw", [
    dict(B=0), dict(B=1025), dict(R=0), dict(B=1000, R=66), dict(hq=0), dict(hkv=0), dict(N=0), dict(P=8),
    dict(P=48), dict(M=0), dict(ldt=3), dict(rd=-2), dict(rd=258), dict(rd=3), dict(ldp=0), dict(kp=A + 8),
    dict(vp=A + 2), dict(hq=20000), dict(qg=None), dict(k=None), dict(v=None), dict(qnw=None), dict(knw=None),
    dict(f=None), dict(pos=None), dict(q=None), dict(kp=None), dict(vp=None), dict(table=None),
])
def test_capi_prep_rejects(capi, kw):
    assert c_prep(capi, **kw) == INVALID


def test_capi_pages_reject(capi):
    lib = capi.load()
    free = dict(t=A, ldt=4, ref=A, first=A, last=A, B=3, M=4, N=5, P=16)
    for kw in (dict(t=None), dict(ref=None), dict(first=None), dict(last=None), dict(B=0), dict(B=1025), dict(M=0),
               dict(ldt=3), dict(N=0), dict(N=(1 << 24) + 1), dict(P=0), dict(P=20), dict(M=1 << 20, ldt=1 << 20)):
        assert lib.qe_kv_pages_free(*{**free, **kw}.values(), None) == INVALID, kw
    ext = dict(t=A, ldt=4, ref=A, pos=A, count=A, missing=A, B=3, M=4, N=5, P=16)
    for kw in (dict(pos=None), dict(count=None), dict(missing=None), dict(N=0), dict(P=15)):
        assert lib.qe_kv_pages_extend(*{**ext, **kw}.values(), None) == INVALID, kw
    fork = dict(t=A, ldt=4, ref=A, src=A, dst=A, length=A, m=2, kp=A, vp=A, layers=1, pb=16384, missing=A, ws=A,
                B=3, M=4, N=5, P=16)
    for kw in (dict(src=None), dict(dst=None), dict(length=None), dict(m=0), dict(m=1025), dict(kp=None),
               dict(vp=A + 8), dict(layers=0), dict(pb=0), dict(pb=24), dict(missing=None), dict(ws=None),
               dict(ws=A + 2), dict(layers=65535, pb=1 << 30)):
        assert lib.qe_kv_pages_fork(*{**fork, **kw}.values(), None) == INVALID, kw
    comp = dict(t=A, ldt=4, ref=A, kp=A, vp=A, layers=1, pb=16384, ws=A, B=3, M=4, N=5)
    for kw in (dict(t=None), dict(ws=None), dict(kp=A + 4), dict(N=0), dict(layers=0)):
        assert lib.qe_kv_pages_compact(*{**comp, **kw}.values(), None) == INVALID, kw
    copy = dict(kp=A, vp=A, layers=1, pb=16384, src=A, dst=A, m=2, N=5)
    for kw in (dict(src=None), dict(dst=None), dict(m=0), dict(m=65536), dict(kp=None), dict(N=0)):
        assert lib.qe_kv_pages_copy(*{**copy, **kw}.values(), None) == INVALID, kw
    assert lib.qe_kv_pages_ws_size(5) == 72 and lib.qe_kv_pages_ws_size(0) == 0


def test_cache_helpers(native):
    """Sizes of the host-side helpers, and the cache's refusals (built on the CPU)."""
    import qengine_amd as qe
    from qengine_amd.layer import PagedCache
    assert qe.default_paged_splits(131072, 4, cus=256) == 64
    assert qe.default_paged_splits(1000, 4, cus=256) == 32
    assert qe.default_paged_splits(16, 4, cus=256) == 4
    assert qe.default_paged_splits(131072, 500, cus=256) == 4
    assert qe.alloc_pages_ws(100, device="cpu").numel() == 208
    c = PagedCache(2, 100, 3, 7, page_size=32, layers=2, device="cpu")
    assert c.kp.shape == c.vp.shape == (2, 7, 2, 32, 256) and c.kp.dtype == torch.bfloat16
    assert c.table.shape == (3, 4) and (c.table == -1).all() and c.max_len == 128 and not c.ref.any()
    assert PagedCache(1, 16, 1, 1, 16, kv8=True, device="cpu").kp.dtype == torch.float8_e4m3fn
    for bad in (0, 8, 48, 65536):
        with pytest.raises(ValueError, match="power of two"):
            PagedCache(2, 100, 3, 7, page_size=bad, device="cpu")
