"""CPU tests of the contract of the linear layers on 4-bit weights: what the torch ops and the C ABI accept, and each
refusal (raised before any launch). No kernel runs here."""
import pytest
import torch

BF, F32, U8 = torch.bfloat16, torch.float32, torch.uint8
FP8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
INVALID = 1   # hipErrorInvalidValue
A = 1 << 20   # an aligned address; the C ABI validates before touching it


def z(*s, dt=BF):
    return torch.zeros(*s, dtype=dt)


def test_sizes(native):
    assert native.mx4_bytes(16, 512) == 4 * 1024 + 256
    assert native.mx4_bytes(1, 1) == 1024 + 256
    assert native.mx4_bytes(17, 513) == 2 * 5 * 1024 + 2 * 2 * 256
    assert native.mx4_bytes(34816, 5120) == 34816 * 5120 * 17 // 32
    for N, K in ((0, 1), (1, 0), (-1, 5), (2 ** 24 + 1, 1), (1, 2 ** 20 + 1), (2 ** 33, 1)):
        with pytest.raises(RuntimeError, match="must be 1"):
            native.mx4_bytes(N, K)
        with pytest.raises(RuntimeError, match="must be 1"):
            native.mx4_ws_bytes(1, N, K)
    for n in (0, -1, 2 ** 40):
        with pytest.raises(RuntimeError, match="must be 1"):
            native.mx4_ws_bytes(n, 16, 32)
    assert native.mx4_ws_bytes(2 ** 24, 2 ** 24, 2 ** 20) >= 0


def wq_for(native, N, K):
    return z(native.mx4_bytes(N, K), dt=U8)


def test_weight_contract(native):
    assert native._check_mx4_weight(z(5, 40), wq_for(native, 5, 40)) == [5, 40, 40]
    assert native._check_mx4_weight(z(5, 48)[:, 3:43], wq_for(native, 5, 40)) == [5, 40, 48]
    assert native._check_mx4_weight(z(1, 48)[:, :40], wq_for(native, 1, 40)) == [1, 40, 40]
    wq = wq_for(native, 5, 40)
    for w, q, why in ((z(5, 40, dt=F32), wq, "dtype"), (z(40), wq, r"\[N, K\]"), (z(40, 5).t(), wq, "inner stride"),
                      (z(1, 40).expand(5, 40), wq, "overlap"), (z(17, 40), wq, "wq must hold"),
                      (z(5, 600), wq, "wq must hold"), (z(5, 40), wq[:-1], "wq must hold"),
                      (z(5, 40), z(wq.numel() + 1, dt=U8)[1:], "aligned"),
                      (z(5, 40), z(2 * wq.numel(), dt=U8)[::2], "contiguous"),
                      (z(5, 40), wq.view(torch.int8), "dtype"), (z(0, 40), wq, "rows"), (z(5, 0), wq, "no columns")):
        with pytest.raises(RuntimeError, match=why):
            native._check_mx4_weight(w, q)


@pytest.mark.parametrize("glu", [False, True])
def test_act_contract(native, glu):
    m = 2 if glu else 1
    ok = lambda **k: native._check_act_mx8(  # noqa: E731
        *{**dict(x=z(3, m * 40), q=z(3, 64, dt=FP8), s=z(3, 2, dt=U8), glu=glu), **k}.values())
    assert ok() == [3, 40, m * 40, 64, 2]
    assert ok(q=z(3, 80, dt=U8)[:, :64], s=z(3, 5, dt=U8).view(E8)[:, 1:3]) == [3, 40, m * 40, 80, 5]
    assert ok(x=z(m * 40), q=z(64, dt=FP8), s=z(2, dt=E8)) == [1, 40, m * 40, 64, 2]
    for kw, why in ((dict(x=z(3, m * 40, dt=F32)), "dtype"), (dict(q=z(3, 64)), "float8_e4m3fn"),
                    (dict(s=z(3, 2, dt=FP8)), "float8_e8m0fnu"), (dict(q=z(3, 32, dt=FP8)), "64 wide"),
                    (dict(q=z(3, 40, dt=FP8)), "64 wide"), (dict(s=z(3, 1, dt=U8)), "2 wide"),
                    (dict(q=z(2, 64, dt=FP8)), "3 rows"), (dict(s=z(4, 2, dt=U8)), "3 rows"),
                    (dict(q=z(3, 72, dt=U8)[:, :64]), "aligned"), (dict(q=z(3, 80, dt=U8)[:, 8:72]), "aligned"),
                    (dict(q=z(1, 64, dt=U8).expand(3, 64)), "overlap"),
                    (dict(x=z(m * 40, 3).t()), "inner stride"), (dict(x=z(0, m * 40)), "rows"),
                    (dict(x=z(3, 2, m * 20)), r"\[n, w\]")):
        with pytest.raises(RuntimeError, match=why):
            ok(**kw)
    if glu:
        with pytest.raises(RuntimeError, match="gate"):
            ok(x=z(3, 81))


def test_norm_contract(native):
    def ok(**k):
        a = dict(x=z(3, 40), delta=z(3, 40), w=z(40), q=z(3, 64, dt=FP8), s=z(3, 2, dt=E8), sum=None)
        a.update(k)
        return native._check_rmsnorm1p_mx8(*a.values())
    assert ok() == [3, 40, 40, 40, 40, 64, 2]
    assert ok(x=z(3, 50)[:, :40], delta=z(3, 44)[:, 2:42], sum=z(3, 60)[:, 20:]) == [3, 40, 50, 44, 60, 64, 2]
    assert ok(delta=None) == [3, 40, 40, 0, 0, 64, 2]
    for kw, why in ((dict(delta=None, sum=z(3, 40)), "needs delta"), (dict(w=z(41)), "x's width"),
                    (dict(w=z(40, dt=F32)), "dtype"), (dict(w=z(80)[::2]), "contiguous"),
                    (dict(delta=z(2, 40)), "3 rows"), (dict(delta=z(3, 41)), "40 wide"),
                    (dict(sum=z(3, 39)), "40 wide"), (dict(sum=z(1, 40).expand(3, 40)), "overlap"),
                    (dict(q=z(3, 32, dt=FP8)), "64 wide")):
        with pytest.raises(RuntimeError, match=why):
            ok(**kw)


def test_gemm_contract(native):
    def ok(**k):
        a = dict(wq=wq_for(native, 7, 96), xq=z(3, 96, dt=FP8), xs=z(3, 3, dt=E8), out=z(3, 7), ws=None)
        a.update(k)
        return native._check_gemm_mx4(*a.values())
    assert ok() == [3, 7, 96, 96, 3, 7]
    assert ok(ws=z(0, dt=U8)) and ok(ws=z(64, dt=U8))
    assert ok(xq=z(3, 112, dt=U8)[:, 16:], xs=z(3, 9, dt=U8)[:, 2:5], out=z(3, 9)[:, 1:8]) == [3, 7, 96, 112, 9, 9]
    for kw, why in ((dict(xq=z(3, 80, dt=FP8)), "multiple of 32"), (dict(xq=z(3, 128, dt=FP8)), "4 wide"),
                    (dict(out=z(3, 17)), "wq must hold"), (dict(out=z(2, 7)), "3 rows"),
                    (dict(out=z(3, 7, dt=F32)), "dtype"), (dict(out=z(1, 7).expand(3, 7)), "overlap"),
                    (dict(xs=z(2, 3, dt=E8)), "3 rows"), (dict(xq=z(3, 104, dt=U8)[:, 8:]), "aligned"),
                    (dict(wq=wq_for(native, 7, 96)[16:]), "wq must hold"), (dict(ws=z(65, dt=U8)[1:]), "aligned"),
                    (dict(ws=z(64)), "dtype"), (dict(ws=z(64, dt=U8)[::2]), "contiguous"),
                    (dict(out=z(7, 3).t()), "inner stride")):
        with pytest.raises(RuntimeError, match=why):
            ok(**kw)


def test_gpu_tensors_are_asked_for(native):
    wq = wq_for(native, 7, 96)
    for call in (lambda: native.mx4_quant(z(7, 96), wq), lambda: native.mx4_dequant(wq, z(7, 96)),
                 lambda: native.quant_mx8(z(3, 96), z(3, 96, dt=FP8), z(3, 3, dt=E8)),
                 lambda: native.swiglu_mx8(z(3, 192), z(3, 96, dt=FP8), z(3, 3, dt=E8)),
                 lambda: native.rmsnorm1p_mx8(z(3, 96), None, z(96), z(3, 96, dt=FP8), z(3, 3, dt=E8), 1e-6),
                 lambda: native.gemm_mx4(wq, z(3, 96, dt=FP8), z(3, 3, dt=E8), z(3, 7))):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            call()


C_CALLS = {
    "qe_mx4_quant": dict(w=A, ldw=96, wq=A, N=7, K=96, stream=None),
    "qe_mx4_dequant": dict(wq=A, out=A, ldo=96, N=7, K=96, stream=None),
    "qe_quant_mx8": dict(x=A, ldx=96, q=A, ldq=96, s=A, lds=3, n=3, K=96, stream=None),
    "qe_swiglu_mx8": dict(gu=A, ldg=192, q=A, ldq=96, s=A, lds=3, n=3, K=96, stream=None),
    "qe_rmsnorm1p_mx8": dict(x=A, ldx=96, delta=A, ldd=96, w=A, sum=A, ldsum=96, q=A, ldq=96, s=A, lds=3, n=3, K=96,
                             eps=1e-6, stream=None),
    "qe_gemm_mx4": dict(wq=A, xq=A, ldx=96, xs=A, lds=3, out=A, ldo=7, n=3, N=7, K=96, ws=None, ws_bytes=0,
                        stream=None),
}
BAD = {
    "qe_mx4_quant": [dict(w=None), dict(wq=None), dict(ldw=95), dict(wq=A + 8), dict(N=0), dict(K=0), dict(w=A + 1),
                     dict(ldw=1 << 23), dict(K=(1 << 20) + 1, ldw=1 << 21), dict(N=(1 << 24) + 1)],
    "qe_mx4_dequant": [dict(wq=None), dict(out=None), dict(ldo=95), dict(wq=A + 8), dict(N=0), dict(K=-1)],
    "qe_quant_mx8": [dict(x=None), dict(q=None), dict(s=None), dict(ldx=95), dict(ldq=95), dict(ldq=104),
                     dict(q=A + 8), dict(lds=2), dict(n=0), dict(K=0), dict(K=97, ldx=97), dict(x=A + 1)],
    "qe_swiglu_mx8": [dict(gu=None), dict(ldg=191), dict(ldq=64), dict(n=(1 << 24) + 1)],
    "qe_rmsnorm1p_mx8": [dict(x=None), dict(w=None), dict(delta=None), dict(sum=None), dict(ldd=95), dict(ldsum=95),
                         dict(q=A + 4), dict(lds=2), dict(K=0), dict(n=-3)],
    "qe_gemm_mx4": [dict(wq=None), dict(xq=None), dict(xs=None), dict(out=None), dict(ldx=95), dict(ldx=104),
                    dict(K=80), dict(lds=2), dict(ldo=6), dict(n=0), dict(N=0), dict(xq=A + 8), dict(wq=A + 8),
                    dict(out=A + 1), dict(ldo=1 << 23), dict(ws=A + 8, ws_bytes=64)],
}


@pytest.mark.parametrize("name", sorted(BAD))
def test_capi_rejects(capi, name):
    fn = getattr(capi.load(), name)
    for kw in BAD[name]:
        assert fn(*{**C_CALLS[name], **kw}.values()) == INVALID, kw
    assert capi.load().qe_mx4_bytes(0, 5) == 0 and capi.load().qe_mx4_bytes(5, 1 << 21) == 0


def test_workspace_of_any_width(native):
    """A weight's own width asks for the workspace of the product, whose rows are filled up to a multiple of 32."""
    import qengine_amd as qa
    from qengine_amd import capi
    assert native.mx4_ws_bytes(128, 5120, 17408) > 0  # K is split here
    for n, N, K in ((128, 5120, 17401), (128, 5120, 17377), (100, 513, 17400), (40, 100, 9351), (300, 5120, 6113),
                    (17, 1, 1), (1, 7, 33)):
        want = native.mx4_ws_bytes(n, N, -(-K // 32) * 32)
        assert native.mx4_ws_bytes(n, N, K) == want, (n, N, K)
        assert capi.load().qe_gemm_mx4_ws_size(n, N, K) == want
        assert qa.alloc_mx4_ws(n, N, K, device="cpu").numel() == want
    assert native.mx4_ws_bytes(128, 5120, 2 ** 20) == native.mx4_ws_bytes(128, 5120, 2 ** 20 - 31)
