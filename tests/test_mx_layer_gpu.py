"""The linear layers on 4-bit weights together, as a step uses them: MX4MLP (norm with the residual's addition, gate
and up, SwiGLU, down) for decode rows, a verify pass and a prompt's chunk, every step checked against the 64-bit
oracle on what the step before it wrote; and captured."""
import pytest
import torch

import mx_cases as C
from oracle import mx_oracle as M

pytestmark = pytest.mark.gpu
BF, F64, DEV = C.BF, C.F64, C.DEV
H, I, EPS = 1024, 2736, 1e-6


@pytest.fixture(scope="module")
def mlp(native):
    from qengine_amd.layer import MX4MLP
    g = C.gen(11)
    norm, gu, down = C.randn(g, H, scale=0.1), C.randn(g, 2 * I, H, scale=H ** -0.5), C.randn(g, H, I, scale=I ** -0.5)
    return MX4MLP(norm.to(DEV), gu.to(DEV), down.to(DEV), EPS, rows=400), (norm, gu, down)


@pytest.mark.parametrize("n", [1, 5, 8, 40, 333])
def test_mlp(mlp, n):
    layer, (norm, gu, down) = mlp
    g = C.gen(n)
    h, d = C.randn(g, n, H, scale=3.0), C.randn(g, n, H)
    hd, dd = h.to(DEV), d.to(DEV)
    out = torch.empty(n, H, dtype=BF, device=DEV)
    layer(hd, dd, out)
    want, y = M.rmsnorm1p(h, d, norm, EPS)
    assert torch.equal(hd.cpu(), want)
    xq, xs = (t[:n].cpu() for t in layer.x)
    C.check_rows(xq, xs, y, 29 * 2.0 ** -24)
    C.check_product(layer.gu[:n], M.values8(xq, xs), M.values4(*M.quant4(gu)), H)
    got = layer.gu[:n].cpu()
    aq, as_ = (t[:n].cpu() for t in layer.act)
    C.check_rows(aq, as_, M.swiglu(got), (float(got[:, :I].float().abs().max()) + 8) * 2.0 ** -23)
    C.check_product(out, M.values8(aq, as_), M.values4(*M.quant4(down)), I)
    # the output may take the residual's place
    layer(h.to(DEV), dd, dd)
    assert torch.equal(dd, out)


def test_verify_rows_equal_plain_decoding(mlp):
    layer, _ = mlp
    g = C.gen(77)
    h, d = C.randn(g, 8, H).to(DEV), C.randn(g, 8, H).to(DEV)
    alone = torch.empty(8, H, dtype=BF, device=DEV)
    for r in range(8):
        layer(h[r: r + 1].clone(), d[r: r + 1], alone[r: r + 1])
    for n in (2, 5, 8):
        out = torch.empty(n, H, dtype=BF, device=DEV)
        layer(h[:n].clone(), d[:n], out)
        assert torch.equal(out, alone[:n])


@pytest.mark.parametrize("n", [1, 5, 200])
def test_captured(mlp, n):
    """A pass as one graph, replayed on changed rows with eager passes between."""
    layer, _ = mlp
    g = C.gen(n + 50)
    h, d, out = (torch.zeros(n, H, dtype=BF, device=DEV) for _ in range(3))
    layer(h, d, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(h, d, out)
    for k in range(4):
        a, b = C.randn(g, n, H), C.randn(g, n, H)
        h.copy_(a)
        d.copy_(b)
        graph.replay()
        kept, after = out.clone(), h.clone()
        ref, h2 = torch.empty_like(out), a.to(DEV)
        layer(h2, b.to(DEV), ref)
        torch.cuda.synchronize()
        assert torch.equal(kept, ref) and torch.equal(after, h2), k


@pytest.mark.parametrize("K", [17401, 17377])
def test_linear_of_any_width(native, K):
    """A layer whose width is no multiple of 32 has the workspace of its filled-up rows, and so the bits of a layer
    that is filled up with zeros."""
    from qengine_amd import alloc_mx8
    from qengine_amd.layer import MX4Linear
    n, N, Kp = 100, 513, -(-K // 32) * 32
    g = C.gen(K)
    w, x = C.randn(g, N, K, scale=K ** -0.5), C.randn(g, n, K).to(DEV)
    layer, wide = (MX4Linear(t.to(DEV), rows=n) for t in (w, torch.nn.functional.pad(w, (0, Kp - K))))
    assert layer.ws.numel() == wide.ws.numel() > 0
    q, s = alloc_mx8(n, K)
    native.quant_mx8(x, q, s)
    out, same = torch.empty(n, N, dtype=BF, device=DEV), torch.empty(n, N, dtype=BF, device=DEV)
    layer(q, s, out)
    C.check_product(out, M.values8(q.cpu(), s.cpu()), M.values4(*M.quant4(w)), Kp)
    wide(q, s, same)
    assert torch.equal(out, same)


def test_layers_that_share_their_scratch(native):
    """Two layers one after another on one scratch: the bits of layers that own theirs, eagerly and as one graph."""
    from qengine_amd.layer import MX4MLP
    g = C.gen(21)
    n, hidden, inner = 70, 512, 17408  # the second product has a workspace
    made = []
    for _ in range(2):
        made.append([t.to(DEV) for t in (C.randn(g, hidden, scale=0.1), C.randn(g, 2 * inner, hidden, scale=hidden ** -0.5),
                                         C.randn(g, hidden, inner, scale=inner ** -0.5))])
    own = [MX4MLP(*w, EPS, rows=n) for w in made]
    first = MX4MLP(*made[0], EPS, rows=n)
    second = MX4MLP(*made[1], EPS, rows=n, share=first)
    assert first.down.ws.numel() > 0
    for a, b in ((first.x, second.x), (first.act, second.act), ((first.gu, first.down.ws), (second.gu, second.down.ws))):
        assert [t.data_ptr() for t in a] == [t.data_ptr() for t in b]
    h, d = C.randn(g, n, hidden, scale=3.0).to(DEV), C.randn(g, n, hidden).to(DEV)

    def run(layers, h, d, out):
        for layer in layers:
            layer(h, d, out)
            d = out
    want, want_h = torch.empty_like(h), h.clone()
    run(own, want_h, d, want)
    got, got_h = torch.empty_like(h), h.clone()
    run((first, second), got_h, d, got)
    assert torch.equal(got, want) and torch.equal(got_h, want_h)
    static, out = h.clone(), torch.empty_like(h)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run((first, second), static, d, out)
    for _ in range(3):
        static.copy_(h)
        graph.replay()
        run((first, second), h.clone(), d, got)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(static, want_h) and torch.equal(got, want)
