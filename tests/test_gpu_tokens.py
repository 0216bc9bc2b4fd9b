"""GPU: token embedding (csrc/embed.hip) against plain float64, over types, odd sizes, strides, token distributions and both sorting paths."""
import numpy as np
import pytest
import torch

import diffsvc_amd  # noqa: F401
from diffsvc_amd import tokens as T

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF = {t: torch.finfo(t).eps / 2 for t in DTYPES}
TINY = {t: torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2 for t in DTYPES}       # half a step among the subnormals


def ids(kind, N, V, g):
    if kind == "zipf":
        t = (torch.exp(torch.rand(N, generator=g, dtype=torch.float64) * np.log(V)).long() - 1) * 31 % V
    elif kind == "one":
        t = torch.full((N,), V - 1)
    elif kind == "sorted":
        t = torch.sort(torch.randint(0, V, (N,), generator=g))[0]
    else:
        t = torch.randint(0, V, (N,), generator=g)
    return t.clamp_(0, V - 1)


def grad64(t, dy, V, scale, pad):
    """(dW, bound of a float32 sum in any order, before the last rounding) in float64 on the CPU."""
    t, d = t.cpu().long().reshape(-1), dy.detach().cpu().double().reshape(t.numel(), -1)
    ok = (t >= 0) & (t < V) & (t != (-1 if pad is None else pad))
    w, a = torch.zeros(V, d.shape[1], dtype=torch.float64), torch.zeros(V, d.shape[1], dtype=torch.float64)
    w.index_add_(0, t[ok], d[ok])
    a.index_add_(0, t[ok], d[ok].abs())
    n = torch.bincount(t[ok], minlength=V).double()[:, None]
    # n - 1 additions of at most 2^-24 of the sum of magnitudes each, one product, second-order terms below one more
    return w * scale, (n + 2) * 2.0 ** -24 * a * abs(scale)


def check_grad(got, want, bound):
    got = got.cpu()
    e = (got.double() - want).abs()
    lim = bound + (HALF[got.dtype] * (want.abs() + bound) + TINY[got.dtype])
    assert torch.isfinite(got).all() and bool((e <= lim).all()), float((e / lim.clamp_min(1e-300)).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N, V, H", [(1, 1, 1), (1, 65536, 2048), (3, 7, 5), (861, 256, 256), (65, 300, 333), (1000, 50, 8), (257, 33, 1040), (5, 9, 4100)])
def test_lookup(dtype, N, V, H):
    g = torch.Generator().manual_seed(N * 7 + H)
    w = torch.randn(V, H, generator=g).to(dtype)
    t = ids("even", N, V, g)
    for scale, tt in ((1.0, t), (H ** 0.5, t.int())):
        y = T.embed_tokens(tt.cuda(), w.cuda(), scale=scale).cpu()
        s32 = float(np.float32(scale))
        want = w[t].double() * s32
        if scale == 1.0:
            assert torch.equal(y, w[t])
        else:
            assert bool(((y.double() - want).abs() <= (HALF[dtype] * (1 + 2.0 ** -24) + 2.0 ** -24) * want.abs() + TINY[dtype]).all())


def test_lookup_shapes_strides_and_tokens_outside_the_table():
    g = torch.Generator().manual_seed(1)
    big = torch.randn(20, 48, generator=g).cuda()
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    t = torch.tensor([[0, 19, -1], [20, 7, 1 << 40]]).cuda()
    for w in (big, big[:, 1:34], big.t(), big[::2, :16], big[:, :1]):
        V = w.shape[0]
        flag.zero_()
        y = T.embed_tokens(t, w, scale=2.0, flag=flag)
        assert y.shape == (2, 3, w.shape[1]) and flag.item() == 1
        want = torch.zeros_like(y)
        for a in range(2):
            for b in range(3):
                if 0 <= int(t[a, b]) < V:
                    want[a, b] = 2 * w[int(t[a, b])]
        assert torch.equal(y, want)
    flag.zero_()
    assert T.embed_tokens(t[:1, :2].t(), big, flag=flag).shape == (2, 1, 48) and flag.item() == 0
    assert T.embed_tokens(t[:0], big).shape == (0, 3, 48)
    assert T.embed_tokens(torch.tensor(3).cuda(), big).shape == (48,)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["zipf", "one", "sorted", "even"])
@pytest.mark.parametrize("N, V, H", [
    (1, 2, 1), (2, 300, 256), (31, 5, 7), (32, 5, 8), (33, 5, 130), (64, 1, 64), (1023, 255, 33), (1025, 256, 256), (3000, 70000, 12), (4097, 257, 333),
    (8192, 300, 256), (16384, 1000, 40), (16385, 1000, 40), (20011, 65536, 24), (40000, 3, 520)])
def test_gradient(dtype, kind, N, V, H):
    g = torch.Generator().manual_seed(N + H)
    t = ids(kind, N, V, g)
    dy = (torch.randn(N, H, generator=g) * 0.1).to(dtype)
    scale = float(np.float32(H ** 0.5))
    pad = None if N % 2 else 0
    got = T.embed_tokens_grad((t.int() if H % 2 else t).cuda(), dy.cuda(), V, scale=scale, padding_idx=pad)
    assert got.dtype == dtype and got.shape == (V, H)
    check_grad(got, *grad64(t, dy, V, scale, pad))
    assert torch.equal(got, T.embed_tokens_grad(t.cuda(), dy.cuda(), V, scale=scale, padding_idx=pad))       # fixed order of sums


@pytest.mark.parametrize("kind", ["zipf", "one", "even"])
@pytest.mark.parametrize("N, V, H", [
    (9000, 300, 5), (9000, 255, 5), (5000, 70000, 6), (70000, 510, 3), (140000, 70000, 2), (270000, 200, 1), (270000, 300, 2), (300000, 131071, 2)])
def test_gradient_of_long_texts(kind, N, V, H):
    """Sorts of several blocks: digits of 8 and 9 bits, 4 to 16 places a thread, up to 64 blocks and more."""
    g = torch.Generator().manual_seed(N + V)
    t, dy = ids(kind, N, V, g), torch.randn(N, H, generator=g) * 0.1
    got = T.embed_tokens_grad(t.cuda(), dy.cuda(), V, scale=0.5, padding_idx=1)
    check_grad(got, *grad64(t, dy, V, 0.5, 1))
    assert torch.equal(got, T.embed_tokens_grad(t.int().cuda(), dy.cuda(), V, scale=0.5, padding_idx=1))


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_outputs(dtype):
    """float32 results of any type, accumulation, strided gradients and outputs, broadcast gradients, tokens outside the table, no tokens."""
    g = torch.Generator().manual_seed(5)
    N, V, H = 700, 40, 72
    t = ids("zipf", N, V, g)
    t[::9] = -1
    t[1::50] = V
    t[2::50] = 1 << 40
    big = (torch.randn(N, 2 * H, generator=g)).to(dtype).cuda()
    tc = t.cuda()
    for dy in (big[:, :H], big[:, 1:H + 1], big[:, ::2], big[:1, :H].expand(N, H), big[:, :1].expand(N, H)):
        want, bound = grad64(t, dy.cpu(), V, 1.5, 3)
        check_grad(T.embed_tokens_grad(tc, dy, V, 1.5, 3), want, bound)
        out = torch.full((V, H + 5), 7.0, device="cuda")
        T.embed_tokens_grad(tc, dy, V, 1.5, 3, out=out[:, 2:H + 2])
        check_grad(out[:, 2:H + 2], want, bound)
        assert bool((out[:, :2] == 7).all() and (out[:, H + 2:] == 7).all())
        base = torch.randn(V, H, generator=g).to(dtype)
        acc = base.cuda()
        T.embed_tokens_grad(tc, dy, V, 1.5, 3, out=acc, accumulate=True)
        check_grad(acc, base.double() + want, bound + 2.0 ** -24 * (base.double().abs() + want.abs()))
        gone = torch.bincount(t[(t >= 0) & (t < V)], minlength=V) == 0
        gone[3] = True
        assert torch.equal(acc.cpu()[gone], base[gone])
    none = T.embed_tokens_grad(tc[:0], big[:0, :H], V)
    assert none.shape == (V, H) and not none.any()
    assert not T.embed_tokens_grad(torch.full_like(tc, 3), big[:, :H], V, padding_idx=3 - V).any()
    two = T.embed_tokens_grad(tc.view(7, 100), big[:, :H].reshape(7, 100, H), V)
    assert torch.equal(two, T.embed_tokens_grad(tc, big[:, :H], V))
    with pytest.raises(ValueError, match="out must be"):
        T.embed_tokens_grad(tc, big[:, :H], V, out=torch.empty(V, H, device="cuda", dtype=torch.float64))
    with pytest.raises(ValueError, match="unit stride"):
        T.embed_tokens_grad(tc, big[:, :H], V, out=torch.empty(H, V, device="cuda").t())
    with pytest.raises(ValueError, match="accumulate"):
        T.embed_tokens_grad(tc, big[:, :H], V, accumulate=True)


def test_gradient_of_values_that_are_not_finite():
    """An infinity or NaN reaches the rows of its own token only; ignored places are never read into a sum."""
    t = torch.tensor([0, 1, 2, 2, 5, 9, -1, 4]).cuda()
    dy = torch.ones(8, 16, device="cuda")
    dy[1], dy[3], dy[0], dy[6] = float("nan"), float("inf"), float("nan"), float("nan")
    w = T.embed_tokens_grad(t, dy, 9, padding_idx=0)
    assert torch.isnan(w[1]).all() and (w[2] == float("inf")).all()
    assert torch.equal(w[[0, 3, 4, 5, 6, 7, 8]], torch.tensor([0., 0, 1, 1, 0, 0, 0], device="cuda")[:, None].expand(7, 16))


def test_autograd_and_module():
    g = torch.Generator().manual_seed(2)
    m = T.TokenEmbeddingHip(50, 24, padding_idx=0, scale=2.0).cuda()
    t = ids("zipf", 300, 50, g).view(3, 100)
    r = torch.randn(3, 100, 24, generator=g)
    y = m(t.cuda())
    (y * r.cuda()).sum().backward()
    assert torch.equal(y.detach().cpu(), m.weight.detach().cpu()[t] * 2.0)
    check_grad(m.weight.grad, *grad64(t, r, 50, 2.0, 0))
    m.check()
    m(torch.tensor([50]).cuda())
    with pytest.raises(IndexError):
        m.check()
    m.check()
    with torch.no_grad():
        assert not m(t.cuda()).requires_grad
    # differences of the (linear) map: <r, y(W + h D) - y(W)> / h = <dW, D> exactly up to rounding
    w, D = m.weight.detach(), torch.randn(50, 24, generator=g).cuda()
    D[0] = 0
    f = lambda ww: float((T.embed_tokens(t.cuda(), ww, 2.0).double() * r.cuda().double()).sum())
    num, ana = (f(w + D) - f(w - D)) / 2, float((m.weight.grad.double() * D.double()).sum())
    size = float((T.embed_tokens(t.cuda(), w.abs() + D.abs(), 2.0).double() * r.cuda().double().abs()).sum())
    assert abs(num - ana) <= 300 * 2.0 ** -24 * size


def test_streams_and_graph_replay():
    """On another stream than the default one; captured and replayed on new contents while eager calls run in between."""
    g = torch.Generator().manual_seed(9)
    N, V, H = 20000, 500, 64
    t, dy = ids("zipf", N, V, g).cuda(), torch.randn(N, H, generator=g).cuda()
    want = T.embed_tokens_grad(t, dy, V, padding_idx=0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        w1, y1 = T.embed_tokens_grad(t, dy, V, padding_idx=0), T.embed_tokens(t, want, 0.5)
    s.synchronize()
    assert torch.equal(w1, want) and torch.equal(y1, want[t] * 0.5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        wg = T.embed_tokens_grad(t, dy, V, padding_idx=0)
        yg = T.embed_tokens(t, wg, 0.5)
    for k in range(4):
        t.copy_(ids("even" if k % 2 else "one", N, V, g))
        dy.copy_(torch.randn(N, H, generator=g))
        graph.replay()
        e = T.embed_tokens_grad(t, dy, V, padding_idx=0)
        assert torch.equal(wg, e) and torch.equal(yg, e[t] * 0.5), k
        torch.cuda.synchronize()


def test_offsets_beyond_32_bits():
    """A table of 2^31 + elements (rows and gradients at its end)."""
    V, H = (1 << 20) + 7, 2056
    w = torch.empty(V, H, device="cuda", dtype=torch.bfloat16)
    w[-9:] = torch.arange(9, device="cuda", dtype=torch.bfloat16)[:, None] + 1
    w[:3] = 0.5
    t = torch.tensor([V - 1, 0, V - 9, 2, V - 1], device="cuda")
    y = T.embed_tokens(t, w, 2.0)
    assert torch.equal(y[:, 0].float().cpu(), torch.tensor([18.0, 1, 2, 1, 18])) and bool((y == y[:, :1]).all())
    del w
    g = T.embed_tokens_grad(t, y, V)
    assert torch.equal(g[-1].float(), torch.full((H,), 36.0, device="cuda")) and torch.equal(g[V - 9], y[2]) and torch.equal(g[2], y[3])
    assert not g[3:V - 9].any() and not g[V - 8:V - 1].any()


def test_module_captured_with_its_backward_pass():
    """A first call of the module inside a capture, gradient and all, replayed on new tokens; its flag is not the graph's memory."""
    torch.manual_seed(0)
    m = T.TokenEmbeddingHip(40, 16, padding_idx=0, scale=0.5).cuda()
    t, r = torch.randint(0, 40, (500,), device="cuda"), torch.randn(500, 16, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):                             # (autograd's own first-use work happens outside the capture)
        torch.autograd.grad((T.embed_tokens(t, m.weight) * r).sum(), m.weight)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m(t)
        dw, = torch.autograd.grad(y, m.weight, r)
    for k in range(4):
        t.copy_(torch.randint(0, 40, (500,), device="cuda"))
        r.copy_(torch.randn(500, 16, device="cuda"))
        graph.replay()
        with torch.no_grad():
            assert torch.equal(y.detach(), m.weight[t] * 0.5), k
        assert torch.equal(dw, T.embed_tokens_grad(t, r, 40, 0.5, 0)), k
        torch.cuda.synchronize()
    m.check()
    t[3] = 40
    graph.replay()
    with pytest.raises(IndexError):
        m.check()
    graph.replay()
    with pytest.raises(IndexError):
        m.check()
    assert list(m.state_dict()) == ["weight"]


@pytest.mark.parametrize("V", [1 << 30, (1 << 30) - 15])
def test_gradient_of_a_table_with_the_most_rows(V):
    """2^30 rows: more rows to zero than one launch has waves for."""
    t = torch.tensor([V - 1, 5, V - 1, V - 17, V, 1 << 29], device="cuda")
    dy = torch.arange(1, 7, device="cuda", dtype=torch.float32)[:, None].bfloat16()
    out = torch.full((V, 1), 9.0, device="cuda", dtype=torch.bfloat16)
    T.embed_tokens_grad(t, dy, V, out=out)
    assert [out[i, 0].item() for i in (V - 1, 5, V - 17, 1 << 29)] == [4, 2, 4, 6]
    assert int(torch.count_nonzero(out)) == 4
    T.embed_tokens_grad(t[:2], dy[:2], V, out=out, accumulate=True)
    assert out[V - 1, 0].item() == 5 and out[5, 0].item() == 4 and int(torch.count_nonzero(out)) == 4


@pytest.mark.parametrize("dtype", DTYPES)
def test_lookup_rounds_the_float32_product_whatever_the_alignment(dtype):
    """scale * value in float32, then one rounding: rows of 8 aligned columns, and the same rows element by element.  Among the scales are ones where
    the exact product, rounded once, would be another fp16 number (a float32 product that lies on a tie)."""
    m = (1 + torch.arange(1024) / 1024).half()
    scales = [s for s in (float(np.float32(k ** 0.5)) for k in range(2, 400)) if ((m.double() * s).numpy().astype(np.float16) != (m.float() * s).half().numpy()).any()]
    assert len(scales) >= 5
    g = torch.Generator().manual_seed(3)
    w = torch.cat([m.float().repeat(60), torch.randn(100, generator=g)]).to(dtype)[:61504].view(-1, 64).cuda()
    t = torch.randperm(w.shape[0], generator=g).cuda()
    wide = torch.zeros(w.shape[0], 65, device="cuda", dtype=dtype)
    wide[:, 1:] = w
    for scale in scales[:5] + [16.0, 0.1]:
        want = (w[t].float() * float(np.float32(scale))).to(dtype)
        assert torch.equal(T.embed_tokens(t, w, scale), want) and torch.equal(T.embed_tokens(t, wide[:, 1:], scale), want), scale
