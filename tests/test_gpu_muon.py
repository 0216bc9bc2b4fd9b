"""GPU: the Newton-Schulz orthogonalisation and the optimisation step on it (csrc/ortho.hip) against the formula in float64.

Tolerances.  The iteration is smooth (|d/ds s(a + b s^2 + c s^4)| <= 3.9 on [0, 1.2]) but it amplifies a rounding of an early iterate by up to that
factor per step, in the directions where it grows; a bound over all directions (3.9^4) says nothing.  So the error is measured where it
arises: ``model`` runs the formula with every stored matrix rounded as the operator's description says (one fp16 plane, or two: 11 or 22 bits) and
sums in float32, and its distance from float64 is a sample of the same random rounding errors.  Over many elements that distance
concentrates, so the kernel's may be at most 3 times as large in the 2-norm, plus the float32 sums' own part (2^-24 per step, amplified: 64 * 2^-24)
and the last rounding (half a step of the type).  Matrices of few elements do not average: there the plateau's derivative (at most 4 in
magnitude where the singular value 1 of a single row goes) over ten roundings of a step, 40 half steps of the stored precision, is allowed instead."""
import pytest
import torch

import diffsvc_amd  # noqa: F401
from diffsvc_amd import muon as M

COEF = M.COEFFICIENTS


def planes(x, n, scale):
    """x as n fp16 planes at a power-of-two scale hold it."""
    hi = (x * scale).half()
    if n == 1:
        return hi.double() / scale, (hi.float(),)
    lo = (x * scale - hi.double()).half()
    return (hi.double() + lo.double()) / scale, (hi.float(), lo.float())


def mm(a, b):
    """float32 products of planes, hi hi + lo hi + hi lo."""
    s = a[0] @ b[0]
    if len(a) == 2:
        s = s + a[1] @ b[0] + a[0] @ b[1]
    return s.double()


def exact(g, steps=5, coef=COEF, eps=1e-7, scale=1.0):
    a, b, c = coef
    x = g.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2) if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        A = x @ x.transpose(-1, -2)
        x = a * x + (b * A + c * (A @ A)) @ x
    return (x.transpose(-1, -2) if tall else x) * scale


def model(g, n, steps=5, coef=COEF, eps=1e-7, scale=1.0):
    a, b, c = coef
    out = []
    for x in g.double().reshape(-1, *g.shape[-2:]):
        tall = x.shape[-2] > x.shape[-1]
        x = (x.t() if tall else x).contiguous()
        norm = x.square().sum().sqrt()
        x = x / (norm + eps)
        t = max(float(norm / (norm + eps)), 1e-18)
        S = 4096.0 / max(t, 2.0 ** -60) if t < 0.5 else 4096.0           # tiny iterates are held at a larger scale
        eye = torch.eye(x.shape[0], dtype=torch.float64)
        for k in range(steps):
            x, xp = planes(x, n, S)
            A = mm(xp, tuple(p.t().contiguous() for p in xp)) / (S * S)
            A, Ap = planes(A, n, 1024.0)
            m = a * eye + b * A + c * mm(Ap, Ap) / 1024.0 ** 2
            m, mp = planes(m, n, 1024.0)
            x = mm(mp, xp) / (1024.0 * S)
            S = max(4096.0, S / 4)
        out.append((x.t() if tall else x) * scale)
    return torch.stack(out).reshape(g.shape)


def limit(g, dtype, n, **kw):
    """(exact result, allowed 2-norm of the error, allowed largest error) of one matrix batch, per matrix."""
    want = exact(g, **kw)
    ref = model(g, n, **kw) - want
    num = g.shape[-1] * g.shape[-2]
    norm = want.square().sum((-2, -1)).sqrt()
    half = torch.finfo(dtype).eps / 2
    few = 40 * 2.0 ** (-11 * n) if num < 4096 else 0.0
    two = 3 * ref.square().sum((-2, -1)).sqrt() + (64 * 2.0 ** -24 + few) * norm
    big = 6 * two / num ** 0.5 if num >= 4096 else two                    # six standard deviations of an element, all elements of one size
    return want, two + half * norm, big[..., None, None] + half * want.abs() + torch.finfo(dtype).tiny


def close(got, g, dtype, n, **kw):
    want, two, big = limit(g, dtype, n, **kw)
    e = got.detach().cpu().double() - want
    assert torch.isfinite(e).all()
    f = e.square().sum((-2, -1)).sqrt() / two.clamp_min(1e-300)
    m = (e.abs() / big).amax()
    assert float(f.max()) <= 1 and float(m) <= 1, (float(f.max()), float(m))


def update(shape, seed, size=1e-3):
    g = torch.Generator().manual_seed(seed)
    *b, r, c = shape
    k = max(1, min(r, c) // 16)
    return (torch.randn(*b, r, k, generator=g) @ torch.randn(*b, k, c, generator=g) / k ** 0.5 + torch.randn(*b, r, c, generator=g)) * size


CASES = [(1, 1), (1, 5), (7, 1), (2, 3), (16, 16), (31, 33), (64, 129), (129, 64), (127, 128), (128, 128), (130, 131), (257, 100), (100, 700), (1, 1000), (600, 3),
         (384, 384), (300, 520)]


@pytest.mark.gpu
@pytest.mark.parametrize("r, c", CASES)
@pytest.mark.parametrize("dtype, precision", [(torch.float32, None), (torch.float32, "f16"), (torch.float16, None), (torch.bfloat16, None), (torch.bfloat16, "f16_x3")])
def test_orthogonalize(r, c, dtype, precision):
    g = update((2, r, c), r * 1000 + c).to(dtype)
    got = M.orthogonalize(g.cuda(), precision=precision, scale=1.5)
    assert got.dtype == dtype and got.shape == g.shape
    close(got, g, dtype, 2 if precision == "f16_x3" or (precision is None and dtype != torch.bfloat16) else 1, scale=1.5)
    assert torch.equal(got, M.orthogonalize(g.cuda(), precision=precision, scale=1.5))


@pytest.mark.gpu
@pytest.mark.parametrize("shape, dtype", [((1100, 1300), torch.bfloat16), ((3, 512, 1024), torch.float32), ((2, 150, 4100), torch.float32), ((4100, 70), torch.float16),
                                          ((24, 40, 30), torch.float32), ((300, 20, 31), torch.bfloat16), ((2, 64, 256), torch.float32), ((2, 65, 256), torch.float32),
                                          ((33, 497), torch.float16), ((31, 512), torch.float32), ((513, 32), torch.float32)])
def test_orthogonalize_larger(shape, dtype):
    g = update(shape, 77).to(dtype)
    close(M.orthogonalize(g.cuda()), g, dtype, 1 if dtype == torch.bfloat16 else 2)


@pytest.mark.gpu
def test_steps_and_coefficients():
    g = update((3, 90, 140), 4)
    for steps in (1, 2, 3, 8, 12):
        close(M.orthogonalize(g.cuda(), steps=steps, coefficients=(1.5, -0.5, 0.0)), g, torch.float32, 2, steps=steps, coef=(1.5, -0.5, 0.0))
    close(M.orthogonalize(g.cuda(), steps=1), g, torch.float32, 2, steps=1)
    q = M.orthogonalize(g.cuda(), steps=30, coefficients=(1.875, -1.25, 0.375)).double()
    eye = torch.eye(90, device="cuda", dtype=torch.float64)
    # converged: the fixed point 1 is reached to the stored precision; 90 columns of 140 products of two values with 22 bits
    assert float((q @ q.transpose(1, 2) - eye).abs().max()) < 1e-5


@pytest.mark.gpu
def test_sizes_of_updates():
    """Tiny, huge and zero updates, and ones that eps swamps: the norm is summed in 64 bits, small iterates are held at their own scale."""
    g = update((60, 100), 5, 1.0)
    for size in (1e-30, 1e-18, 1e12, 1e30):
        close(M.orthogonalize((g * size).cuda(), eps=0.0), g * size, torch.float32, 2, eps=0.0)
    for size in (1e-7, 1e-9, 1e-11, 1e-14):
        x = g * size
        close(M.orthogonalize(x.cuda()), x, torch.float32, 2)
        close(M.orthogonalize(x.cuda(), precision="f16"), x, torch.float32, 1)
    assert not M.orthogonalize(torch.zeros(5, 7, device="cuda")).any()
    assert torch.isnan(M.orthogonalize(torch.zeros(5, 7, device="cuda"), eps=0.0)).all()
    z = torch.stack([g, torch.zeros_like(g), g]).cuda()
    o = M.orthogonalize(z)
    assert torch.equal(o[0], o[2]) and not o[1].any()
    z[1, 3, 4] = float("nan")
    z[0, 0, 0] = float("inf")
    p = M.orthogonalize(z)
    assert torch.equal(p[2], o[2]) and torch.isnan(p[1]).all() and torch.isnan(p[0]).any()


@pytest.mark.gpu
def test_strides_and_in_place():
    g = update((4, 80, 200), 6)
    buf = torch.zeros(4, 80, 260, device="cuda")
    buf[:, :, 30:230] = g.cuda()
    want = M.orthogonalize(g.cuda())
    assert torch.equal(M.orthogonalize(buf[:, :, 30:230]), want)
    assert torch.equal(M.orthogonalize(g.cuda().transpose(1, 2)).transpose(1, 2), want)
    assert torch.equal(M.orthogonalize(g.cuda().view(2, 2, 80, 200)).view(4, 80, 200), want)
    M.orthogonalize(buf[:, :, 30:230], out=buf[:, :, 30:230])
    assert torch.equal(buf[:, :, 30:230], want) and not buf[:, :, :30].any() and not buf[:, :, 230:].any()
    assert torch.equal(M.orthogonalize(buf.new_zeros(0, 3, 4)), buf.new_zeros(0, 3, 4))
    assert M.orthogonalize(buf.new_zeros(2, 0, 4)).shape == (2, 0, 4)
    for shape in ((6, 20, 30), (6, 80, 90)):                               # one workgroup a matrix, and many
        z = update((shape[0] + 1, *shape[1:]), 9).cuda()
        want = M.orthogonalize(z[:-1].clone())
        assert torch.equal(M.orthogonalize(z[:-1], out=z[1:]), want)      # the result of one matrix where the next one lies
    with pytest.raises(RuntimeError, match="singular values"):
        M.orthogonalize(buf, coefficients=(9.0, 9.0, 9.0))
    with pytest.raises(ValueError, match="in place"):
        M.orthogonalize(g.cuda(), out=torch.empty(4, 200, 80, device="cuda").transpose(1, 2))
    with pytest.raises(ValueError, match="out must be"):
        M.orthogonalize(g.cuda(), out=torch.empty(4, 80, 200, device="cuda", dtype=torch.float16))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(5, 1, 1), (2, 33, 70), (70, 33), (3, 256, 128)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step(dtype, shape, nesterov):
    p, g = update(shape, 1, 1.0).to(dtype), update(shape, 2).to(dtype)
    m = update(shape, 3, 3e-4)
    lr, mu, wd, gs, sc = 0.25, 0.9375, 0.125, 0.5, 0.75                    # exact in fp32
    pc, mc = p.cuda(), m.cuda()
    M.muon_step_(pc, g.cuda(), mc, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=wd, scale=sc, grad_scale=torch.tensor([gs], device="cuda"))
    g64 = g.double() * gs
    m64 = mu * m.double() + (1 - mu) * g64
    # three float32 roundings of terms no larger than these
    assert bool(((mc.cpu().double() - m64).abs() <= 3 * 2.0 ** -24 * (mu * m.double().abs() + (1 - mu) * g64.abs()) + 1e-40).all())
    u = (1 - mu) * g64 + mu * mc.cpu().double() if nesterov else mc.cpu().double()
    want, two, big = limit(u, torch.float32, 1 if dtype == torch.bfloat16 else 2, scale=sc)
    new = (1 - lr * wd) * p.double() - lr * want
    half = torch.finfo(dtype).eps / 2
    # u itself has been rounded to 24 bits, which the iteration treats as any other input's rounding (part of `two`'s float32 share)
    e = (pc.cpu().double() - new).abs()
    assert bool((e <= lr * big + (half + 2.0 ** -23) * (new.abs() + lr * big) + torch.finfo(dtype).tiny).all())
    p2, m2 = p.cuda(), m.cuda()
    M.muon_step_(p2, g.cuda(), m2, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=wd, scale=sc, grad_scale=gs)
    assert torch.equal(p2, pc) and torch.equal(m2, mc)


@pytest.mark.gpu
def test_muon_step_refusals():
    p = torch.zeros(2, 4, 6, device="cuda")
    with pytest.raises(ValueError, match="grad must be"):
        M.muon_step_(p, p.half(), p.clone(), 0.1)
    with pytest.raises(ValueError, match="momentum_buffer"):
        M.muon_step_(p, p.clone(), p.half(), 0.1)
    with pytest.raises(ValueError, match="grad_scale"):
        M.muon_step_(p, p.clone(), p.clone(), 0.1, grad_scale=torch.ones(2, device="cuda"))
    with pytest.raises(ValueError, match="in place"):
        M.muon_step_(p.transpose(1, 2), p.transpose(1, 2), torch.zeros(2, 6, 4, device="cuda"), 0.1)
    with pytest.raises(RuntimeError, match="momentum"):
        M.muon_step_(p, p.clone(), p.clone(), 0.1, momentum=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 3, 4), (2, 0, 3, 4), (2, 2, 0, 5), (2, 3, 4, 0)])
def test_nothing_to_do(shape):
    x = torch.zeros(shape, device="cuda")
    assert M.orthogonalize(x).shape == shape
    assert M.muon_step_(x, torch.zeros_like(x), torch.zeros_like(x), 0.1).shape == shape


@pytest.mark.gpu
def test_streams_and_graph_replay():
    g = update((2, 200, 300), 8).cuda()
    want = M.orthogonalize(g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = M.orthogonalize(g)
    b = M.orthogonalize(g)                                                 # at the same time, on its own workspace
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want)
    p, m = update((2, 200, 300), 9, 1.0).cuda(), torch.zeros(2, 200, 300, device="cuda")
    pe, me = p.clone(), m.clone()
    # (split along K, and small enough for one workgroup: their own counters and LDS on every replay)
    wide, small = update((120, 3000), 10).cuda(), update((5, 20, 40), 11).cuda()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    M.muon_step_(p.clone(), g, m.clone(), 0.1)
    with torch.cuda.graph(graph):
        M.muon_step_(p, g, m, 0.1)
    with torch.cuda.graph(other, pool=graph.pool()):
        o, ow, os = M.orthogonalize(g), M.orthogonalize(wide), M.orthogonalize(small)
    for k in range(4):
        g.copy_(update((2, 200, 300), 20 + k))
        graph.replay()
        M.muon_step_(pe, g, me, 0.1)
        assert torch.equal(p, pe) and torch.equal(m, me), k
        other.replay()
        assert torch.equal(o, M.orthogonalize(g)) and torch.equal(ow, M.orthogonalize(wide)) and torch.equal(os, M.orthogonalize(small))
        torch.cuda.synchronize()


def test_model_is_the_formula():
    """The oracle's own check (CPU): with exact planes the model is the formula, and its rounded form is as far off as its bits say."""
    g = update((40, 64), 3)
    want = exact(g)
    r1, r2 = float((model(g, 1) - want).norm() / want.norm()), float((model(g, 2) - want).norm() / want.norm())
    assert 1e-5 < r1 < 2e-2 and r2 < 1e-5, (r1, r2)
    u, s, v = torch.linalg.svd(g.double() / (g.double().norm() + 1e-7), full_matrices=False)
    for _ in range(5):
        s = s * (COEF[0] + COEF[1] * s ** 2 + COEF[2] * s ** 4)
    assert float((u * s @ v - want).abs().max()) < 1e-12
