"""The lookup under torch's transforms, against nn.functional.embedding under the same: forward-mode derivatives, traces, derivatives of derivatives, torch.func.
On the device, and on the
host with the two kernel launches replaced by numpy -- code that no transform can look into, as the kernels are."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F
from torch.autograd import forward_ad as fw

import diffsvc_amd  # noqa: F401
from diffsvc_amd import tokens as T

V, H, PAD, SCALE = 11, 8, 3, 2.0                       # sums of few small integers: exact in every order


def _lookup(tokens, weight, scale, flag):
    t, w = tokens.numpy(), weight.detach().numpy()
    ok = (t >= 0) & (t < w.shape[0])
    if flag is not None and not ok.all():
        flag.fill_(1)
    return torch.from_numpy(np.where(ok[..., None], w[np.where(ok, t, 0)] * np.float32(scale), np.float32(0)).astype(np.float32))


def _grad(tokens, dy, vocab, scale=1.0, padding_idx=None):
    t, d = tokens.numpy().reshape(-1), dy.detach().numpy().reshape(tokens.numel(), -1)
    ok = (t >= 0) & (t < vocab) & (t != (-1 if padding_idx is None else padding_idx))
    w = np.zeros((vocab, d.shape[1]), np.float32)
    np.add.at(w, t[ok], d[ok] * np.float32(scale))
    return torch.from_numpy(w)


@pytest.fixture(params=["host", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request, monkeypatch):
    if request.param == "host":
        monkeypatch.setattr(T, "_lookup", _lookup)
        monkeypatch.setattr(T, "embed_tokens_grad", _grad)
        return "cpu"
    return "cuda"


def small(*shape, seed=0, dev="cpu"):
    return torch.randint(-4, 5, shape, generator=torch.Generator().manual_seed(seed)).float().to(dev)


def tokens(dev, *shape, seed=1):
    return torch.randint(0, V, shape, generator=torch.Generator().manual_seed(seed)).to(dev)


def plain(t, w):
    return F.embedding(t, w, padding_idx=PAD) * SCALE


def ours(t, w, flag=None):
    return T.embed_tokens(t, w, SCALE, PAD, flag)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("mode", [True, False])
def test_forward_mode(dev, grad, mode):
    """The table's tangent reaches the output: frozen and trained tables, with grad mode on and off."""
    w, dw, t = small(V, H, dev=dev).requires_grad_(grad), small(V, H, seed=2, dev=dev), tokens(dev, 4, 5)
    with fw.dual_level(), torch.set_grad_enabled(mode):
        got, want = (fw.unpack_dual(f(t, fw.make_dual(w, dw))) for f in (ours, plain))
        assert torch.equal(got.primal, want.primal) and torch.equal(got.tangent, want.tangent) and got.tangent.any()
        assert fw.unpack_dual(ours(t, w)).tangent is None
    assert got.primal.requires_grad == (grad and mode)
    if grad and mode:
        got.primal.sum().backward()
        assert not w.grad[PAD].any() and w.grad.any()


def test_derivatives_of_derivatives(dev):
    """d/dr of <dW(r), D> is the lookup of D without the padding's places; the gradient of a gradient's square; forward over backward."""
    t, r0, D = tokens(dev, 4, 5), small(4, 5, H, seed=3, dev=dev), small(V, H, seed=4, dev=dev)
    assert (t == PAD).any()
    res = []
    for f in (ours, plain):
        w, r = small(V, H, dev=dev).requires_grad_(True), r0.clone().requires_grad_(True)
        dw, = torch.autograd.grad((f(t, w) * r).sum(), w, create_graph=True)
        first = torch.autograd.grad((dw * D).sum(), r, retain_graph=True)[0]
        second = torch.autograd.grad((dw * dw).sum(), r, create_graph=True)[0]
        third = torch.autograd.grad((second * second).sum(), r)[0]
        d2 = torch.autograd.grad(((f(t, w) ** 2).sum()), w, create_graph=True)[0]
        hvp = torch.autograd.grad((d2 * D).sum(), w)[0]
        with fw.dual_level():
            x = fw.make_dual(w.detach().clone().requires_grad_(True), D)
            jg = fw.unpack_dual(torch.autograd.grad((f(t, x) ** 2).sum(), x, create_graph=True)[0]).tangent
        res.append((dw, first, second, third, d2, hvp, jg))
    for a, b in zip(*res):
        assert torch.equal(a, b) and b.any()


def test_func_transforms(dev):
    t, tb, w, wb = tokens(dev, 6), tokens(dev, 3, 6, seed=7), small(V, H, dev=dev), small(3, V, H, seed=8, dev=dev)
    assert (tb == PAD).any()
    f = torch.func
    loss = lambda g: lambda t, w: (g(t, w) ** 2).sum()
    calls = [lambda g: f.vmap(g, (0, None))(tb, w), lambda g: f.vmap(g, (None, 0))(t, wb), lambda g: f.vmap(g, (0, 0))(tb, wb), lambda g: f.vmap(g, (1, 2))(tb.t(), wb.permute(1, 2, 0)),
             lambda g: f.vmap(f.vmap(g, (0, None)), (None, 0))(tb, wb), lambda g: f.grad(loss(g), 1)(t, w), lambda g: f.vmap(f.grad(loss(g), 1), (0, None))(tb, w),
             lambda g: f.vmap(f.grad(loss(g), 1), (0, 0))(tb, wb), lambda g: f.jvp(lambda x: g(t, x), (w,), (wb[0],))[1], lambda g: f.vjp(lambda x: g(t, x), w)[1](small(6, H, seed=9, dev=dev))[0],
             lambda g: f.jacrev(g, 1)(t[:2], w), lambda g: f.jacfwd(g, 1)(t[:2], w), lambda g: f.hessian(loss(g), 1)(t[:3], w[:, :2].contiguous()),
             lambda g: f.jvp(f.grad(lambda x: loss(g)(t, x)), (w,), (wb[1],))[1]]
    for i, c in enumerate(calls):
        a, b = c(ours), c(plain)
        assert a.shape == b.shape and torch.equal(a, b) and b.any(), i
    with torch.no_grad():
        assert torch.equal(f.vmap(ours, (0, None))(tb, w), plain(tb, w))


@pytest.mark.gpu
def test_func_transforms_of_the_module():
    """With the module's flag in the call; what torch's older batching cannot look into is refused, not answered."""
    m = T.TokenEmbeddingHip(V, H, padding_idx=PAD, scale=SCALE).cuda()
    m.weight.data.copy_(small(V, H, dev="cuda"))
    t, wb = tokens("cuda", 3, 6, seed=7), small(3, V, H, seed=8, dev="cuda")
    assert torch.equal(torch.func.vmap(m)(t), plain(t, m.weight))
    call = lambda w, t: torch.func.functional_call(m, {"weight": w}, (t,))
    assert torch.equal(torch.func.vmap(call)(wb, t), torch.stack([plain(a, b) for a, b in zip(t, wb)]))
    assert torch.equal(torch.func.grad(lambda w: (call(w, t) ** 2).sum())(wb[0]), torch.func.grad(lambda w: (plain(t, w) ** 2).sum())(wb[0]))
    m.check()
    t[1, 2] = V
    torch.func.vmap(m)(t)
    with pytest.raises(IndexError):
        m.check()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(m(t[0]), m.weight, small(4, 6, H, seed=2, dev="cuda"), is_grads_batched=True)


@pytest.mark.parametrize("trained", [False, True])
def test_trace(dev, trained, tmp_path):
    """A traced lookup is the lookup, on tokens, tables and shapes that it was not traced on, with its gradient and its flag, saved and loaded too."""
    w, t = small(V, H, dev=dev).requires_grad_(trained), tokens(dev, 4, 5)
    flag = torch.zeros(1, dtype=torch.int32, device=dev)
    traced = torch.jit.trace(lambda a, b, c: ours(a, b, c) + 1, (t, w, flag))
    torch.jit.save(traced, str(tmp_path / "t.pt"))
    w2, t2 = small(V, H, seed=5, dev=dev), tokens(dev, 9, seed=6)
    for f in (traced, torch.jit.load(str(tmp_path / "t.pt"))):
        assert "embed_tokens" in str(f.graph)
        for _ in range(3):                                                 # (the executor looks at the first runs before it settles)
            x = w2.clone().requires_grad_(True)
            y = f(t2, x, flag)
            assert torch.equal(y, plain(t2, w2) + 1)
            y.sum().backward()
            z = w2.clone().requires_grad_(True)
            plain(t2, z).sum().backward()
            assert torch.equal(x.grad, z.grad) and not flag.any()
        with torch.no_grad():
            assert torch.equal(f(t2, w2, flag), plain(t2, w2) + 1)
        f(torch.full_like(t2, V), w2, flag)
        assert flag.item() == 1
        flag.zero_()


def test_trace_refuses_what_the_call_refuses(dev):
    w, t = small(V, H, dev=dev), tokens(dev, 4)
    with pytest.raises(ValueError, match="padding_idx"):
        torch.jit.trace(lambda a, b: T.embed_tokens(a, b, 1.0, V), (t, w))


def test_the_module_may_be_loaded_again():
    import os
    import subprocess
    import sys
    code = "import importlib, diffsvc_amd; from diffsvc_amd import tokens; importlib.reload(tokens)"
    subprocess.run([sys.executable, "-c", code], check=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), timeout=300)


@pytest.mark.gpu
def test_other_calls_refuse_to_be_traced():
    from diffsvc_amd import muon
    x, t = small(V, H, dev="cuda"), tokens("cuda", V)
    for f, a in ((muon.orthogonalize, (x,)), (lambda t, d: T.embed_tokens_grad(t, d, V), (t, x))):
        with pytest.raises(RuntimeError, match="a trace would record"):
            torch.jit.trace(f, a)


@pytest.mark.gpu
def test_trace_of_the_module():
    m = T.TokenEmbeddingHip(V, H, padding_idx=PAD, scale=SCALE).cuda()
    with torch.no_grad():
        f = torch.jit.trace(m, (tokens("cuda", 6),))
    m.weight.data.copy_(small(V, H, dev="cuda"))
    t = tokens("cuda", 3, 2, seed=9)
    assert torch.equal(f(t), plain(t, m.weight)) and torch.equal(f(t), m(t))
    m.check()
    f(torch.tensor([V], device="cuda"))
    with pytest.raises(IndexError):
        m.check()


@pytest.mark.gpu
@pytest.mark.parametrize("trained", [False, True])
def test_forward_mode_of_the_module(trained):
    m, e = T.TokenEmbeddingHip(V, H, padding_idx=PAD).cuda(), torch.nn.Embedding(V, H, padding_idx=PAD).cuda()
    m.load_state_dict(e.state_dict())
    for x in (m, e):
        x.requires_grad_(trained)
    dw, t = small(V, H, seed=2, dev="cuda"), tokens("cuda", 7)
    with fw.dual_level():
        a, b = (torch.func.functional_call(x, {"weight": fw.make_dual(x.weight, dw)}, (t,)) for x in (m, e))
        assert torch.equal(fw.unpack_dual(a).tangent, fw.unpack_dual(b).tangent) and torch.equal(a, b)


@pytest.mark.gpu
def test_a_graph_notices_what_is_written_in_place():
    """A tensor that a graph has saved and one of the kernels has written since: backward refuses, as after torch's own in-place operations."""
    from diffsvc_amd import muon
    t, d = tokens("cuda", 6), small(6, H, dev="cuda")
    for write in (lambda x, m: muon.muon_step_(x, d[:4], m, 0.1), lambda x, m: muon.muon_step_(m.clone(), d[:4], x, 0.1), lambda x, m: muon.orthogonalize(d[:4], out=x),
                  lambda x, m: T.embed_tokens_grad(t % 4, d, 4, out=x), lambda x, m: muon.muon_step_(x[1:3], d[:2], m[1:3], 0.1)):
        x, m, y = torch.ones(4, H, device="cuda"), torch.zeros(4, H, device="cuda"), torch.ones(4, H, device="cuda", requires_grad=True)
        loss = (x * y).sum()
        write(x, m)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
