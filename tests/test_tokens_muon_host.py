"""CPU: what the token-embedding and update-orthogonalising entry points refuse -- at the C ABI (argument checks run before any device call) and in
their Python wrappers -- and what the host path of the module computes."""
import ctypes

import pytest
import torch

import diffsvc_amd  # noqa: F401
from diffsvc_amd import _lib, muon, tokens

COEF = (3.4445, -4.7750, 2.0315)
P = ctypes.c_void_p(4096)                  # stands for any address: every call below is refused before it is used


def cfg(dtype=0, planes=0, batch=2, rows=8, cols=5, steps=5, coef=COEF, eps=1e-7, scale=1.0):
    return _lib.OrthoCfg(dtype, planes, batch, rows, cols, steps, (ctypes.c_float * 3)(*coef), eps, scale)


def refused(rc, text):
    msg = _lib.lib().dsvc_last_error().decode()
    assert rc == 1 and text in msg, (rc, msg)


@pytest.mark.parametrize("bad, text", [
    (dict(dtype=3), "type"), (dict(dtype=-1), "type"), (dict(planes=3), "planes"), (dict(batch=-1), "shape"), (dict(rows=-1), "shape"),
    (dict(rows=(1 << 20) + 1), "too large"), (dict(batch=65536), "too large"), (dict(steps=0), "steps"), (dict(steps=65), "steps"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(scale=float("inf")), "scale"),
    (dict(coef=(float("nan"), 0.0, 0.0)), "coefficient"), (dict(coef=(10.0, 10.0, 10.0)), "singular values"), (dict(coef=(3.0, 0.0, 0.0)), "singular values"),
])
def test_ortho_configurations_that_are_refused(bad, text):
    L, n = _lib.lib(), ctypes.c_int64(-1)
    c = cfg(**bad)
    refused(L.dsvc_ortho_workspace(ctypes.byref(c), ctypes.byref(n)), text)
    assert n.value == -1
    refused(L.dsvc_orthogonalize(ctypes.byref(c), P, 8, 64, P, 8, 64, P, 1 << 40, None), text)


def test_ortho_arguments_that_are_refused():
    L, n = _lib.lib(), ctypes.c_int64(-1)
    refused(L.dsvc_ortho_workspace(None, ctypes.byref(n)), "null")
    c = cfg()
    refused(L.dsvc_ortho_workspace(ctypes.byref(c), None), "null")
    assert L.dsvc_ortho_workspace(ctypes.byref(c), ctypes.byref(n)) == 0 and n.value > 0
    c1 = ctypes.byref(c)
    refused(L.dsvc_orthogonalize(c1, None, 5, 40, P, 5, 40, P, n.value, None), "null")
    refused(L.dsvc_orthogonalize(c1, P, 5, 40, None, 5, 40, P, n.value, None), "null")
    refused(L.dsvc_orthogonalize(c1, P, 5, 40, P, 5, 40, None, n.value, None), "null")
    refused(L.dsvc_orthogonalize(c1, P, 5, 40, P, 5, 40, P, n.value - 1, None), "workspace")
    refused(L.dsvc_orthogonalize(c1, P, 5, 40, P, 5, 40, ctypes.c_void_p(4096 + 16), n.value, None), "workspace")
    refused(L.dsvc_orthogonalize(c1, P, 4, 40, P, 5, 40, P, n.value, None), "row stride")
    refused(L.dsvc_orthogonalize(c1, P, 5, -1, P, 5, 40, P, n.value, None), "negative")
    refused(L.dsvc_orthogonalize(c1, P, 5, 40, P, 5, 39, P, n.value, None), "overlap")
    step = lambda p=P, g=P, m=P, ms=40, lr=0.1, mu=0.9, wd=0.0: L.dsvc_muon_step(c1, p, 5, 40, g, 5, 40, m, 5, ms, lr, mu, 1, wd, None, 1.0, P, n.value, None)
    for bad in (dict(p=None), dict(g=None), dict(m=None)):
        refused(step(**bad), "null")
    refused(step(ms=39), "overlap")
    for bad in (dict(mu=1.0), dict(mu=-0.1), dict(mu=float("nan")), dict(lr=float("nan")), dict(wd=float("inf"))):
        refused(step(**bad), "muon_step")
    # nothing to do: no pointer is looked at
    for shape in (dict(batch=0), dict(rows=0), dict(cols=0)):
        e = cfg(**shape)
        assert L.dsvc_ortho_workspace(ctypes.byref(e), ctypes.byref(n)) == 0 and n.value == 0
        assert L.dsvc_orthogonalize(ctypes.byref(e), None, 0, 0, None, 0, 0, None, 0, None) == 0


def test_ortho_accepts_the_usual_coefficients():
    n = ctypes.c_int64(0)
    for coef in (COEF, (1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (2.0, -1.5, 0.5)):
        c = cfg(coef=coef, steps=12)
        assert _lib.lib().dsvc_ortho_workspace(ctypes.byref(c), ctypes.byref(n)) == 0, (coef, _lib.lib().dsvc_last_error())


def test_embed_arguments_that_are_refused():
    L = _lib.lib()
    fwd = lambda t=P, n=3, w=P, wl=8, V=10, H=8, dt=0, s=1.0, o=P, ol=8: L.dsvc_embed_tokens(t, 1, n, w, wl, V, H, dt, s, o, ol, None, None)
    for bad in (dict(dt=3), dict(dt=-1)):
        refused(fwd(**bad), "type")
    for bad in (dict(n=-1), dict(V=0), dict(H=0), dict(H=(1 << 20) + 1)):
        refused(fwd(**bad), "table")
    for bad in (dict(wl=7), dict(ol=7), dict(wl=-8)):
        refused(fwd(**bad), "stride")
    refused(fwd(s=float("nan")), "scale")
    for bad in (dict(t=None), dict(w=None), dict(o=None)):
        refused(fwd(**bad), "null")
    assert fwd(n=0, t=None, w=None, o=None) == 0
    n = ctypes.c_int64(0)
    assert L.dsvc_embed_tokens_grad_workspace(100, 10, 8, ctypes.byref(n)) == 0 and n.value > 0
    bwd = lambda t=P, N=100, d=P, dl=8, dt=0, V=10, H=8, s=1.0, o=P, ol=8, ot=0, ws=P, wb=n.value: L.dsvc_embed_tokens_grad(
        t, 0, N, d, dl, dt, V, H, s, -1, o, ol, ot, 0, ws, wb, None)
    for bad, text in ((dict(N=-1), "tokens"), (dict(N=(1 << 28) + 1), "tokens"), (dict(V=0), "rows"), (dict(V=(1 << 30) + 1), "rows"), (dict(H=0), "columns"),
                      (dict(dt=3), "types"), (dict(dt=0, ot=1), "types"), (dict(dt=1, ot=2), "types"), (dict(dl=7), "strides"), (dict(ol=7), "strides"),
                      (dict(s=float("inf")), "scale"), (dict(t=None), "null"), (dict(d=None), "null"), (dict(o=None), "null"), (dict(ws=None), "null"),
                      (dict(wb=n.value - 1), "workspace"), (dict(ws=ctypes.c_void_p(4096 + 128)), "workspace")):
        refused(bwd(**bad), text)
    refused(L.dsvc_embed_tokens_grad_workspace(100, 10, 8, None), "null")


def test_wrappers_refuse_host_tensors_and_wrong_types():
    w, t = torch.zeros(4, 3), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        tokens.embed_tokens(t, w)
    with pytest.raises(TypeError, match="int32 or int64"):
        tokens.embed_tokens(t.float(), w)
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        tokens.embed_tokens(t, w.double())
    with pytest.raises(ValueError, match="rows, columns"):
        tokens.embed_tokens(t, w[0])
    with pytest.raises(ValueError, match="padding_idx"):
        tokens.embed_tokens(t, w, padding_idx=4)
    with pytest.raises(ValueError, match="flag"):
        tokens.embed_tokens(t, w, flag=torch.zeros(1))
    with pytest.raises(RuntimeError, match="no CPU path"):
        tokens.embed_tokens_grad(t, torch.zeros(2, 3), 4)
    with pytest.raises(ValueError, match="shape mismatch"):
        tokens.embed_tokens_grad(t, torch.zeros(3, 3), 4)
    with pytest.raises(TypeError, match="gradients"):
        tokens.embed_tokens_grad(t, torch.zeros(2, 3, dtype=torch.float64), 4)
    with pytest.raises(ValueError, match="0 rows"):
        tokens.embed_tokens_grad(t, torch.zeros(2, 3), 0)
    for f in (muon.orthogonalize, lambda x: muon.muon_step_(x, x, x, 0.1)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            f(torch.zeros(3, 3))
        with pytest.raises(ValueError, match="matrix"):
            f(torch.zeros(3))
        with pytest.raises(TypeError, match="must be float32"):
            f(torch.zeros(3, 3, dtype=torch.float64))


def test_in_place_tensors_must_not_overlap():
    for bad in (torch.zeros(3).expand(4, 3), torch.zeros(4, 4).t()[:, :3], torch.zeros(4, 3).expand(2, 4, 3)):
        with pytest.raises(ValueError, match="in place"):
            muon._matrices("out", bad, False)
        assert muon._matrices("x", bad, True).is_contiguous()
    ok = torch.zeros(5, 4, 6)[1:, :, 1:4]
    assert muon._matrices("out", ok, False).data_ptr() == ok.data_ptr()
    with pytest.raises(ValueError, match="three coefficients"):
        muon._cfg(torch.zeros(1, 2, 2), 5, COEF[:2], 1e-7, 1.0, None)
    with pytest.raises(ValueError, match="precision"):
        muon._cfg(torch.zeros(1, 2, 2), 5, COEF, 1e-7, 1.0, "bf16")


def test_module_on_the_host_is_the_plain_embedding():
    torch.manual_seed(3)
    m = tokens.TokenEmbeddingHip(7, 5, padding_idx=0, scale=3.0)
    assert list(m.state_dict()) == ["weight"] and not m.weight[0].any()
    t = torch.tensor([[1, 0, 6], [2, 2, 1]])
    y = m(t)
    assert torch.equal(y, torch.nn.functional.embedding(t, m.weight) * 3.0)
    y.sum().backward()
    assert not m.weight.grad[0].any() and torch.equal(m.weight.grad[2], torch.full((5,), 6.0))
    with pytest.raises(NotImplementedError):
        tokens.TokenEmbeddingHip(7, 5, sparse=True)
    assert muon.rms_scale(4, 25) == pytest.approx(1.0)


def test_embedding_gradients_are_refused_before_anything_runs():
    """The workspace query and the call refuse the same sizes: none gets past the query and fails after its first launches."""
    L, n = _lib.lib(), ctypes.c_int64(-1)
    for N, V, H in ((1 << 28, 10, 1 << 20), (1 << 25, 10, 1 << 20), (1 << 28, 1 << 30, 1 << 17)):
        refused(L.dsvc_embed_tokens_grad_workspace(N, V, H, ctypes.byref(n)), "too many")
        assert n.value == -1
        for dt in (0, 1, 2):
            refused(L.dsvc_embed_tokens_grad(P, 0, N, P, H, dt, V, H, 1.0, -1, P, H, dt, 0, P, 1 << 60, None), "too many")
    for N, V, H in ((0, 1 << 30, 1), (1 << 28, 1 << 30, 1), (5, 1 << 30, 1 << 20), (1 << 24, 7, 1 << 20)):
        assert L.dsvc_embed_tokens_grad_workspace(N, V, H, ctypes.byref(n)) == 0, (N, V, H)


def test_coefficients_are_read_at_every_call():
    """One-element tensors are numbers too, and may have changed since the last call."""
    a, x = torch.tensor(1.5), torch.zeros(1, 2, 2)
    coef = (a, -0.5, 0.0)
    assert muon._cfg(x, 5, coef, 1e-7, 1.0, None).coef[0] == 1.5
    a.fill_(1.25)
    assert list(muon._cfg(x, 5, coef, 1e-7, 1.0, None).coef) == [1.25, -0.5, 0.0]
