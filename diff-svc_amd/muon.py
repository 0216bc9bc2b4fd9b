"""Orthogonalised updates of matrix parameters (csrc/ortho.hip): the Newton-Schulz iteration and the optimisation step built on it.

  X = G / (||G||_F + eps);  steps times:  A = X X^T,  X <- (a I + b A + c A A) X;  O = scale * X

takes every singular value s of the normalised update through s (a + b s^2 + c s^4): with the default coefficients all of them end between about
0.7 and 1.2, so O is close to U V^T of G = U S V^T.  (Coefficients under which the iterate shrinks lose the bits that it shrinks by.)  ``muon_step_`` orthogonalises the (Nesterov) momentum of a gradient and takes the weight step.

Types: float32, float16 and bfloat16 tensors run on split fp16 operands (``precision="f16_x3"``, the default: fp32-class, three matrix-core products
per product).  ``"f16"`` asks for single fp16 operands: up to three times as fast, but a rounding of an early iterate grows by up to a^steps where the
update has next to nothing -- 2e-3 of the result for an update of full rank, 4e-2 at rank 16, 1e-1 at rank 1.
Accumulation, norms and momentum are float32 or wider."""
import ctypes
import math

import torch
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import check, lib
from .tokens import DTYPES, launch, refuse_trace

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
PLANES = {None: 0, "f16": 1, "f16_x3": 2}


def rms_scale(rows, cols, rms=0.2):
    """The scale at which an orthogonalised [rows, cols] update has elements of root mean square ``rms``: 0.2 is about an AdamW step's, so that one
    learning rate serves both."""
    return rms * math.sqrt(max(rows, cols))


_Coefficients = ctypes.c_float * 3


def _cfg(t, steps, coefficients, eps, scale, precision):
    planes = PLANES.get(precision, -1)
    if planes < 0:
        raise ValueError("precision must be one of %s, got %r" % ([k for k in PLANES if k], precision))
    if len(coefficients) != 3:
        raise ValueError("three coefficients, got %r" % (coefficients,))
    B, m, n = t.shape
    return _lib.OrthoCfg(DTYPES[t.dtype], planes, B, m, n, steps, _Coefficients(*coefficients), eps, scale)


def _check(name, t):
    if t.dtype not in DTYPES:
        raise TypeError("diffsvc_amd: %s must be float32, float16 or bfloat16, got %s" % (name, t.dtype))
    if t.dim() < 2:
        raise ValueError("%s must be a matrix or a batch of matrices, got shape %s" % (name, tuple(t.shape)))
    if not t.is_cuda:
        raise RuntimeError("diffsvc_amd: %s must live on the HIP device; there is no CPU path" % name)


def _matrices(name, t, copy):
    """t as [batch, rows, columns] with unit stride along the rows; ``copy``: in a new tensor where it does not lie so, else refused."""
    m, n = t.shape[-2:]
    d = t.dim()
    v = t if d == 3 else t.unsqueeze(0) if d == 2 else t.reshape(math.prod(t.shape[:-2]), m, n) if copy else t.view(math.prod(t.shape[:-2]), m, n)
    bs, ld, one = v.stride()
    if (n <= 1 or one == 1) and (m <= 1 or ld >= n) and (v.shape[0] <= 1 or bs >= (m - 1) * ld + n):
        return v
    if copy:
        return v.contiguous()
    raise ValueError("%s is written in place: it needs rows of unit stride and matrices that do not overlap, got strides %s" % (name, t.stride()))


def _workspace(L, cfg, t):
    need = ctypes.c_int64(0)
    check(L.dsvc_ortho_workspace(ctypes.byref(cfg), ctypes.byref(need)))
    return torch.empty(need.value, device=t.device, dtype=torch.uint8), need.value


@torch.no_grad()
def orthogonalize(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7, scale=1.0, precision=None, out=None):
    """scale * the Newton-Schulz iterate of every matrix of x [..., rows, cols], in x's type.  ``out`` may be x itself.  The result carries no autograd
    graph: an update is made of gradients, it is not differentiated."""
    refuse_trace()
    _check("x", x)
    v = _matrices("x", x, True)
    if out is None:
        out = x.new_empty(x.shape)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError("out must be %s %s on %s" % (tuple(x.shape), x.dtype, x.device))
    o = _matrices("out", out, False)
    if out.untyped_storage().data_ptr() == v.untyped_storage().data_ptr() and (out.data_ptr() != v.data_ptr() or o.stride() != v.stride()):
        v = v.clone()                  # shares memory, but not matrix by matrix: one may be written before another is read
    cfg = _cfg(v, steps, coefficients, eps, scale, precision)
    L = lib()
    ws, size = _workspace(L, cfg, v)
    launch(v, L.dsvc_orthogonalize, ctypes.byref(cfg), v.data_ptr(), v.stride(1), v.stride(0), o.data_ptr(), o.stride(1), o.stride(0), ws.data_ptr(), size)
    increment_version(out)             # (a graph that saved it must not use it unawares)
    return out


@torch.no_grad()
def muon_step_(param, grad, momentum_buffer, lr, momentum=0.95, nesterov=True, weight_decay=0.0, scale=1.0, steps=5, coefficients=COEFFICIENTS, eps=1e-7,
               precision=None, grad_scale=None):
    """One step of every matrix of param [..., rows, cols], in place:

      g = grad * grad_scale;  m <- momentum m + (1 - momentum) g;  u = nesterov ? momentum m + (1 - momentum) g : m
      param <- (1 - lr weight_decay) param - lr * scale * orthogonalize(u)

    momentum_buffer is float32; grad has param's type; the three do not overlap.  grad_scale: a number or a one-element float32 device tensor (a
    clip coefficient)."""
    refuse_trace()
    _check("param", param)
    if grad.shape != param.shape or grad.dtype != param.dtype or grad.device != param.device:
        raise ValueError("grad must be %s %s on %s" % (tuple(param.shape), param.dtype, param.device))
    if momentum_buffer.shape != param.shape or momentum_buffer.dtype != torch.float32 or momentum_buffer.device != param.device:
        raise ValueError("momentum_buffer must be %s float32 on %s" % (tuple(param.shape), param.device))
    dev_scale, num_scale = None, 1.0
    if torch.is_tensor(grad_scale):
        if grad_scale.dtype != torch.float32 or grad_scale.numel() != 1 or grad_scale.device != param.device:
            raise ValueError("grad_scale must be a number or one float32 on %s" % param.device)
        dev_scale = grad_scale.data_ptr()
    elif grad_scale is not None:
        num_scale = float(grad_scale)
    p, g, m = _matrices("param", param, False), _matrices("grad", grad, True), _matrices("momentum_buffer", momentum_buffer, False)
    cfg = _cfg(p, steps, coefficients, eps, scale, precision)
    L = lib()
    ws, size = _workspace(L, cfg, p)
    launch(p, L.dsvc_muon_step, ctypes.byref(cfg), p.data_ptr(), p.stride(1), p.stride(0), g.data_ptr(), g.stride(1), g.stride(0), m.data_ptr(), m.stride(1),
           m.stride(0), lr, momentum, nesterov, weight_decay, dev_scale, num_scale, ws.data_ptr(), size)
    increment_version((param, momentum_buffer))
    return param
