"""Token embedding on the HIP kernels: lookup with scaling and its gradient by sorted tokens (csrc/embed.hip) -- what the reference's embedding
tables do through ``nn.Embedding`` and its autograd (modules/fastspeech/fs2.py:73,81-82,240-247).

  * ``embed_tokens(tokens, weight, scale, padding_idx)``   y[i] = scale * weight[tokens[i]], differentiable in ``weight``
  * ``embed_tokens_grad(tokens, dy, vocab, ...)``          dW[v] (+)= scale * sum of dy over the places of token v
  * ``TokenEmbeddingHip``                                  the module: an ``nn.Embedding`` (same parameters, same state dict)

Tables and gradients are float32, float16 or bfloat16; tokens int32 or int64 of any shape.  Sums run in float32 in a fixed order: the gradient is
bit-identical from call to call.  A token outside [0, vocab) gives a zero row and no gradient; a sticky device flag records it
(``TokenEmbeddingHip.check()`` raises the IndexError that ``nn.Embedding`` would have raised)."""
import ctypes

import torch
from torch import nn
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import check, lib

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_tracing = torch._C._is_tracing


def launch(t, fn, *args):
    """fn(*args, stream) on t's device and that device's current stream; raises what the library reports."""
    i = t.device.index
    if i == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    if rc:
        check(rc)


def refuse_trace():
    if _tracing():
        raise RuntimeError("diffsvc_amd: a trace would record the memory of this call without the kernels that fill it")


def rows_of(t):
    """t with unit stride along its rows and rows that do not overlap (a copy where they do), for a 2-d tensor."""
    return t if t.is_contiguous() or (t.shape[1] <= 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1]) else t.contiguous()


def _check_tokens(tokens, other):
    if tokens.dtype is not torch.int64 and tokens.dtype is not torch.int32:
        raise TypeError("diffsvc_amd: tokens must be int32 or int64, got %s" % tokens.dtype)
    if not other.is_cuda or tokens.device != other.device:
        raise RuntimeError("diffsvc_amd: tokens (%s) and tensors (%s) must live on one HIP device; there is no CPU path" % (tokens.device, other.device))


def _padding(padding_idx, vocab):
    if padding_idx is None:
        return -1
    if not -vocab <= padding_idx < vocab:
        raise ValueError("padding_idx %d outside a table of %d rows" % (padding_idx, vocab))
    return padding_idx % vocab


def _lookup(tokens, weight, scale, flag):
    shape = weight.shape
    if len(shape) != 2 or not shape[0] or not shape[1]:
        raise ValueError("the table must be [rows, columns], got %s" % (tuple(shape),))
    V, H = shape
    dtype = DTYPES.get(weight.dtype)
    if dtype is None:
        raise TypeError("diffsvc_amd: tables are float32, float16 or bfloat16, got %s" % weight.dtype)
    _check_tokens(tokens, weight)
    w, t = rows_of(weight), tokens if tokens.is_contiguous() else tokens.contiguous()
    out = w.new_empty((*t.shape, H))
    launch(w, lib().dsvc_embed_tokens, t.data_ptr(), t.dtype is torch.int64, t.numel(), w.data_ptr(), w.stride(0), V, H, dtype, scale, out.data_ptr(), H,
           None if flag is None else flag.data_ptr())
    return out


def embed_tokens_grad(tokens, dy, vocab, scale=1.0, padding_idx=None, out=None, accumulate=False):
    """Gradient of ``embed_tokens`` in its table, [vocab, H]: dy is [..., H] over tokens of shape [...].  ``out`` (dy's type or float32) is
    written whole, zeros where a token does not occur; with ``accumulate`` the sums are added to what it holds instead.  It does not overlap dy.
    The result carries no autograd graph (``torch.autograd.grad`` of ``embed_tokens`` with ``create_graph`` gives one that does)."""
    refuse_trace()
    if dy.dtype not in DTYPES:
        raise TypeError("diffsvc_amd: gradients are float32, float16 or bfloat16, got %s" % dy.dtype)
    if dy.dim() < 1 or tuple(dy.shape[:-1]) != tuple(tokens.shape) or not dy.shape[-1]:
        raise ValueError("shape mismatch: tokens %s, gradient %s" % (tuple(tokens.shape), tuple(dy.shape)))
    if vocab < 1:
        raise ValueError("a table of %d rows" % vocab)
    _check_tokens(tokens, dy)
    H, n = dy.shape[-1], tokens.numel()
    pad = _padding(padding_idx, vocab)
    d = dy if dy.dim() == 2 else dy.reshape(n, H)
    d, t = rows_of(d), tokens if tokens.is_contiguous() else tokens.contiguous()
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs the tensor to add to (out)")
        out = torch.empty(vocab, H, device=d.device, dtype=d.dtype)
    elif tuple(out.shape) != (vocab, H) or out.device != d.device or out.dtype not in (d.dtype, torch.float32):
        raise ValueError("out must be [%d, %d] of %s or float32 on %s" % (vocab, H, d.dtype, d.device))
    elif (H > 1 and out.stride(1) != 1) or (vocab > 1 and out.stride(0) < H):
        raise ValueError("out needs rows of unit stride that do not overlap, got strides %s" % (out.stride(),))
    else:
        increment_version(out)             # (a graph that saved it must not use it unawares)
    L = lib()
    need = ctypes.c_int64(0)
    check(L.dsvc_embed_tokens_grad_workspace(n, vocab, H, ctypes.byref(need)))
    ws = torch.empty(need.value, device=d.device, dtype=torch.uint8)
    launch(d, L.dsvc_embed_tokens_grad, t.data_ptr(), t.dtype is torch.int64, n, d.data_ptr(), d.stride(0), DTYPES[d.dtype], vocab, H, scale, pad, out.data_ptr(),
           out.stride(0), DTYPES[out.dtype], accumulate, ws.data_ptr(), need.value)
    return out


# torch.func wants a function's forward and setup_context apart, at 15 us of host time a call: it has subclasses of its own (.func)
_func_active = torch._C._are_functorch_transforms_active


def _apply(f, *args):
    return (f.func if _func_active() else f).apply(*args)


def _each(f, info, in_dims, *args):
    """vmap by hand: f on every slice of the batched arguments."""
    return torch.stack([_apply(f, *(a if d is None else a.select(d, i) for a, d in zip(args, in_dims))) for i in range(info.batch_size)]), 0


class _EmbedTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding_idx, flag):
        ctx.save_for_backward(tokens)
        ctx.save_for_forward(tokens)
        ctx.args = weight.shape[0], scale, padding_idx
        return _lookup(tokens, weight, scale, flag)

    @staticmethod
    def backward(ctx, dy):
        args = (ctx.saved_tensors[0], dy, *ctx.args)
        if torch.is_grad_enabled() or forward_ad._current_level >= 0 or _func_active():      # (create_graph, or a dy with a tangent or a batch)
            return None, _apply(_EmbedTokensGrad, *args), None, None, None
        return None, embed_tokens_grad(*args), None, None, None

    @staticmethod
    def jvp(ctx, _, dw, *__):                      # linear in the table; its row padding_idx counts forwards, as in nn.Embedding
        return _apply(_EmbedTokens, ctx.saved_tensors[0], dw, ctx.args[1], ctx.args[2], None)


class _EmbedTokensFunc(_EmbedTokens):
    @staticmethod
    def forward(tokens, weight, scale, padding_idx, flag):
        return _lookup(tokens, weight, scale, flag)

    @staticmethod
    def setup_context(ctx, inputs, output):
        tokens, weight, scale, padding_idx, _ = inputs
        ctx.save_for_backward(tokens)
        ctx.save_for_forward(tokens)
        ctx.args = weight.shape[0], scale, padding_idx

    @staticmethod
    def vmap(info, in_dims, tokens, weight, *rest):
        if in_dims[1] is None:                     # one table: the batch is one more dimension of the tokens
            return _apply(_EmbedTokens, tokens.movedim(in_dims[0], 0), weight, *rest), 0
        return _each(_EmbedTokens, info, in_dims, tokens, weight, *rest)


_EmbedTokens.func = _EmbedTokensFunc


class _EmbedTokensGrad(torch.autograd.Function):
    """embed_tokens_grad as a linear map of dy: its own backward pass is the lookup without the places of padding_idx."""

    @staticmethod
    def forward(ctx, tokens, dy, *args):
        ctx.save_for_backward(tokens)
        ctx.save_for_forward(tokens)
        ctx.args = args
        return embed_tokens_grad(tokens, dy, *args)

    @staticmethod
    def backward(ctx, dw):
        (tokens,), (_, scale, padding_idx) = ctx.saved_tensors, ctx.args
        if padding_idx is not None:
            tokens = torch.where(tokens == padding_idx, -1, tokens)
        return None, embed_tokens(tokens, dw, scale), None, None, None

    @staticmethod
    def jvp(ctx, _, d_dy, *__):
        return _apply(_EmbedTokensGrad, ctx.saved_tensors[0], d_dy, *ctx.args)


class _EmbedTokensGradFunc(_EmbedTokensGrad):
    @staticmethod
    def forward(tokens, dy, vocab, scale, padding_idx):
        return embed_tokens_grad(tokens, dy, vocab, scale, padding_idx)

    @staticmethod
    def setup_context(ctx, inputs, output):
        tokens, _, *ctx.args = inputs
        ctx.save_for_backward(tokens)
        ctx.save_for_forward(tokens)

    @staticmethod
    def vmap(info, in_dims, *args):
        return _each(_EmbedTokensGrad, info, in_dims, *args)


_EmbedTokensGrad.func = _EmbedTokensGradFunc


def embed_tokens(tokens, weight, scale=1.0, padding_idx=None, flag=None):
    """scale * weight[tokens], [..., H] for tokens [...]; differentiable in ``weight`` (backwards and forwards), whose row ``padding_idx`` gets no gradient.
    flag: an int32 device tensor that is set to 1 where a token lies outside the table (its row is zero)."""
    scale = float(scale)
    if _tracing():                                                 # a trace sees no kernel launch: it records the operator
        return torch.ops.diffsvc_amd.embed_tokens(tokens, weight, scale, padding_idx, flag)
    if padding_idx is not None:
        padding_idx = _padding(padding_idx, weight.shape[0])
    if flag is not None and (flag.dtype != torch.int32 or flag.device != weight.device or flag.numel() < 1):
        raise ValueError("flag must be an int32 tensor on %s" % weight.device)
    # (a table that takes no gradient and has no tangent has no use for the graph)
    if weight.requires_grad and torch.is_grad_enabled() or forward_ad._current_level >= 0 or _func_active():
        return _apply(_EmbedTokens, tokens, weight, scale, padding_idx, flag)
    return _lookup(tokens, weight, scale, flag)


# embed_tokens as an operator of torch's own, for torch.jit.trace: its graph calls back here (whoever loads one imports this package)
if not hasattr(torch.ops.diffsvc_amd, "embed_tokens"):              # (a module that is loaded again finds it)
    _library = torch.library.Library("diffsvc_amd", "FRAGMENT")
    _library.define("embed_tokens(Tensor tokens, Tensor weight, float scale, int? padding_idx, Tensor(a!)? flag) -> Tensor")
    _library.impl("embed_tokens", embed_tokens, "CompositeImplicitAutograd")


class TokenEmbeddingHip(nn.Embedding):
    """``nn.Embedding`` whose device path runs on the HIP kernels, with an output scale.  Host tensors take ``nn.Embedding``'s own path."""

    def __init__(self, num_embeddings, embedding_dim, padding_idx=None, scale=1.0, **kw):
        for k in ("max_norm", "scale_grad_by_freq", "sparse"):
            if kw.get(k):
                raise NotImplementedError("TokenEmbeddingHip: %s" % k)
        super().__init__(num_embeddings, embedding_dim, padding_idx, **kw)
        self.scale = float(scale)
        # sticky flag: a token outside the table (check).  A buffer, so that it is there before a first call that is being captured into a graph
        self.register_buffer("_flag", torch.zeros(1, dtype=torch.int32), persistent=False)

    def forward(self, tokens):
        if not self.weight.is_cuda:
            y = super().forward(tokens)
            return y * self.scale if self.scale != 1.0 else y
        if self._flag.device != self.weight.device:        # (a weight that was moved by itself)
            self._flag = torch.zeros(1, device=self.weight.device, dtype=torch.int32)
        return embed_tokens(tokens, self.weight, self.scale, self.padding_idx, self._flag)

    def check(self):
        """Raise IndexError if a lookup on the device since the last check was given a token outside the table.  Synchronises."""
        if int(self._flag.item()):
            self._flag.zero_()
            raise IndexError("diffsvc_amd: a token lies outside [0, %d); its row was zero" % self.num_embeddings)
