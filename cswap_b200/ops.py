"""Operators of a training step that save little for backward.

What autograd keeps of a transformer's layers is mostly the scores of its attention (three tensors of tokens x tokens
a layer), the two tensors around the activation of its feed-forward part, and the inputs of its norms.  These
operators keep less to begin with, beside the codecs that shrink or move what is kept:

* ``q8_compress`` / ``q8_decompress``: a tensor as an 8-bit checkpoint on the device (a group of 128 consecutive values
  shares a float32 scale, 1.03 bytes a value).
* ``gelu`` keeps its input as such a checkpoint, written in the pass that computes the output; ``gelu_linear`` with the
  linear layer behind it keeps nothing else: backward forms the activation again for the weight's gradient.
* ``layer_norm``, optionally of a sum of two tensors, keeps what is normed and two numbers a row.
* ``attention`` keeps its output and one number a row besides its operands; backward forms the probabilities again.

``gelu``, ``gelu_linear``, ``layer_norm`` and ``attention`` are differentiable (once).  Below them lie the passes
themselves, ``*_forward`` and ``*_backward``, for programs that drive their own backward pass; they take contiguous
CUDA tensors (attention: any strides) and know nothing of autograd.  All run on torch's current stream of the tensors'
device, take float32, float16 or bfloat16 (attention: the last two), compute in float32 and round a result to its type
once.  The same call gives the same bits every time.  There is no CPU implementation.

A step that is captured into a CUDA graph must not share a leaf with a live graph of another stream (autograd would
hand that leaf's gradient over to the other stream inside the capture); a call on such a leaf, or on a view or a copy of
one, raises.  A leaf that lies further back (a weight of a projection, say) is the step's own to look after.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch
import torch.nn.functional as F
from torch.amp import custom_bwd, custom_fwd
from torch.autograd.function import once_differentiable

from . import codec
from ._lib import check, lib

Q8_GROUP = 128


def _ext():
    return codec._native or codec._load()


# ---------------------------------------------------------------------------
# 8-bit checkpoints
# ---------------------------------------------------------------------------

def q8_bytes(n: int) -> int:
    """Bytes of the checkpoint of n values: n codes, and from the next multiple of 16 on a float32 scale for each
    group of 128."""
    out = C.c_size_t()
    if n < 0:
        raise ValueError("n must not be negative")
    check(lib().csw_q8_bytes(n, C.byref(out)), "csw_q8_bytes")
    return out.value


def q8_compress(t: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The 8-bit checkpoint (uint8 tensor of q8_bytes(t.numel()) bytes) of `t`, whatever its shape.

    With m the largest magnitude of a group of 128 consecutive values, its scale is m / 127 and a value's code
    rint(x * (127 / m)); a value is off by at most m / 254 and a rounding.  A group below 2**-120 is held as zeros, a
    group with a NaN or an infinity as NaNs.  `out` (16-byte aligned, apart from `t`) may be longer than needed."""
    return _ext().q8_compress(t, out)


def q8_decompress(packed: torch.Tensor, numel: int, dtype: torch.dtype = torch.float32,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The `numel` values that a checkpoint holds, flat, or in `out` (whose type then counts, apart from `packed`)."""
    return _ext().q8_decompress(packed, numel, dtype, out)


# ---------------------------------------------------------------------------
# GELU on checkpoints
# ---------------------------------------------------------------------------

def gelu_forward(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(x Phi(x), the 8-bit checkpoint of x) in one pass; Phi is the normal distribution function."""
    return _ext().gelu_forward(x)


def gelu_backward(dy: torch.Tensor, packed: torch.Tensor, recompute: bool = False):
    """dy (Phi(x) + x phi(x)) for the values x that the checkpoint holds; with `recompute` also x Phi(x)."""
    return _ext().gelu_backward(dy, packed, recompute)


class _Gelu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        y, packed = gelu_forward(x)
        ctx.save_for_backward(packed)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        packed, = ctx.saved_tensors
        return gelu_backward(dy.contiguous(), packed)


class _GeluLinear(torch.autograd.Function):
    @staticmethod
    @custom_fwd(device_type="cuda")
    def forward(ctx, x, weight, bias):
        y, packed = gelu_forward(x)
        ctx.save_for_backward(packed, weight)
        return F.linear(y, weight, bias)

    @staticmethod
    @custom_bwd(device_type="cuda")
    @once_differentiable
    def backward(ctx, dy):
        packed, weight = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad
        dx = dw = db = None
        if want_x or want_w:
            dx = torch.matmul(dy, weight).contiguous()
            dx = gelu_backward(dx, packed, want_w)
            if want_w:
                dx, y = dx
                dw = torch.matmul(dy.flatten(0, -2).t(), y.flatten(0, -2))
        if want_b:
            db = dy.flatten(0, -2).sum(0)
        return dx, dw, db


def gelu(x: torch.Tensor) -> torch.Tensor:
    """x Phi(x).  Keeps x as an 8-bit checkpoint, on which the gradient is taken."""
    x = x.contiguous()
    _ext().check_capture(x)
    return _Gelu.apply(x)


def gelu_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """linear(gelu(x), weight, bias), of which an 8-bit checkpoint of x is all that is kept: backward forms gelu(x) on
    it for the weight's gradient.  The products themselves are torch's."""
    if x.dim() < 2:
        raise ValueError("x needs two axes at least")
    x = x.contiguous()
    _ext().check_capture(x, weight, bias)
    return _GeluLinear.apply(x, weight, bias)


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------

def layer_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                       eps: float = 1e-5, residual: Optional[torch.Tensor] = None):
    """(y, s, mean, rstd): s is x, or x + residual as rounded to its type, y its norm over the last axis, mean and
    rstd (float32, one of each a row) what backward needs besides s."""
    return _ext().layer_norm_forward(x, weight, bias, eps, residual)


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: Optional[torch.Tensor] = None, sums: bool = True):
    """(dx, dweight, dbias) from the s, mean and rstd of layer_norm_forward; dx is the gradient of both terms of a sum.
    The last two are None without a weight, or without `sums`."""
    return _ext().layer_norm_backward(dy, x, mean, rstd, weight, sums)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        y, s, mean, rstd = layer_norm_forward(x, weight, bias, eps, residual)
        ctx.save_for_backward(s, mean, rstd, weight)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        s, mean, rstd, weight = ctx.saved_tensors
        want_x, want_r, want_w, want_b, _ = ctx.needs_input_grad
        dx, dw, db = layer_norm_backward(dy.contiguous(), s, mean, rstd, weight, want_w or want_b)
        return dx if want_x else None, dx if want_r else None, dw if want_w else None, db if want_b else None, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Layer norm of x, or of x + residual (same shape and type), over the last axis.  weight and bias hold one value
    a column, in the type of x or in float32; a bias needs a weight."""
    x = x.contiguous()
    if residual is not None:
        residual = residual.contiguous()
    _ext().check_capture(x, residual, weight, bias)
    return _LayerNorm.apply(x, residual, weight, bias, eps)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = False,
                      kv_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None
                      ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(o, lse): o as of `attention`, lse (float32, [batch, heads, q_len]) the natural logarithm of each row's sum of
    exp(scale q.k)."""
    return _ext().attention_forward(q, k, v, causal, kv_lens, scale)


def attention_backward(do: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor,
                       lse: torch.Tensor, causal: bool = False, kv_lens: Optional[torch.Tensor] = None,
                       scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dk, dv) from the gradient of o and what attention_forward took and gave."""
    return _ext().attention_backward(do, q, k, v, causal, kv_lens, scale, o, lse)


def device_status(device=None) -> None:
    """Waits for the current stream of `device` (the current one unless given) and raises CswapError where a kernel there
    gave up on a wait for its own copies or products; it is told once.  The results of such a call are NaN, and the next
    call of an attention pass on the device raises the same, so that a program need not ask."""
    with torch.cuda.device(device):
        check(lib().csw_device_status(torch.cuda.current_stream().cuda_stream), "csw_device_status")


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, kv_lens, scale):
        o, lse = attention_forward(q, k, v, causal, kv_lens, scale)
        ctx.save_for_backward(q, k, v, o, lse, kv_lens)
        ctx.causal, ctx.scale = causal, scale
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, kv_lens = ctx.saved_tensors
        dq, dk, dv = attention_backward(do, q, k, v, o, lse, ctx.causal, kv_lens, ctx.scale)
        return dq, dk, dv, None, None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = False,
              kv_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """softmax(scale q k^T) v for each head, scale 1 / sqrt(dim) unless given.

    q is [batch, heads, q_len, dim], k and v are [batch, kv_heads, k_len, dim], float16 or bfloat16, dim a multiple of
    8 up to 128, heads a multiple of kv_heads (each key head serves heads / kv_heads consecutive query heads).  Any
    strides will do; tensors whose rows do not lie on 16-byte boundaries are copied first.  `causal`: query i sees the
    keys up to i + k_len - q_len.  `kv_lens` (int32, on the device, one for each batch entry): the number of keys of
    that entry, taken into 0 ... k_len; keys and values behind it are not used, whatever they hold (those that only
    `causal` hides count with a probability of zero, and must be finite).  A query that sees no key gives zeros, and no
    gradient passes through it, whatever it and its gradient hold."""
    _ext().check_capture(q, k, v)
    return _Attention.apply(q, k, v, causal, kv_lens, scale)
