"""Linear layers whose products take 8-bit floating-point operands.

* ``fp8_quantize`` / ``fp8_dequantize``: a matrix as e4m3 codes with a power of two for each block of 128 x 128 values.
* ``fp8_matmul``: the product of two such matrices, either one taken transposed, on the tensor cores.
* ``fp8_linear``: a linear layer on them, differentiable (once).  All three of its products run in 8 bits, and of its input
  it keeps what its forward product read: 1.00006 bytes a value.

A block's scale 2^E is the least power of two (2^-126 at least) for which its largest magnitude is at most 448 2^E; a value's
code is the e4m3 number nearest to x / 2^E, ties to even.  A value of at least 2^-14.8 of its block's largest is off by at most
a sixteenth of itself, a smaller one by 2^-19 of the block's largest or so.  A NaN or an infinity is held as NaN, and shows in
every result that it goes into; the scale goes by the others.

Everything runs on torch's current stream of the tensors' device, on float32, float16 and bfloat16 values, and rounds a result to
its type once.  Sums are float32 numbers, but the tensor cores cut off what an addend has below them where a float32 product of
torch's rounds it: over 4096 products a result is off by 7e-7 of its norm, there by 2e-7.  The same call gives the same bits every
time.  There is no CPU implementation.  Waits inside
the products are bounded as those of attention are (``device_status``).
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import codec

FP8_BLOCK = 128

Quantized = Tuple[torch.Tensor, torch.Tensor]


def _ext():
    return codec._native or codec._load()


def fp8_quantize(x: torch.Tensor, sums: bool = False):
    """(codes, scales) of x as a matrix of rows of its last axis; with `sums` also the float32 sum of each column.

    codes is float8_e4m3fn [rows, cols], whose rows begin on 16 bytes (they are padded to that in memory), scales
    float8_e8m0fnu [blocks of rows, blocks of columns].  A matrix may have any distance between its rows; other tensors are
    contiguous."""
    return _ext().fp8_quantize(x, sums)


def fp8_dequantize(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that codes and scales stand for, rounded to `dtype`."""
    return _ext().fp8_dequantize(codes, scales, dtype)


def fp8_matmul(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, transpose_a: bool = False,
               transpose_b: bool = False, bias: Optional[torch.Tensor] = None,
               dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a b + bias in `dtype`, a and b as fp8_quantize gives them, or transposed."""
    return _ext().fp8_matmul(a, a_scales, b, b_scales, transpose_a, transpose_b, bias, dtype)


def fp8_linear(x: torch.Tensor, weight: Union[torch.Tensor, Quantized], bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x weight^T + bias in the type of x, every product on operands in 8 bits.

    x is [..., in], weight [out, in], bias [out], each of its own type; their gradients have it, too.  x is kept as codes, and
    the weight's are for the input's gradient; both go through the program's saved-tensor hooks, which may give back tensors of
    the same type, shape and device that lie otherwise.  Execution's policies, which are for float32 tensors, leave them alone.
    A weight that does not change may be given as fp8_quantize(weight), and takes no gradient then (nor do x and the bias)."""
    if isinstance(weight, torch.Tensor):
        return _ext().fp8_linear(x, weight, bias)
    codes, scales = weight
    return _ext().fp8_linear_held(x, codes, scales, bias)
