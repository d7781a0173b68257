"""Functional operations on weights and other matrices held in 4-bit blocks (the reference has 8-bit values only).

Format: ``block`` consecutive values of a row have the scale ``s = max|x|``, held exactly in x's own type (bfloat16 or float16), and
every value the code ``rint(7 x / s)``, -7 to 7 (the quotient in exact arithmetic, ties to even), which stands for ``s * code / 7``.
Codes are uint8 ``[..., ceil(K/2)]``: two to a byte, offset by 8, the even one in the low half; a row of odd length ends in a code 0.
Scales ("state") are ``[..., ceil(K/block)]`` in x's type, row by row (not transposed as the int8 ones are).  An all-zero block has
scale 0; one that holds an infinity or a NaN has the scale NaN and reads as NaN throughout.

Blocks have 32, 64 or 128 values: ``block_linear_config.GROUP_SIZE`` read at call time unless ``fblock_size`` is given.  The functions
run on the current CUDA stream of their operands' device; they have no derivatives and refuse tensors that want a gradient (outside
``torch.no_grad()``) or bring a forward-mode tangent: biases, scales and rotary tables as much as activations.
"""
from __future__ import annotations

import torch

from . import _lib
from . import block_linear_config
from .triton_functions import _block

__all__ = ["quantize_block_int4", "dequantize_block_int4", "int4_matmul"]

_native = _lib.native


def quantize_block_int4(x: torch.Tensor, fblock_size=None):
    """``x [..., K]`` (bfloat16 or float16) in 4 bits: ``(codes, state)`` as described above, both dense."""
    return _native().quantize_int4(x, _block(fblock_size))


def dequantize_block_int4(codes: torch.Tensor, state: torch.Tensor, fblock_size=None, *, features: int = None, dtype: torch.dtype = None):
    """What ``codes`` stand for, ``[..., K]``: ``state * code / 7``, the quotient rounded to fp32 once, cast to ``dtype`` (default
    ``INPUT_OUTPUT_TORCH_TYPE``).  ``features`` is K where it is odd; by default every code counts."""
    return _native().dequantize_int4(codes, state, _block(fblock_size), -1 if features is None else features,
                                     dtype or block_linear_config.INPUT_OUTPUT_TORCH_TYPE)


def int4_matmul(x: torch.Tensor, codes: torch.Tensor, state: torch.Tensor, bias=None, *, residual=None, fblock_size=None, dtype: torch.dtype = None):
    """``x [..., K] @ W^T (+ bias) (+ residual)`` for weights ``[N, K]`` held in 4 bits (``quantize_block_int4(W)``, of x's type).

    The activations stay what they are: products with the codes are summed in fp32, times the block's scale, in a fixed order; bias ``[N]``
    and ``residual [..., N]`` (of the output's type) are added in fp32 and the result is rounded once, to ``dtype`` (default
    ``INPUT_OUTPUT_TORCH_TYPE``).  Made for the few rows of a decode step: up to 64 rows read the weights once (half of an int8
    layer's bytes), more are taken 64 at a time.  A row of x that holds an infinity or a NaN gives
    infinities and NaN."""
    return _native().matmul_int4(x, codes, state, bias, residual, _block(fblock_size), dtype or block_linear_config.INPUT_OUTPUT_TORCH_TYPE)
