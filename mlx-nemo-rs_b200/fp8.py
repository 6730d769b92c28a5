"""8-bit floating-point linears, their gradients and the LayerNorm's forward
and backward pass on torch CUDA tensors (nrp_fp8_*, nrp_layer_norm*).

A pre-norm linear's training step, with its activations kept in 8 bits:

    h, mean, rstd = layer_norm(x, gamma, beta)
    hq = fp8_quantize(h)                       # the product's operand and
    y = fp8_linear(hq, wq, bias)               # the checkpoint of h
    xq = fp8_quantize(x)                       # x and h may go
    ...
    dh = fp8_linear_input_grad(dy, wq)
    dw, db = fp8_linear_weight_grad(dy, hq, bias=True)
    dx, dgamma, dbeta = layer_norm_backward(dh, xq, mean, rstd, gamma)

Tensors are contiguous and on one device; the work is queued on that device's
current torch stream, and autograd does not record it: the gradients are the
calls above.  The checks, the outputs' allocation and the calls are
native (torch_binding.cpp); what they refuse raises NrpError.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import NRP_ERR_UNSUPPORTED, Context, NrpError, lib

lib()  # (names the build command if the library is missing)
try:
    from . import _nrp_torch as _native  # noqa: E402
except ImportError as e:
    raise NrpError(NRP_ERR_UNSUPPORTED,
                   "the torch binding is missing or was built for another torch or Python: run "
                   f"python mlx-nemo-rs_b200/build.py ({e})") from e


class Fp8Tensor(NamedTuple):
    """Block-scaled e4m3 matrix: codes torch.float8_e4m3fn [..., cols] and
    scales float32 [ceil(rows / block_rows), ceil(cols / 128)], rows the
    product of the leading dimensions; block_rows 1 (activations) or 128
    (weights)."""
    codes: object
    scales: object
    block_rows: int


_native.setup(NrpError, Fp8Tensor, Context.default)


def fp8_quantize(x, block_rows: int = 1, ctx: Optional[Context] = None,
                 out: Optional[Fp8Tensor] = None) -> Fp8Tensor:
    """e4m3 codes of x (f32 or bf16 [..., cols], cols % 16 == 0) with one
    power-of-two scale per block_rows x 128 block: the smallest with which
    the block's largest value is at most 448.  block_rows 1 for activations
    and gradients, 128 for weights.  NaN and infinities become NaN."""
    return _native.quantize(x, block_rows, ctx, out)


def fp8_dequantize(q: Fp8Tensor, dtype=torch.bfloat16, ctx: Optional[Context] = None, out=None):
    """The values q stands for, in bf16 (default) or f32."""
    return _native.dequantize(q, dtype, ctx, out)


def fp8_linear(x, w: Fp8Tensor, bias=None, dtype=None, ctx: Optional[Context] = None, out=None,
               codes: Optional[Fp8Tensor] = None):
    """y = x . w^T (+ bias) of 8-bit operands, f32 sums.  w [N, K] with 128 x
    128 blocks.  x: an Fp8Tensor [..., K] (y in `dtype`, default bf16), or an
    f32 or bf16 tensor, quantised in the call -- into `codes` when given, the
    checkpoint that fp8_linear_weight_grad takes -- and y in its type.  bias
    [N] in y's type."""
    return _native.product(x, w, bias, dtype, ctx, out, codes, False)


def fp8_linear_input_grad(dy, w: Fp8Tensor, dtype=None, ctx: Optional[Context] = None, out=None,
                          codes: Optional[Fp8Tensor] = None):
    """dx = dy . w, the gradient of fp8_linear's input; dy [..., N] as
    fp8_linear's x."""
    return _native.product(dy, w, None, dtype, ctx, out, codes, True)


def fp8_linear_weight_grad(dy, x: Fp8Tensor, bias: bool = False, dtype=torch.float32,
                           ctx: Optional[Context] = None, out=None, bias_out=None):
    """(dw [N, K], dbias [N] or None) from dy (bf16 [..., N], N % 8 == 0) and
    the 8-bit checkpoint x [..., K] of the linear's input; dw and dbias in
    `dtype` (default f32)."""
    return _native.weight_grad(dy, x, bias, dtype, ctx, out, bias_out)


def layer_norm(x, gamma, beta, eps: float = 1e-5, ctx: Optional[Context] = None, out=None):
    """(y, mean, rstd): LayerNorm over the last dimension of x (f32 or bf16);
    gamma, beta f32 [cols]; mean, rstd f32 [rows].  out may be x."""
    return _native.layer_norm(x, gamma, beta, eps, ctx, out)


def layer_norm_backward(dy, x, mean, rstd, gamma, ctx: Optional[Context] = None, out=None):
    """(dx, dgamma, dbeta) of layer_norm: dx in dy's type, dgamma and dbeta
    f32.  x: the exact input (dy's type) or its 8-bit checkpoint, an
    Fp8Tensor with block_rows 1; mean, rstd as layer_norm returned them."""
    return _native.layer_norm_backward(dy, x, mean, rstd, gamma, ctx, out)
