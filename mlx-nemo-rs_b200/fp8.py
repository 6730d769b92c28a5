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
current torch stream.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

from . import BF16, F32, NRP_ERR_INVALID, NRP_ERR_UNSUPPORTED, Context, NrpError, _check, lib


class Fp8Tensor(NamedTuple):
    """Block-scaled e4m3 matrix: codes torch.float8_e4m3fn [..., cols] and
    scales float32 [ceil(rows / block_rows), ceil(cols / 128)], rows the
    product of the leading dimensions; block_rows 1 (activations) or 128
    (weights)."""
    codes: object
    scales: object
    block_rows: int


def _fail(msg: str):
    raise NrpError(NRP_ERR_INVALID, msg)


def _tensor(name: str, t, dtypes, device=None):
    if not t.is_cuda:
        _fail(f"{name}: a CUDA tensor is needed")
    if device is not None and t.device != device:
        _fail(f"{name}: on {t.device}, the others on {device}")
    if t.dtype not in dtypes:
        raise NrpError(NRP_ERR_UNSUPPORTED, f"{name}: dtype {t.dtype}")
    if not t.is_contiguous():
        _fail(f"{name}: must be contiguous")
    return t


def _matrix(name: str, t, dtypes, device=None):
    _tensor(name, t, dtypes, device)
    if t.dim() < 1 or t.shape[-1] == 0:
        _fail(f"{name}: shape {tuple(t.shape)}")
    cols = t.shape[-1]
    return t.numel() // cols, cols


def _vector(name: str, t, n: int, dtype, device):
    _tensor(name, t, (dtype,), device)
    if t.numel() != n:
        _fail(f"{name}: {t.numel()} values, {n} needed")
    return t.data_ptr()


def _blocks(n: int) -> int:
    return (n + 127) // 128


def _codes(name: str, q: Fp8Tensor, block_rows: int, device=None):
    """(rows, cols) of a valid Fp8Tensor."""
    import torch
    if not isinstance(q, Fp8Tensor):
        _fail(f"{name}: an Fp8Tensor is needed")
    rows, cols = _matrix(name, q.codes, (torch.float8_e4m3fn,), device)
    if q.block_rows != block_rows:
        _fail(f"{name}: block_rows {q.block_rows}, {block_rows} needed")
    _tensor(name + " scales", q.scales, (torch.float32,), q.codes.device)
    if q.scales.numel() != (rows if block_rows == 1 else _blocks(rows)) * _blocks(cols):
        _fail(f"{name}: scales {tuple(q.scales.shape)} for {rows} x {cols} codes")
    return rows, cols


def _float_types():
    import torch
    return (torch.bfloat16, torch.float32)


def _dt(dtype) -> int:
    import torch
    return BF16 if dtype == torch.bfloat16 else F32


def _out(name: str, out, shape, dtype, device):
    import torch
    if dtype not in _float_types():
        raise NrpError(NRP_ERR_UNSUPPORTED, f"{name}: dtype {dtype}")
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    _tensor(name, out, (dtype,), device)
    if tuple(out.shape) != tuple(shape):
        _fail(f"{name}: shape {tuple(out.shape)}, {tuple(shape)} needed")
    return out


def _call(fn: str, device, ctx: Optional[Context], *args):
    """fn(context, the device's current stream, *args), with the thread's
    current device left as it was (the library makes the context's current)."""
    import torch
    if ctx is None:
        ctx = Context.default(device.index)
    elif ctx.device != device.index:
        _fail(f"context of device {ctx.device}, tensors on {device}")
    current = torch.cuda.current_device()
    try:
        _check(getattr(lib(), fn)(ctx.handle, torch.cuda.current_stream(device).cuda_stream, *args))
    finally:
        if current != device.index:
            torch.cuda.set_device(current)


def _new_codes(shape, rows: int, cols: int, block_rows: int, device) -> Fp8Tensor:
    import torch
    return Fp8Tensor(
        torch.empty(shape, dtype=torch.float8_e4m3fn, device=device),
        torch.empty((rows if block_rows == 1 else _blocks(rows), _blocks(cols)),
                    dtype=torch.float32, device=device), block_rows)


def fp8_quantize(x, block_rows: int = 1, ctx: Optional[Context] = None,
                 out: Optional[Fp8Tensor] = None) -> Fp8Tensor:
    """e4m3 codes of x (f32 or bf16 [..., cols], cols % 16 == 0) with one
    power-of-two scale per block_rows x 128 block: the smallest with which
    the block's largest value is at most 448.  block_rows 1 for activations
    and gradients, 128 for weights.  NaN and infinities become NaN."""
    rows, cols = _matrix("quantize", x, _float_types())
    if out is None:
        if block_rows not in (1, 128):
            raise NrpError(NRP_ERR_UNSUPPORTED, f"block_rows {block_rows} (supported: 1, 128)")
        out = _new_codes(x.shape, rows, cols, block_rows, x.device)
    elif _codes("quantize out", out, block_rows, x.device) != (rows, cols):
        _fail(f"quantize out: codes {tuple(out.codes.shape)} for {tuple(x.shape)}")
    _call("nrp_fp8_quantize", x.device, ctx, _dt(x.dtype), x.data_ptr(), rows, cols, block_rows,
          out.codes.data_ptr(), out.scales.data_ptr())
    return out


def fp8_dequantize(q: Fp8Tensor, dtype=None, ctx: Optional[Context] = None, out=None):
    """The values q stands for, in bf16 (default) or f32."""
    import torch
    rows, cols = _codes("dequantize", q, q.block_rows)
    out = _out("dequantize out", out, q.codes.shape, dtype or torch.bfloat16, q.codes.device)
    _call("nrp_fp8_dequantize", q.codes.device, ctx, q.codes.data_ptr(), q.scales.data_ptr(), rows,
          cols, q.block_rows, _dt(out.dtype), out.data_ptr())
    return out


def _product(fn: str, name: str, x, w: Fp8Tensor, trans: bool, bias, dtype, ctx, out, codes):
    import torch
    n, k = _codes(name + " weight", w, 128)
    red, cols = (n, k) if trans else (k, n)
    device = w.codes.device
    if isinstance(x, Fp8Tensor):
        if codes is not None:
            _fail(f"{name}: codes= takes the codes of a tensor that the call quantises")
        m, r = _codes(name + " input", x, 1, device)
        shape, src, q = x.codes.shape, None, x
        dtype = dtype or torch.bfloat16
    else:
        m, r = _matrix(name + " input", x, _float_types(), device)
        if dtype is not None and dtype != x.dtype:
            raise NrpError(NRP_ERR_UNSUPPORTED, f"{name}: input {x.dtype}, output {dtype}")
        shape, src, dtype = x.shape, x.data_ptr(), x.dtype
        if codes is None:
            q = _new_codes(shape, m, r, 1, device)
        else:
            q = codes
            if _codes(name + " codes", q, 1, device) != (m, r):
                _fail(f"{name}: codes {tuple(q.codes.shape)} for {tuple(shape)}")
    if r != red:
        _fail(f"{name}: input {tuple(shape)}, weight {tuple(w.codes.shape)}")
    out = _out(name + " out", out, (*shape[:-1], cols), dtype, device)
    args = [_dt(dtype), src, q.codes.data_ptr(), q.scales.data_ptr(), m, red, w.codes.data_ptr(),
            w.scales.data_ptr(), cols]
    if not trans:
        args.append(None if bias is None else _vector(name + " bias", bias, cols, dtype, device))
    _call(fn, device, ctx, *args, out.data_ptr())
    return out


def fp8_linear(x, w: Fp8Tensor, bias=None, dtype=None, ctx: Optional[Context] = None, out=None,
               codes: Optional[Fp8Tensor] = None):
    """y = x . w^T (+ bias) of 8-bit operands, f32 sums.  w [N, K] with 128 x
    128 blocks.  x: an Fp8Tensor [..., K] (y in `dtype`, default bf16), or an
    f32 or bf16 tensor, quantised in the call -- into `codes` when given, the
    checkpoint that fp8_linear_weight_grad takes -- and y in its type.  bias
    [N] in y's type."""
    return _product("nrp_fp8_linear", "fp8_linear", x, w, False, bias, dtype, ctx, out, codes)


def fp8_linear_input_grad(dy, w: Fp8Tensor, dtype=None, ctx: Optional[Context] = None, out=None,
                          codes: Optional[Fp8Tensor] = None):
    """dx = dy . w, the gradient of fp8_linear's input; dy [..., N] as
    fp8_linear's x."""
    return _product("nrp_fp8_linear_input_grad", "fp8_linear_input_grad", dy, w, True, None, dtype,
                    ctx, out, codes)


def fp8_linear_weight_grad(dy, x: Fp8Tensor, bias: bool = False, dtype=None,
                           ctx: Optional[Context] = None, out=None, bias_out=None):
    """(dw [N, K], dbias [N] or None) from dy (bf16 [..., N], N % 8 == 0) and
    the 8-bit checkpoint x [..., K] of the linear's input; dw and dbias in
    `dtype` (default f32)."""
    import torch
    m, n = _matrix("fp8_linear_weight_grad dy", dy, (torch.bfloat16,))
    mx, k = _codes("fp8_linear_weight_grad input", x, 1, dy.device)
    if m != mx:
        _fail(f"fp8_linear_weight_grad: {m} rows of dy, {mx} of x")
    dtype = dtype or torch.float32
    dw = _out("fp8_linear_weight_grad out", out, (n, k), dtype, dy.device)
    db = None
    if bias or bias_out is not None:
        db = _out("fp8_linear_weight_grad bias_out", bias_out, (n,), dtype, dy.device)
    _call("nrp_fp8_linear_weight_grad", dy.device, ctx, dy.data_ptr(), x.codes.data_ptr(),
          x.scales.data_ptr(), m, n, k, _dt(dtype), dw.data_ptr(),
          None if db is None else db.data_ptr())
    return dw, db


def layer_norm(x, gamma, beta, eps: float = 1e-5, ctx: Optional[Context] = None, out=None):
    """(y, mean, rstd): LayerNorm over the last dimension of x (f32 or bf16);
    gamma, beta f32 [cols]; mean, rstd f32 [rows].  out may be x."""
    import torch
    rows, cols = _matrix("layer_norm", x, _float_types())
    g = _vector("layer_norm gamma", gamma, cols, torch.float32, x.device)
    b = _vector("layer_norm beta", beta, cols, torch.float32, x.device)
    y = _out("layer_norm out", out, x.shape, x.dtype, x.device)
    stats = torch.empty((2, *x.shape[:-1]), dtype=torch.float32, device=x.device)
    mean, rstd = stats[0], stats[1]
    _call("nrp_layer_norm", x.device, ctx, _dt(x.dtype), x.data_ptr(), rows, cols, g, b, eps,
          y.data_ptr(), mean.data_ptr(), rstd.data_ptr())
    return y, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, gamma, ctx: Optional[Context] = None, out=None):
    """(dx, dgamma, dbeta) of layer_norm: dx in dy's type, dgamma and dbeta
    f32.  x: the exact input (dy's type) or its 8-bit checkpoint, an
    Fp8Tensor with block_rows 1; mean, rstd as layer_norm returned them."""
    import torch
    rows, cols = _matrix("layer_norm_backward dy", dy, _float_types())
    device = dy.device
    scales = None
    if isinstance(x, Fp8Tensor):
        shape = _codes("layer_norm_backward input", x, 1, device)
        x, scales = x.codes, x.scales.data_ptr()
    else:
        shape = _matrix("layer_norm_backward input", x, (dy.dtype,), device)
    if shape != (rows, cols):
        _fail(f"layer_norm_backward: dy {tuple(dy.shape)}, x {tuple(x.shape)}")
    mu = _vector("layer_norm_backward mean", mean, rows, torch.float32, device)
    rs = _vector("layer_norm_backward rstd", rstd, rows, torch.float32, device)
    g = _vector("layer_norm_backward gamma", gamma, cols, torch.float32, device)
    dx = _out("layer_norm_backward out", out, dy.shape, dy.dtype, device)
    dgb = torch.empty((2, cols), dtype=torch.float32, device=device)
    need = C.c_int64()
    _check(lib().nrp_layer_norm_backward_workspace(rows, cols, C.byref(need)))
    ws = torch.empty(max(need.value, 1), dtype=torch.uint8, device=device)
    _call("nrp_layer_norm_backward", device, ctx, _dt(dy.dtype), x.data_ptr(), scales,
          dy.data_ptr(), mu, rs, g, rows, cols, dx.data_ptr(), dgb[0].data_ptr(),
          dgb[1].data_ptr(), ws.data_ptr(), need.value)
    return dx, dgb[0], dgb[1]
