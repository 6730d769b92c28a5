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

import torch

from . import BF16, F32, NRP_ERR_INVALID, NRP_ERR_UNSUPPORTED, Context, NrpError, lib

_F32, _BF16, _E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
_FLOATS = {_BF16: BF16, _F32: F32}
_raw_stream = torch._C._cuda_getCurrentRawStream
_get_device = torch._C._cuda_getDevice


class Fp8Tensor(NamedTuple):
    """Block-scaled e4m3 matrix: codes torch.float8_e4m3fn [..., cols] and
    scales float32 [ceil(rows / block_rows), ceil(cols / 128)], rows the
    product of the leading dimensions; block_rows 1 (activations) or 128
    (weights)."""
    codes: object
    scales: object
    block_rows: int


def _fail(msg: str, code: int = NRP_ERR_INVALID):
    raise NrpError(code, msg)


# A small linear's kernels take a few microseconds, so the checks below ask
# for little when all is well; _explain finds out what was wrong.
def _explain(name: str, t, dtypes, dev: int):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _fail(f"{name}: a CUDA tensor is needed")
    if t.get_device() != dev:
        _fail(f"{name}: on {t.device}, the others on device {dev}")
    if t.dtype not in dtypes:
        _fail(f"{name}: dtype {t.dtype}", NRP_ERR_UNSUPPORTED)
    _fail(f"{name}: shape {tuple(t.shape)}, strides {t.stride()}: must be contiguous, with columns")


def _device(name: str, t) -> int:
    dev = t.get_device() if hasattr(t, "get_device") else -1
    if dev < 0:
        _fail(f"{name}: a CUDA tensor is needed")
    return dev


def _good(t, dtype, dev: int) -> bool:
    try:
        return t.dtype is dtype and t.get_device() == dev and t.is_contiguous()
    except AttributeError:
        return False


def _matrix(name: str, t, dtype, dev: int):
    """(rows, cols) of a contiguous tensor on device dev, its leading
    dimensions taken together."""
    shape = t.shape if _good(t, dtype, dev) else ()
    if not shape or not shape[-1]:
        _explain(name, t, (dtype,), dev)
    if len(shape) == 2:
        return shape[0], shape[1]
    return t.numel() // shape[-1], shape[-1]


def _vector(name: str, t, n: int, dtype, dev: int) -> int:
    if not _good(t, dtype, dev):
        _explain(name, t, (dtype,), dev)
    if t.numel() != n:
        _fail(f"{name}: {t.numel()} values, {n} needed")
    return t.data_ptr()


def _float(name: str, t):
    """The type of a float tensor that may be f32 or bf16."""
    dtype = getattr(t, "dtype", None)
    if dtype is not _BF16 and dtype is not _F32:
        _fail(f"{name}: dtype {dtype}", NRP_ERR_UNSUPPORTED)
    return dtype


def _scale_count(rows: int, cols: int, block_rows: int) -> int:
    return (rows if block_rows == 1 else (rows + 127) // 128) * ((cols + 127) // 128)


def _codes(name: str, q: Fp8Tensor, block_rows: int, dev: int):
    """(rows, cols) of a valid Fp8Tensor."""
    if not isinstance(q, Fp8Tensor):
        _fail(f"{name}: an Fp8Tensor is needed")
    codes, scales, block = q
    rows, cols = size = _matrix(name, codes, _E4M3, dev)
    if block != block_rows:
        _fail(f"{name}: block_rows {block}, {block_rows} needed")
    if not _good(scales, _F32, dev):
        _explain(name + " scales", scales, (_F32,), dev)
    if scales.numel() != _scale_count(rows, cols, block):
        _fail(f"{name}: {scales.numel()} scales for {rows} x {cols} codes")
    return size


def _out(name: str, out, shape, dtype, dev: int):
    if dtype not in _FLOATS:
        _fail(f"{name}: dtype {dtype}", NRP_ERR_UNSUPPORTED)
    _matrix(name, out, dtype, dev)
    if out.shape != torch.Size(shape):
        _fail(f"{name}: shape {tuple(out.shape)}, {tuple(shape)} needed")
    return out


def _new(like, shape, dtype, name: str):
    """A tensor on like's device (cheapest where like has its type)."""
    if dtype is like.dtype:
        return like.new_empty(shape)
    if dtype not in _FLOATS:
        _fail(f"{name}: dtype {dtype}", NRP_ERR_UNSUPPORTED)
    return like.new_empty(shape, dtype=dtype)


def _call(fn, dev: int, ctx: Optional[Context], *args):
    """fn(context, the device's current stream, *args), with the thread's
    current device left as it was (the library makes the context's current)."""
    if ctx is None:
        ctx = Context._default.get(dev) or Context.default(dev)
    elif ctx.device != dev:
        _fail(f"context of device {ctx.device}, tensors on device {dev}")
    current = _get_device()
    rc = fn(ctx.handle, _raw_stream(dev), *args)
    if current != dev:
        torch.cuda.set_device(current)
    if rc < 0:
        raise NrpError(rc, lib().nrp_last_error().decode())


def _new_codes(shape, rows: int, cols: int, block_rows: int, like) -> Fp8Tensor:
    return Fp8Tensor(
        like.new_empty(shape, dtype=_E4M3),
        like.new_empty((rows if block_rows == 1 else (rows + 127) // 128, (cols + 127) // 128),
                       dtype=_F32), block_rows)


def fp8_quantize(x, block_rows: int = 1, ctx: Optional[Context] = None,
                 out: Optional[Fp8Tensor] = None) -> Fp8Tensor:
    """e4m3 codes of x (f32 or bf16 [..., cols], cols % 16 == 0) with one
    power-of-two scale per block_rows x 128 block: the smallest with which
    the block's largest value is at most 448.  block_rows 1 for activations
    and gradients, 128 for weights.  NaN and infinities become NaN."""
    dev = _device("quantize", x)
    rows, cols = _matrix("quantize", x, _float("quantize", x), dev)
    if out is None:
        if block_rows not in (1, 128):
            _fail(f"block_rows {block_rows} (supported: 1, 128)", NRP_ERR_UNSUPPORTED)
        out = _new_codes(x.shape, rows, cols, block_rows, x)
    elif _codes("quantize out", out, block_rows, dev) != (rows, cols):
        _fail(f"quantize out: codes {tuple(out.codes.shape)} for {tuple(x.shape)}")
    _call(lib().nrp_fp8_quantize, dev, ctx, _FLOATS[x.dtype], x.data_ptr(), rows, cols, block_rows,
          out[0].data_ptr(), out[1].data_ptr())
    return out


def fp8_dequantize(q: Fp8Tensor, dtype=_BF16, ctx: Optional[Context] = None, out=None):
    """The values q stands for, in bf16 (default) or f32."""
    if not isinstance(q, Fp8Tensor):
        _fail("dequantize: an Fp8Tensor is needed")
    dev = _device("dequantize", q.codes)
    rows, cols = _codes("dequantize", q, q.block_rows, dev)
    if out is None:
        out = _new(q.scales, q.codes.shape, dtype, "dequantize out")
    else:
        _out("dequantize out", out, q.codes.shape, dtype, dev)
    _call(lib().nrp_fp8_dequantize, dev, ctx, q.codes.data_ptr(), q.scales.data_ptr(), rows, cols,
          q.block_rows, _FLOATS[dtype], out.data_ptr())
    return out


def _product(fn, name: str, x, w: Fp8Tensor, trans: bool, bias, dtype, ctx, out, codes):
    if not isinstance(w, Fp8Tensor):
        _fail(f"{name} weight: an Fp8Tensor is needed")
    dev = _device(name + " weight", w[0])
    n, k = _codes(name + " weight", w, 128, dev)
    red, cols = (n, k) if trans else (k, n)
    if isinstance(x, Fp8Tensor):
        if codes is not None:
            _fail(f"{name}: codes= takes the codes of a tensor that the call quantises")
        m, r = _codes(name + " input", x, 1, dev)
        t, src, xq, xs = x[0], None, x[0].data_ptr(), x[1].data_ptr()
        dtype = dtype or _BF16
    else:
        t = x
        tx = _float(name + " input", x)
        m, r = _matrix(name + " input", x, tx, dev)
        if dtype is not None and dtype is not tx:
            _fail(f"{name}: input {tx}, output {dtype}", NRP_ERR_UNSUPPORTED)
        src, dtype = x.data_ptr(), tx
        if codes is None:  # not wanted: both in one buffer of this call
            words = (m * r + 15) // 16 * 4
            buf = w[1].new_empty(words + _scale_count(m, r, 1))
            xq = buf.data_ptr()
            xs = xq + 4 * words
        else:
            if _codes(name + " codes", codes, 1, dev) != (m, r):
                _fail(f"{name}: codes {tuple(codes.codes.shape)} for {tuple(x.shape)}")
            xq, xs = codes[0].data_ptr(), codes[1].data_ptr()
    shape = t.shape
    if r != red:
        _fail(f"{name}: input {tuple(shape)}, weight {tuple(w.codes.shape)}")
    shape = (*shape[:-1], cols)
    if out is None:
        out = _new(t, shape, dtype, name)
    else:
        _out(name + " out", out, shape, dtype, dev)
    dt = _FLOATS[dtype]
    if trans:
        _call(fn, dev, ctx, dt, src, xq, xs, m, red, w[0].data_ptr(), w[1].data_ptr(), cols,
              out.data_ptr())
    else:
        _call(fn, dev, ctx, dt, src, xq, xs, m, red, w[0].data_ptr(), w[1].data_ptr(), cols,
              None if bias is None else _vector(name + " bias", bias, cols, dtype, dev),
              out.data_ptr())
    return out


def fp8_linear(x, w: Fp8Tensor, bias=None, dtype=None, ctx: Optional[Context] = None, out=None,
               codes: Optional[Fp8Tensor] = None):
    """y = x . w^T (+ bias) of 8-bit operands, f32 sums.  w [N, K] with 128 x
    128 blocks.  x: an Fp8Tensor [..., K] (y in `dtype`, default bf16), or an
    f32 or bf16 tensor, quantised in the call -- into `codes` when given, the
    checkpoint that fp8_linear_weight_grad takes -- and y in its type.  bias
    [N] in y's type."""
    return _product(lib().nrp_fp8_linear, "fp8_linear", x, w, False, bias, dtype, ctx, out, codes)


def fp8_linear_input_grad(dy, w: Fp8Tensor, dtype=None, ctx: Optional[Context] = None, out=None,
                          codes: Optional[Fp8Tensor] = None):
    """dx = dy . w, the gradient of fp8_linear's input; dy [..., N] as
    fp8_linear's x."""
    return _product(lib().nrp_fp8_linear_input_grad, "fp8_linear_input_grad", dy, w, True, None,
                    dtype, ctx, out, codes)


def fp8_linear_weight_grad(dy, x: Fp8Tensor, bias: bool = False, dtype=_F32,
                           ctx: Optional[Context] = None, out=None, bias_out=None):
    """(dw [N, K], dbias [N] or None) from dy (bf16 [..., N], N % 8 == 0) and
    the 8-bit checkpoint x [..., K] of the linear's input; dw and dbias in
    `dtype` (default f32)."""
    name = "fp8_linear_weight_grad"
    dev = _device(name + " dy", dy)
    m, n = _matrix(name + " dy", dy, _BF16, dev)
    mx, k = _codes(name + " input", x, 1, dev)
    if m != mx:
        _fail(f"{name}: {m} rows of dy, {mx} of x")
    like = dy if dtype is _BF16 else x[1]
    dw = (_new(like, (n, k), dtype, name) if out is None
          else _out(name + " out", out, (n, k), dtype, dev))
    if bias_out is not None:
        db = _out(name + " bias_out", bias_out, (n,), dtype, dev)
    else:
        db = like.new_empty(n) if bias else None
    _call(lib().nrp_fp8_linear_weight_grad, dev, ctx, dy.data_ptr(), x[0].data_ptr(),
          x[1].data_ptr(), m, n, k, _FLOATS[dtype], dw.data_ptr(),
          None if db is None else db.data_ptr())
    return dw, db


def layer_norm(x, gamma, beta, eps: float = 1e-5, ctx: Optional[Context] = None, out=None):
    """(y, mean, rstd): LayerNorm over the last dimension of x (f32 or bf16);
    gamma, beta f32 [cols]; mean, rstd f32 [rows].  out may be x."""
    dev = _device("layer_norm", x)
    dtype = _float("layer_norm", x)
    rows, cols = _matrix("layer_norm", x, dtype, dev)
    g = _vector("layer_norm gamma", gamma, cols, _F32, dev)
    b = _vector("layer_norm beta", beta, cols, _F32, dev)
    y = torch.empty_like(x) if out is None else _out("layer_norm out", out, x.shape, dtype, dev)
    mean = gamma.new_empty(x.shape[:-1])
    rstd = torch.empty_like(mean)
    _call(lib().nrp_layer_norm, dev, ctx, _FLOATS[dtype], x.data_ptr(), rows, cols, g, b, eps,
          y.data_ptr(), mean.data_ptr(), rstd.data_ptr())
    return y, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, gamma, ctx: Optional[Context] = None, out=None):
    """(dx, dgamma, dbeta) of layer_norm: dx in dy's type, dgamma and dbeta
    f32.  x: the exact input (dy's type) or its 8-bit checkpoint, an
    Fp8Tensor with block_rows 1; mean, rstd as layer_norm returned them."""
    name = "layer_norm_backward"
    dev = _device(name + " dy", dy)
    dtype = _float(name + " dy", dy)
    size = rows, cols = _matrix(name + " dy", dy, dtype, dev)
    scales = None
    if isinstance(x, Fp8Tensor):
        xsize = _codes(name + " input", x, 1, dev)
        x, scales = x[0], x[1].data_ptr()
    else:
        xsize = _matrix(name + " input", x, dtype, dev)
    if xsize != size:
        _fail(f"{name}: dy {tuple(dy.shape)}, x {tuple(x.shape)}")
    mu = _vector(name + " mean", mean, rows, _F32, dev)
    rs = _vector(name + " rstd", rstd, rows, _F32, dev)
    g = _vector(name + " gamma", gamma, cols, _F32, dev)
    dx = torch.empty_like(dy) if out is None else _out(name + " out", out, dy.shape, dtype, dev)
    dgamma = gamma.new_empty(cols)
    dbeta = torch.empty_like(dgamma)
    need = C.c_int64()
    lib().nrp_layer_norm_backward_workspace(rows, cols, C.byref(need))
    bytes_ = need.value
    ws = gamma.new_empty(bytes_ // 4) if bytes_ else None
    _call(lib().nrp_layer_norm_backward, dev, ctx, _FLOATS[dtype], x.data_ptr(), scales,
          dy.data_ptr(), mu, rs, g, rows, cols, dx.data_ptr(), dgamma.data_ptr(),
          dbeta.data_ptr(), None if ws is None else ws.data_ptr(), bytes_)
    return dx, dgamma, dbeta
