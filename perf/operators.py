"""What is measured of the 8-bit linear layers' and the layer norm's training
and serving operators: the cases, their inputs, the plain forms and the
64-bit definitions.

Operators (entry points of the package):
  quantize      fp8_quantize            e4m3 codes, one power-of-two scale per
                                        1 x 128 (activations) or 128 x 128
                                        (weights) block
  linear        fp8_linear              y = q(x) . w^T + b
  input_grad    fp8_linear_input_grad   dx = q(dy) . w
  weight_grad   fp8_linear_weight_grad  dw = dy^T . x~, db = sum dy, x~ the
                                        8-bit checkpoint of the layer's input
  norm          layer_norm              y, mean, rstd
  norm_grad     layer_norm_backward     dx, dgamma, dbeta; x exact or the
                                        8-bit checkpoint

Sizes are the encoder's: d_model 1024 (512 for the small models), ff_dim
4096, 14-frame streaming chunks, one to 32 utterances of up to 12500 frames.
"""
import math

import torch

own = False

E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # a feed-forward weight after an optimizer step, requantised from f32
        {"name": "quantize_weight", "op": "quantize", "rows": 4096, "cols": 1024, "block": 128,
         "dtype": "f32"},
        # the feed-forward's inner activations of a 32-utterance batch
        {"name": "quantize_batch", "op": "quantize", "rows": 16000, "cols": 4096, "block": 1,
         "dtype": "bf16"},
        # one streaming session's chunk through a feed-forward's first linear
        {"name": "linear_chunk", "op": "linear", "m": 14, "k": 1024, "n": 4096, "x": "bf16",
         "dtype": "bf16"},
        # a training batch through it, the input quantised on the way
        {"name": "linear_batch", "op": "linear", "m": 16000, "k": 1024, "n": 4096, "x": "bf16",
         "dtype": "bf16"},
        # 64 sessions' chunks back through a projection
        {"name": "input_grad_chunks", "op": "input_grad", "m": 896, "k": 1024, "n": 1024,
         "x": "bf16", "dtype": "bf16"},
        # the batch back through the feed-forward's first linear
        {"name": "input_grad_batch", "op": "input_grad", "m": 16000, "k": 1024, "n": 4096,
         "x": "fp8", "dtype": "bf16"},
        # one utterance of odd length, a projection's weight
        {"name": "weight_grad_utterance", "op": "weight_grad", "m": 749, "k": 1024, "n": 1024,
         "dtype": "f32", "bias": True},
        # the batch, the feed-forward's first weight
        {"name": "weight_grad_batch", "op": "weight_grad", "m": 16000, "k": 1024, "n": 4096,
         "dtype": "f32", "bias": True},
        # one chunk of a small model
        {"name": "norm_chunk", "op": "norm", "rows": 14, "cols": 512, "dtype": "f32"},
        # four long-form utterances
        {"name": "norm_long", "op": "norm", "rows": 50000, "cols": 1024, "dtype": "bf16"},
        # one utterance of odd length, the exact input kept
        {"name": "norm_grad_utterance", "op": "norm_grad", "rows": 749, "cols": 512,
         "x": "same", "dtype": "bf16"},
        # the long-form batch, its input kept in 8 bits
        {"name": "norm_grad_long", "op": "norm_grad", "rows": 50000, "cols": 1024, "x": "fp8",
         "dtype": "bf16"},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi, max(lo, round(v / step) * step)))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "input_grad", "weight_grad", "norm",
                     "norm_grad"])
    if op == "quantize":
        return {"op": op, "rows": _log(rng, 1, 16000), "cols": _log(rng, 16, 4096, 16),
                "block": rng.choice([1, 1, 128]), "dtype": rng.choice(["bf16", "f32"])}
    if op == "linear":
        return {"op": op, "m": _log(rng, 1, 16000), "k": _log(rng, 64, 2048, 16),
                "n": _log(rng, 64, 2048), "x": rng.choice(["bf16", "fp8", "f32"]),
                "dtype": rng.choice(["bf16", "bf16", "f32"])}
    if op == "input_grad":
        return {"op": op, "m": _log(rng, 1, 16000), "k": _log(rng, 64, 2048, 16),
                "n": _log(rng, 64, 2048, 16), "x": rng.choice(["bf16", "fp8"]),
                "dtype": "bf16"}
    if op == "weight_grad":
        return {"op": op, "m": _log(rng, 1, 16000), "k": _log(rng, 64, 2048, 16),
                "n": _log(rng, 64, 2048, 8), "dtype": rng.choice(["f32", "f32", "bf16"]),
                "bias": rng.random() < 0.7}
    if op == "norm":
        return {"op": op, "rows": _log(rng, 1, 50000), "cols": _log(rng, 16, 1024),
                "dtype": rng.choice(["bf16", "bf16", "f32"])}
    x = rng.choice(["same", "fp8"])
    return {"op": op, "rows": _log(rng, 1, 50000), "cols": _log(rng, 16, 1024, 16 if x == "fp8" else 1),
            "x": x, "dtype": rng.choice(["bf16", "bf16", "f32"])}


# ------------------------------------------------------------------ inputs
def _pkg():
    from __graft_entry__ import load_package
    return load_package()


def _activations(g, rows, cols, dtype):
    """Residual-stream rows: per-channel spread and offset, a few large
    channels, and rows of different loudness."""
    spread = torch.exp(0.5 * torch.randn(cols, device="cuda", generator=g))
    offset = 0.3 * torch.randn(cols, device="cuda", generator=g)
    loud = torch.exp(0.3 * torch.randn(rows, 1, device="cuda", generator=g))
    x = torch.randn(rows, cols, device="cuda", generator=g).mul_(spread).add_(offset).mul_(loud)
    return x.to(dtype)


def _gradients(g, rows, cols, dtype):
    """Output gradients: small, rows of very different size."""
    size = 1e-3 * torch.exp(torch.randn(rows, 1, device="cuda", generator=g))
    return torch.randn(rows, cols, device="cuda", generator=g).mul_(size).to(dtype)


def _weight(g, n, k):
    return torch.randn(n, k, device="cuda", generator=g).div_(math.sqrt(k))


def _codes(x, block):
    """Codes and scales of x, made here so that both sides start alike."""
    return _plain_quantize(x, block)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], {"case": dict(case)}
    dt = DTYPES[case["dtype"]]
    if op == "quantize":
        if case["block"] == 128:
            s["x"] = _weight(g, case["rows"], case["cols"]).to(dt)
        else:
            s["x"] = _activations(g, case["rows"], case["cols"], dt)
    elif op in ("linear", "input_grad"):
        m, k, n = case["m"], case["k"], case["n"]
        s["w"] = _codes(_weight(g, n, k), 128)
        if op == "linear":
            x = _activations(g, m, k, torch.float32)
            s["bias"] = (0.1 * torch.randn(n, device="cuda", generator=g)).to(_out_dtype(case))
        else:
            x = _gradients(g, m, n, torch.float32)
        s["x"] = _codes(x.to(torch.bfloat16), 1) if case["x"] == "fp8" else x.to(DTYPES[case["x"]])
    elif op == "weight_grad":
        s["dy"] = _gradients(g, case["m"], case["n"], torch.bfloat16)
        s["x"] = _codes(_activations(g, case["m"], case["k"], torch.bfloat16), 1)
    else:
        x = _activations(g, case["rows"], case["cols"], dt)
        s["gamma"] = 1 + 0.2 * torch.randn(case["cols"], device="cuda", generator=g)
        s["beta"] = 0.1 * torch.randn(case["cols"], device="cuda", generator=g)
        s["x"] = x
        if op == "norm_grad":
            s["dy"] = _gradients(g, case["rows"], case["cols"], dt)
            _, s["mean"], s["rstd"] = _plain_norm(x, s["gamma"], s["beta"])
            if case["x"] == "fp8":
                s["x"] = _codes(x, 1)
    return s


def _out_dtype(case):
    """The output's type: with x in f32 or bf16 the operands share it."""
    return DTYPES[case["dtype"] if case["x"] == "fp8" else case["x"]]


# ------------------------------------------------------------- plain forms
def _blocks(x, block):
    """x as [row blocks, block, column blocks, 128], the rest filled with zeros."""
    rows, cols = x.shape
    rb, cb = -(-rows // block), -(-cols // 128)
    p = torch.nn.functional.pad(x, (0, cb * 128 - cols, 0, rb * block - rows))
    return p.view(rb, block, cb, 128)


def _plain_quantize(x, block):
    """The smallest power of two s with amax / s <= 448, codes = e4m3(x / s)."""
    rows, cols = x.shape
    p = _blocks(x.float(), block)
    amax = p.abs().amax(dim=(1, 3))
    m, e = torch.frexp(amax)  # amax = m * 2^e, 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(amax > 0, e, torch.zeros_like(e)).clamp(-117, 119)
    scales = torch.ldexp(torch.ones_like(amax), e)
    q = (p / scales[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    q = q.reshape(p.shape[0] * block, -1)[:rows, :cols]
    return q.to(torch.float8_e4m3fn).contiguous(), scales


def _plain_dequantize(codes, scales, block):
    rows, cols = codes.shape
    p = _blocks(codes.float(), block) * scales[:, None, :, None]
    return p.reshape(p.shape[0] * block, -1)[:rows, :cols]


def _plain_operand(x, block=1):
    return _plain_dequantize(*(x if isinstance(x, tuple) else _plain_quantize(x, block)), block)


def _plain_norm(x, gamma, beta, eps=1e-5):
    v = x.float()
    mean = v.mean(dim=1, dtype=torch.float64)  # its sum may cancel
    d = v - mean[:, None]
    rstd = 1 / torch.sqrt(d.square().mean(dim=1) + eps)
    y = d * rstd[:, None] * gamma.double() + beta.double()
    return y.to(x.dtype), mean.float(), rstd.float()


def _plain_run(s):
    case = s["case"]
    op = case["op"]
    if op == "quantize":
        return list(_plain_quantize(s["x"], case["block"]))
    if op == "linear":
        y = _plain_operand(s["x"]) @ _plain_operand(s["w"], 128).t() + s["bias"].float()
        return y.to(_out_dtype(case))
    if op == "input_grad":
        return (_plain_operand(s["x"]) @ _plain_operand(s["w"], 128)).to(_out_dtype(case))
    if op == "weight_grad":
        dw = s["dy"].float().t() @ _plain_operand(s["x"])
        db = s["dy"].sum(dim=0, dtype=torch.float64) if case["bias"] else None
        dt = DTYPES[case["dtype"]]
        return [dw.to(dt)] + ([db.to(dt)] if case["bias"] else [])
    if op == "norm":
        return list(_plain_norm(s["x"], s["gamma"], s["beta"]))
    x = _plain_operand(s["x"]) if isinstance(s["x"], tuple) else s["x"].float()
    dy = s["dy"].float()
    xhat = (x - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * s["gamma"]
    c1 = g.mean(dim=1, keepdim=True)
    c2 = (g * xhat).mean(dim=1, keepdim=True)
    dx = s["rstd"][:, None] * (g - c1 - xhat * c2)
    dgamma = (dy * xhat).sum(dim=0, dtype=torch.float64).float()
    dbeta = dy.sum(dim=0, dtype=torch.float64).float()
    return [dx.to(s["dy"].dtype), dgamma, dbeta]


# --------------------------------------------------------------------- run
def _own_run(s):
    case, pkg = s["case"], _pkg()
    op = case["op"]
    x = s["x"]
    if isinstance(x, tuple):
        x = pkg.Fp8Tensor(*x, 1)
    if op == "quantize":
        q = pkg.fp8_quantize(x, case["block"])
        return [q.codes, q.scales]
    if op == "linear":
        return pkg.fp8_linear(x, pkg.Fp8Tensor(*s["w"], 128), s["bias"], dtype=_out_dtype(case))
    if op == "input_grad":
        return pkg.fp8_linear_input_grad(x, pkg.Fp8Tensor(*s["w"], 128), dtype=_out_dtype(case))
    if op == "weight_grad":
        dw, db = pkg.fp8_linear_weight_grad(s["dy"], x, bias=case["bias"],
                                            dtype=DTYPES[case["dtype"]])
        return [dw] + ([db] if case["bias"] else [])
    if op == "norm":
        return list(pkg.layer_norm(x, s["gamma"], s["beta"]))
    return list(pkg.layer_norm_backward(s["dy"], x, s["mean"], s["rstd"], s["gamma"]))


def run(state):
    if own:
        return _own_run(state)
    return _plain_run(state)


# -------------------------------------------------------------------- work
def _scale_bytes(rows, cols, block):
    return 4 * (-(-rows // block)) * (-(-cols // 128))


def work(case):
    op = case["op"]
    size = {"bf16": 2, "f32": 4}
    if op == "quantize":
        r, c = case["rows"], case["cols"]
        return {"bytes": r * c * (size[case["dtype"]] + 1) + _scale_bytes(r, c, case["block"]),
                "flops": 2 * r * c}
    if op in ("linear", "input_grad"):
        m, k, n = case["m"], case["k"], case["n"]
        red, out = (k, n) if op == "linear" else (n, k)
        x = m * red + _scale_bytes(m, red, 1) if case["x"] == "fp8" else m * red * size[case["x"]]
        w = n * k + _scale_bytes(n, k, 128)
        o = size[case["dtype"] if case["x"] == "fp8" else case["x"]]
        return {"bytes": x + w + m * out * o + (n * o if op == "linear" else 0),
                "flops": 2 * m * n * k}
    if op == "weight_grad":
        m, k, n, o = case["m"], case["k"], case["n"], size[case["dtype"]]
        return {"bytes": m * n * 2 + m * k + _scale_bytes(m, k, 1) + n * k * o
                + (n * o if case["bias"] else 0), "flops": 2 * m * n * k}
    r, c, e = case["rows"], case["cols"], size[case["dtype"]]
    if op == "norm":
        return {"bytes": 2 * r * c * e + 8 * r + 8 * c, "flops": 7 * r * c}
    x = r * c + _scale_bytes(r, c, 1) if case["x"] == "fp8" else r * c * e
    return {"bytes": x + 2 * r * c * e + 8 * r + 12 * c, "flops": 13 * r * c}


# ------------------------------------------------- the definitions, 64 bits
def _exact_values(x, block):
    """What the codes of x stand for, block by block in 64 bits; x is a tensor
    to quantise or a (codes, scales) pair."""
    if not isinstance(x, torch.Tensor):
        codes, scales = x[0].to(torch.float64), x[1].to(torch.float64)
        s = scales.repeat_interleave(block, 0)[:codes.shape[0]]
        return codes * s.repeat_interleave(128, 1)[:, :codes.shape[1]]
    v = x.to(torch.float64)
    out = torch.empty_like(v)
    for c in range(0, v.shape[1], 128):
        part = v[:, c:c + 128]
        top = part.abs().amax(dim=1, keepdim=True)
        s = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp(-117, 119))
        # log2 next to a whole number may land on either side of it
        s = torch.where(top > 448 * s, 2 * s, s)
        s = torch.where(top <= 224 * s, s / 2, s)
        s = torch.where(top > 0, s.clamp(2.0 ** -117, 2.0 ** 119), torch.ones_like(s))
        t = part / s
        # e4m3: three bits after the leading one, steps of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3)
        out[:, c:c + 128] = torch.round(t / step) * step * s
    return out


def exact(case, seed):
    op = case["op"]
    if op == "quantize":
        return None
    s = prepare(case, seed)
    if op in ("linear", "input_grad"):
        x, w = _exact_values(s["x"], 1), _exact_values(s["w"], 128)
        return x @ w.t() + s["bias"].to(torch.float64) if op == "linear" else x @ w
    if op == "weight_grad":
        dy = s["dy"].to(torch.float64)
        dw = dy.t() @ _exact_values(s["x"], 1)
        return [dw] + ([dy.sum(dim=0)] if case["bias"] else [])
    gamma = s["gamma"].to(torch.float64)
    if op == "norm":
        x = s["x"].to(torch.float64)
        mean = x.mean(dim=1)
        var = ((x - mean[:, None]) ** 2).mean(dim=1)
        rstd = (var + 1e-5) ** -0.5
        y = (x - mean[:, None]) * rstd[:, None] * gamma + s["beta"].to(torch.float64)
        return [y, mean, rstd]
    x = s["x"].to(torch.float64) if isinstance(s["x"], torch.Tensor) else _exact_values(s["x"], 1)
    dy = s["dy"].to(torch.float64)
    mean, rstd = s["mean"].to(torch.float64)[:, None], s["rstd"].to(torch.float64)[:, None]
    n = x.shape[1]
    u = (x - mean) * rstd
    dgamma, dbeta = (dy * u).sum(dim=0), dy.sum(dim=0)
    dy *= gamma
    dx = rstd * (dy - dy.sum(dim=1, keepdim=True) / n - u * ((dy * u).sum(dim=1, keepdim=True) / n))
    return [dx, dgamma, dbeta]
