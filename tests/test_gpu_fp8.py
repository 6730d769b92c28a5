"""8-bit floating-point linears and their gradients on the device, against
plain 64-bit forms.

Tolerances (u = 2^-24, half a step of f32, relative):
- quantisation and dequantisation are exact: codes, scales and values equal;
- products: every product of two codes (or of a bf16 dy and a bf16 value) is
  exact in f32.  A tensor-core step aligns its products and the running sum to
  the largest and may cut each at 2^-23 of it, so a chain of n additions is off
  by at most n * 2^-23 * S, S = sum |a| |b|: n = 132 within a 128-block plus
  one f32 rounding (u S) per block sum, or n = M + M/16 over M tokens, plus
  the splits' additions.  Then the output's rounding, 2^-8 |y| in bf16 (half
  of its eps), u |y| in f32;
- the bias gradient: chains of at most M + 16 f32 additions, u each.
"""
import math

import numpy as np
import pytest

from __graft_entry__ import load_package

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def nrp():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return load_package()


def quantize_ref(x, block_rows):
    """(codes, scales) of a CPU tensor by the definition, in 64 bits."""
    import torch
    rows, cols = x.shape
    v = x.double().numpy()
    rb, cb = -(-rows // block_rows), -(-cols // 128)
    scales = np.ones((rb, cb))
    t = np.empty_like(v)
    for i in range(rb):
        for j in range(cb):
            at = np.s_[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128]
            part = np.abs(v[at])
            part = part[np.isfinite(part)]
            top = part.max() if part.size else 0.0
            if top > 0:
                m, e = math.frexp(top)
                k = min(max(e - 9 if m <= 0.875 else e - 8, -117), 119)
                scales[i, j] = 2.0 ** k
            t[at] = v[at] / scales[i, j]
    t[~np.isfinite(t)] = np.nan
    t = np.clip(t, -448, 448)
    with np.errstate(invalid="ignore", divide="ignore"):
        step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(t), 2.0 ** -6))) - 3)
        t = np.round(t / step) * step  # numpy rounds to nearest even
    return (torch.from_numpy(t).float().to(torch.float8_e4m3fn),
            torch.from_numpy(scales).float())


def values(q):
    """float64 values of an Fp8Tensor on the CPU."""
    c, s = q.codes.cpu().double(), q.scales.cpu().double()
    c = c.reshape(-1, c.shape[-1])
    s = s.repeat_interleave(q.block_rows, 0)[:c.shape[0]].repeat_interleave(128, 1)
    return c * s[:, :c.shape[1]]


def close(got, ref, tol):
    d = (got.double().cpu().reshape(ref.shape) - ref).abs()
    bad = ~(d <= tol)
    assert not bad.any(), (int(bad.sum()), float((d / tol.clamp(min=1e-300)).max()))


def rand(shape, seed, scale=1.0):
    import torch
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale


def half_step(dtype):
    import torch
    return torch.finfo(dtype).eps / 2


# --------------------------------------------------------------- quantise
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols,block", [(1, 16, 1), (1, 128, 1), (3, 144, 1), (14, 1024, 1),
                                             (33, 2000, 1), (1, 16, 128), (127, 144, 128),
                                             (128, 128, 128), (129, 1040, 128), (300, 272, 128)])
def test_quantize_exact(nrp, dtype, rows, cols, block):
    import torch
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    x = (rand((rows, cols), rows + cols) * torch.exp2(rand((rows, 1), 5) * 6)).to(dt)
    codes, scales = quantize_ref(x, block)
    q = nrp.fp8_quantize(x.cuda(), block)
    assert torch.equal(q.scales.cpu(), scales)
    assert torch.equal(q.codes.cpu().view(torch.uint8), codes.view(torch.uint8))
    for out in (torch.bfloat16, torch.float32):  # exact in both
        assert torch.equal(nrp.fp8_dequantize(q, out).cpu().double(), values(q))
    y = torch.full((rows + 1, cols), 3.0, dtype=dt, device="cuda")
    nrp.fp8_dequantize(q, dt, out=y[:rows])
    assert (y[rows] == 3).all()


@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantize_special_values(nrp, dtype, block):
    """Zeros, subnormals, the largest values, exact powers and the scale's
    border 448 * 2^k, ties, NaN and infinities; one block of each."""
    import torch
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    inf, nan = float("inf"), float("nan")
    tops = [0.0, 448.0, 449.0 if dtype == "f32" else 450.0, 447.0 if dtype == "f32" else 446.0, 1.0,
            torch.finfo(dt).max, torch.finfo(dt).tiny, 1e-40, 2.0 ** -126, 224.0, 2.0 ** 127]
    rows = []
    for t in tops:
        r = torch.zeros(128)
        r[0] = -t
        r[1:64] = torch.linspace(-1, 1, 63) * t / 8
        rows.append(r)
    ties = torch.zeros(128)
    ties[:8] = torch.tensor([448.0, 17.0, 19.0, 27.0, 2.0 ** -10, 3 * 2.0 ** -10, 13.5, -17.0])
    rows.append(ties)
    for special in ([inf], [nan], [-inf, nan, 3.0], [inf] * 128):
        r = torch.zeros(128)
        r[:len(special)] = torch.tensor(special)
        rows.append(r)
    x = torch.stack(rows).to(dt)
    if block == 128:  # each row in a 128 x 128 block of its own
        wide = torch.zeros(128, 128 * x.shape[0], dtype=dt)
        wide[5] = x.reshape(-1)
        x = wide
    codes, scales = quantize_ref(x, block)
    q = nrp.fp8_quantize(x.cuda(), block)
    assert torch.equal(q.scales.cpu(), scales)
    got, ref = q.codes.cpu().float(), codes.float()
    assert torch.equal(got.isnan(), ref.isnan())
    ok = ~ref.isnan()
    assert torch.equal(got[ok], ref[ok])
    assert got[~x.float().isfinite()].isnan().all()
    assert nrp.fp8_dequantize(q, torch.float32).cpu()[ok].isfinite().all()


# --------------------------------------------------------------- products
SHAPES = [(1, 16, 1), (1, 1024, 4096), (2, 144, 130), (14, 1024, 1024), (15, 528, 97),
          (16, 4096, 512), (17, 128, 256), (33, 256, 64), (64, 1040, 300), (65, 400, 513),
          (127, 128, 128), (128, 384, 384), (129, 640, 255), (300, 1024, 1000), (896, 1024, 1024),
          (1000, 272, 2048),
          # 256-column tiles: ragged rows and columns, one to nine reduction blocks
          (4737, 144, 1008), (2433, 1040, 2040), (2304, 112, 2048), (19000, 128, 250)]


def product_tol(x, w, red, y, dtype):
    s = x.abs() @ w.abs()
    return s * (132 * 2.0 ** -23 + (red // 128 + 4) * U) + y.abs() * half_step(dtype)


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("kind", ["bf16", "f32", "fp8-bf16", "fp8-f32"])
def test_linear(nrp, m, k, n, kind):
    import torch
    dt = torch.float32 if kind.endswith("f32") else torch.bfloat16
    w = nrp.fp8_quantize(rand((n, k), 2).cuda() / math.sqrt(k), 128)
    b = rand((n,), 3).to(dt) if n % 2 == 0 else None
    x = (rand((m, k), 4) * torch.exp2(rand((m, 1), 6) * 3)).to(dt)
    q = nrp.fp8_quantize(x.cuda())
    codes = None
    if kind.startswith("fp8"):
        y = nrp.fp8_linear(q, w, None if b is None else b.cuda(), dtype=dt)
    else:
        codes = nrp.Fp8Tensor(torch.empty_like(q.codes), torch.empty_like(q.scales), 1)
        y = nrp.fp8_linear(x.cuda(), w, None if b is None else b.cuda(), codes=codes)
        assert torch.equal(codes.codes.view(torch.uint8), q.codes.view(torch.uint8))
        assert torch.equal(codes.scales, q.scales)
    assert y.dtype == dt and y.shape == (m, n)
    xv, wv = values(q), values(w)
    ref = xv @ wv.t()
    tol = product_tol(xv, wv.t(), k, ref, torch.float32)
    if b is not None:
        ref = ref + b.double()
    close(y, ref, tol + ref.abs() * half_step(dt) + ref.abs() * U)
    nrp.Context.default().check()


@pytest.mark.parametrize("m,k,n", [(1, 16, 16), (1, 1024, 4096), (14, 1024, 1024), (15, 144, 528),
                                   (17, 256, 128), (65, 528, 400), (128, 384, 384),
                                   (129, 240, 640), (300, 1008, 1024), (896, 1024, 1024),
                                   (1000, 2048, 272), (4737, 1008, 144), (2433, 2032, 1040),
                                   (2304, 2048, 112), (19000, 240, 128)])
@pytest.mark.parametrize("kind", ["bf16", "f32", "fp8-bf16", "fp8-f32"])
def test_input_grad(nrp, m, k, n, kind):
    import torch
    dt = torch.float32 if kind.endswith("f32") else torch.bfloat16
    w = nrp.fp8_quantize(rand((n, k), 2).cuda() / math.sqrt(k), 128)
    g = (rand((m, n), 4, 1e-3) * torch.exp2(rand((m, 1), 6) * 3)).to(dt)
    q = nrp.fp8_quantize(g.cuda())
    dx = nrp.fp8_linear_input_grad(q if kind.startswith("fp8") else g.cuda(), w, dtype=dt)
    assert dx.dtype == dt and dx.shape == (m, k)
    gv, wv = values(q), values(w)
    ref = gv @ wv
    close(dx, ref, product_tol(gv, wv, n, ref, dt))
    nrp.Context.default().check()


@pytest.mark.parametrize("m", [1, 14, 40, 300, 1000])
def test_products_with_any_scales(nrp, m):
    """Scales that are not powers of two, zero and negative ones; leading
    dimensions; rows behind the last one stay."""
    import torch
    k, n = 400, 336
    g = torch.Generator().manual_seed(m)
    x = nrp.fp8_quantize(rand((m, k), 7).cuda())
    w = nrp.fp8_quantize(rand((n, k), 8).cuda(), 128)
    x.scales.copy_(torch.randn(x.scales.shape, generator=g))
    w.scales.copy_(torch.randn(w.scales.shape, generator=g))
    x.scales[0] = 0
    for trans in (False, True):
        if trans:
            x = nrp.fp8_quantize(rand((m, n), 9).cuda())
            x.scales.copy_(torch.randn(x.scales.shape, generator=g))
        cols = k if trans else n
        out = torch.full((m + 3, cols), 7.0, device="cuda")
        call = nrp.fp8_linear_input_grad if trans else nrp.fp8_linear
        call(x, w, dtype=torch.float32, out=out[:m])
        assert (out[m:] == 7).all()
        xv, wv = values(x), values(w) if trans else values(w).t()
        # one more rounding: the two scales' product
        close(out[:m], xv @ wv, product_tol(xv, wv, n if trans else k, xv @ wv, torch.float32)
              + (xv.abs() @ wv.abs()) * 4 * U)


@pytest.mark.parametrize("m", [3, 20, 200])
def test_nan_rows_stay_rows(nrp, m):
    """A NaN or an infinity of one token reaches that token's row only; one of
    the weight its feature only."""
    import torch
    x = rand((m, 256), 1)
    x[1, 5], x[2, 200] = float("nan"), float("inf")
    w = rand((130, 256), 2)
    w[7, 3] = float("nan")
    y = nrp.fp8_linear(x.bfloat16().cuda(), nrp.fp8_quantize(w.cuda(), 128)).float().cpu()
    bad = torch.zeros(m, 130, dtype=torch.bool)
    bad[1:3] = True
    bad[:, 7] = True
    assert torch.equal(y.isnan(), bad) and y[~bad].isfinite().all()


def test_empty_and_shapes(nrp):
    import torch
    w = nrp.fp8_quantize(rand((48, 64), 2).cuda(), 128)
    assert nrp.fp8_linear(torch.zeros(0, 64, device="cuda"), w).shape == (0, 48)
    assert nrp.fp8_linear_input_grad(torch.zeros(2, 0, 48, device="cuda"), w).shape == (2, 0, 64)
    x = rand((2, 3, 64), 5).bfloat16().cuda()
    y = nrp.fp8_linear(x, w)
    assert y.shape == (2, 3, 48)
    assert torch.equal(y.reshape(6, 48), nrp.fp8_linear(x.reshape(6, 64), w))
    dw, db = nrp.fp8_linear_weight_grad(torch.zeros(0, 48, device="cuda", dtype=torch.bfloat16),
                                        nrp.fp8_quantize(torch.zeros(0, 64, device="cuda")),
                                        bias=True)
    assert (dw == 0).all() and dw.shape == (48, 64) and (db == 0).all()


# ---------------------------------------------------------- weight gradient
@pytest.mark.parametrize("m,k,n", [(1, 16, 8), (14, 128, 256), (63, 144, 264), (64, 1024, 1024),
                                   (65, 400, 1000), (129, 128, 24), (749, 512, 512),
                                   (1000, 1040, 504), (2500, 256, 256),
                                   # one CTA per tile; more k tiles than 8-column chunks
                                   (1, 1040, 2504), (515, 2320, 2000), (70, 4240, 264)])
@pytest.mark.parametrize("dtype,bias", [("f32", True), ("f32", False), ("bf16", True)])
def test_weight_grad(nrp, m, k, n, dtype, bias):
    import torch
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    dy = (rand((m, n), 1, 1e-3) * torch.exp2(rand((m, 1), 3) * 2)).bfloat16()
    q = nrp.fp8_quantize((rand((m, k), 2) * torch.exp2(rand((m, 1), 4) * 3)).bfloat16().cuda())
    guard = torch.full((n + 1, k), 5.0, dtype=dt, device="cuda")
    dw, db = nrp.fp8_linear_weight_grad(dy.cuda(), q, bias=bias, dtype=dt, out=guard[:n])
    assert (guard[n] == 5).all()
    d, x = dy.double(), values(q)
    ref = d.t() @ x
    tol = (d.abs().t() @ x.abs()) * (m + m / 16 + 16) * 2.0 ** -23
    close(dw, ref, tol + ref.abs() * half_step(dt))
    assert (db is not None) == bias
    if bias:
        ref = d.sum(0)
        close(db, ref, d.abs().sum(0) * (m + 16) * U + ref.abs() * half_step(dt))
    nrp.Context.default().check()


def test_weight_grad_is_a_derivative(nrp):
    """<dw, V> equals the change of sum dy * (x~ . w^T) along V (linear in w),
    and <dx, V> that along an input V."""
    import torch
    m, k, n = 333, 272, 144
    dy = rand((m, n), 1).bfloat16()
    q = nrp.fp8_quantize(rand((m, k), 2).cuda())
    w = nrp.fp8_quantize(rand((n, k), 3).cuda(), 128)
    dw, _ = nrp.fp8_linear_weight_grad(dy.cuda(), q)
    v = rand((n, k), 4).double()
    loss = lambda x, ww: (dy.double() * (x @ ww.t())).sum()  # noqa: E731
    x, wv = values(q), values(w)
    diff = (loss(x, wv + v) - loss(x, wv - v)) / 2
    size = ((dy.double().abs().t() @ x.abs()) * v.abs()).sum() * (m + m / 16 + 16) * 2.0 ** -23
    assert abs(float((dw.double().cpu() * v).sum() - diff)) <= float(size)
    g = nrp.fp8_quantize(dy.float().cuda())  # the gradient as the call sees it
    dx = nrp.fp8_linear_input_grad(g, w, dtype=torch.float32)
    v, gv = rand((m, k), 5).double(), values(g)
    diff = ((gv * ((x + v) @ wv.t())).sum() - (gv * ((x - v) @ wv.t())).sum()) / 2
    size = (product_tol(gv, wv, n, gv @ wv, torch.float32) * v.abs()).sum()
    assert abs(float((dx.double().cpu() * v).sum() - diff)) <= float(size)


def device_values(q):
    """float64 values of an Fp8Tensor on the device."""
    s = q.scales.double().repeat_interleave(q.block_rows, 0)[:q.codes.shape[0]]
    return q.codes.double() * s.repeat_interleave(128, 1)[:, :q.codes.shape[1]]


@pytest.mark.parametrize("m,k,n", [(16000, 1024, 4096), (5000, 1024, 1024), (3000, 2048, 1040),
                                   (16000, 144, 256), (12500, 512, 1024)])
def test_long_sums_and_repeats(nrp, m, k, n):
    """Many turns of the kernels' stage rings and many waves of tiles: each
    direction against 64 bits on the device, and twenty times the same bits
    (a stage handed back too early shows in some of them only)."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(m)
    x = torch.randn(m, k, device="cuda", generator=g).mul_(
        torch.exp2(torch.randn(m, 1, device="cuda", generator=g) * 3)).bfloat16()
    dy = torch.randn(m, n, device="cuda", generator=g).mul_(1e-3).bfloat16()
    w = nrp.fp8_quantize(torch.randn(n, k, device="cuda", generator=g) / math.sqrt(k), 128)
    xq, gq = nrp.fp8_quantize(x), nrp.fp8_quantize(dy)
    runs = {
        "linear": lambda: [nrp.fp8_linear(xq, w, dtype=torch.float32)],
        "input_grad": lambda: [nrp.fp8_linear_input_grad(gq, w, dtype=torch.float32)],
        "weight_grad": lambda: list(nrp.fp8_linear_weight_grad(dy, xq, bias=True)),
    }
    first = {name: f() for name, f in runs.items()}
    for _ in range(20):
        for name, f in runs.items():
            assert all(torch.equal(a, b) for a, b in zip(f(), first[name])), name
    nrp.Context.default().check()
    xv, wv, gv, d = device_values(xq), device_values(w), device_values(gq), dy.double()

    def check(got, a, b, chain):
        ref, size = a @ b, a.abs() @ b.abs()
        off = (got.double() - ref).abs()
        assert (off <= size * chain + ref.abs() * U).all(), float((off / size).max())

    check(first["linear"][0], xv, wv.t(), 132 * 2.0 ** -23 + (k // 128 + 4) * U)
    check(first["input_grad"][0], gv, wv, 132 * 2.0 ** -23 + (n // 128 + 4) * U)
    check(first["weight_grad"][0], d.t(), xv, (m + m / 16 + 16) * 2.0 ** -23)
    off = (first["weight_grad"][1].double() - d.sum(0)).abs()
    assert (off <= d.abs().sum(0) * (m + 16) * U).all()


@pytest.mark.parametrize("m,k,n", [(33, 1024, 1024), (64, 4096, 1024), (100, 1040, 200),
                                   (129, 2176, 1040), (200, 4224, 136), (600, 4096, 1024),
                                   (896, 2064, 1000), (1100, 4096, 1024), (1100, 2048, 512),
                                   (200, 4096, 640)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_shared_reductions(nrp, m, k, n, dtype):
    """Few tiles and a long reduction, which several CTAs share: the rows,
    columns and blocks at the ends, the bias added once, the same bits in every
    run, and nothing written behind the last row."""
    import torch
    dt = {"bf16": torch.bfloat16, "f32": torch.float32}[dtype]
    u = 2.0 ** -8 if dt == torch.bfloat16 else U
    g = torch.Generator(device="cuda").manual_seed(m + k)
    x = nrp.fp8_quantize(torch.randn(m, k, device="cuda", generator=g))
    w = nrp.fp8_quantize(torch.randn(n, k, device="cuda", generator=g) / math.sqrt(k), 128)
    bias = torch.randn(n, device="cuda", generator=g).to(dt)
    # the same reduction for the input's gradient: w [k, n] there
    n16 = n // 16 * 16
    wt = nrp.fp8_quantize(torch.randn(k, n16, device="cuda", generator=g) / math.sqrt(k), 128)
    held = torch.full((m + 1, n), 7.0, device="cuda", dtype=dt)
    y = nrp.fp8_linear(x, w, bias, dtype=dt, out=held[:m])
    dx = nrp.fp8_linear_input_grad(x, wt, dtype=dt)
    for _ in range(5):
        assert torch.equal(nrp.fp8_linear(x, w, bias, dtype=dt), y)
        assert torch.equal(nrp.fp8_linear_input_grad(x, wt, dtype=dt), dx)
    assert (held[m] == 7).all()
    xv = device_values(x)
    for got, b, add in ((y, device_values(w).t(), bias.double()), (dx, device_values(wt), None)):
        ref, size = xv @ b, xv.abs() @ b.abs()
        if add is not None:
            ref, size = ref + add, size + add.abs()
        off = (got.double() - ref).abs()
        assert (off <= size * (132 * 2.0 ** -23 + (k // 128 + 5) * U) + ref.abs() * u).all()


@pytest.mark.parametrize("m,k,n", [(5000, 768, 768), (12000, 208, 488), (1500, 80, 1656),
                                   (400, 512, 512), (9000, 560, 120), (700, 1536, 1024),
                                   (450, 144, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_shared_tokens(nrp, m, k, n, dtype):
    """Weight gradients whose tiles' tokens 2 to 8 CTAs share, odd numbers of
    them too, in every tile width: against 64 bits, five times the same bits."""
    import torch
    dt = {"bf16": torch.bfloat16, "f32": torch.float32}[dtype]
    u = 2.0 ** -8 if dt == torch.bfloat16 else U
    g = torch.Generator(device="cuda").manual_seed(m)
    xq = nrp.fp8_quantize(torch.randn(m, k, device="cuda", generator=g))
    dy = torch.randn(m, n, device="cuda", generator=g).bfloat16()
    dw, db = nrp.fp8_linear_weight_grad(dy, xq, bias=True, dtype=dt)
    for _ in range(5):
        a, b = nrp.fp8_linear_weight_grad(dy, xq, bias=True, dtype=dt)
        assert torch.equal(a, dw) and torch.equal(b, db)
    nrp.Context.default().check()
    xv, d = device_values(xq), dy.double()
    ref, size = d.t() @ xv, d.t().abs() @ xv.abs()
    off = (dw.double() - ref).abs()
    assert (off <= size * (m + m / 16 + 16) * 2.0 ** -23 + ref.abs() * u).all()
    off = (db.double() - d.sum(0)).abs()
    assert (off <= d.abs().sum(0) * (m + 16) * U + d.sum(0).abs() * u).all()


def test_repeatable(nrp):
    """Two calls on the same inputs give the same bits."""
    import torch
    for m in (5, 200, 1500):
        x = rand((m, 512), 1).bfloat16().cuda()
        w = nrp.fp8_quantize(rand((512, 512), 2).cuda(), 128)
        q = nrp.fp8_quantize(x)
        assert torch.equal(nrp.fp8_linear(x, w), nrp.fp8_linear(x, w))
        assert torch.equal(nrp.fp8_linear_input_grad(x, w), nrp.fp8_linear_input_grad(x, w))
        a, b = (nrp.fp8_linear_weight_grad(x, q, bias=True) for _ in range(2))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_python_refusals_on_device(nrp):
    import torch
    w = nrp.fp8_quantize(rand((64, 64), 2).cuda(), 128)
    x = rand((4, 64), 1).cuda()
    q = nrp.fp8_quantize(x)
    cases = [
        lambda: nrp.fp8_quantize(x.t()),                              # not contiguous
        lambda: nrp.fp8_quantize(x[:, :40].contiguous()),             # 40 columns
        lambda: nrp.fp8_quantize(x.half()),
        lambda: nrp.fp8_quantize(x, 64),
        lambda: nrp.fp8_quantize(x.reshape(-1)[1:49].reshape(3, 16)),  # 4-byte aligned
        lambda: nrp.fp8_linear(x, q),                                 # 1 x 128 weight blocks
        lambda: nrp.fp8_linear(rand((4, 48), 1).cuda(), w),
        lambda: nrp.fp8_linear(x, w, dtype=torch.bfloat16),           # f32 in, bf16 out
        lambda: nrp.fp8_linear(x, w, torch.zeros(63, device="cuda")),
        lambda: nrp.fp8_linear(x, w, torch.zeros(64, device="cuda").bfloat16()),
        lambda: nrp.fp8_linear(q, w, codes=q),
        lambda: nrp.fp8_linear(x, w, out=torch.zeros(4, 63, device="cuda")),
        lambda: nrp.fp8_linear(x.cpu(), w),
        lambda: nrp.fp8_linear(nrp.Fp8Tensor(q.codes, q.scales[:3], 1), w),
        lambda: nrp.fp8_linear_weight_grad(x, q),                     # dy must be bf16
        lambda: nrp.fp8_linear_weight_grad(x.bfloat16()[:3], q),
        lambda: nrp.fp8_linear_weight_grad(rand((4, 36), 1).bfloat16().cuda(), q),
    ]
    for i, c in enumerate(cases):
        with pytest.raises(nrp.NrpError):
            c()
            pytest.fail(f"case {i} was not refused")


# ------------------------------------------------- streams, graphs, together
def test_other_stream_and_graphs(nrp):
    """A side stream, and two captured graphs that are replayed in turn with
    new inputs, give what eager calls give."""
    import torch
    w = nrp.fp8_quantize(rand((256, 384), 2).cuda(), 128)
    x = [rand((m, 384), m).bfloat16().cuda() for m in (14, 300)]
    dy = [rand((m, 256), m + 1).bfloat16().cuda() for m in (14, 300)]
    gamma, beta = rand((384,), 5).cuda(), rand((384,), 6).cuda()

    def step(x, dy):
        h, mean, rstd = nrp.layer_norm(x, gamma, beta)
        hq = nrp.fp8_quantize(h)
        y = nrp.fp8_linear(hq, w)
        dh = nrp.fp8_linear_input_grad(dy, w)
        dw, db = nrp.fp8_linear_weight_grad(dy, hq, bias=True)
        return (y, dw, db, *nrp.layer_norm_backward(dh, nrp.fp8_quantize(x), mean, rstd, gamma))

    ref = [step(a, b) for a, b in zip(x, dy)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x[1], dy[1])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ref[1]))
    graphs, ins, outs = [], [], []
    for i in range(2):
        a, b = torch.zeros_like(x[i]), torch.zeros_like(dy[i])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = step(a, b)
        graphs.append(g), ins.append((a, b)), outs.append(o)
    for rep in range(2):
        for i in range(2):
            ins[i][0].copy_(x[i] * (1 + rep)), ins[i][1].copy_(dy[i])
            graphs[i].replay()
        for i in range(2):
            want = step(x[i] * (1 + rep), dy[i])
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want))
    nrp.Context.default().check()


def test_training_step_together(nrp):
    """LayerNorm -> 8-bit linear and back, as a fine-tuning step runs it: every
    gradient against the 64-bit formulas on the values the 8-bit operands
    stand for, within the sum of the single operators' tolerances (a bf16
    rounding of h, dh and dx, 2^-8 each, and one e4m3 rounding of dy, 2^-4,
    where the reference keeps it)."""
    import torch
    m, k, n = 500, 384, 640
    x = rand((m, k), 1).bfloat16()
    gamma, beta = 1 + 0.1 * rand((k,), 2), 0.1 * rand((k,), 3)
    bias = rand((n,), 4).bfloat16()
    dy = rand((m, n), 5, 1e-3).bfloat16()
    w = nrp.fp8_quantize(rand((n, k), 6).cuda() / math.sqrt(k), 128)
    h, mean, rstd = nrp.layer_norm(x.cuda(), gamma.cuda(), beta.cuda())
    hq = nrp.fp8_quantize(h)
    y = nrp.fp8_linear(hq, w, bias.cuda())
    xq = nrp.fp8_quantize(x.cuda())
    gq = nrp.Fp8Tensor(torch.empty((m, n), dtype=torch.float8_e4m3fn, device="cuda"),
                       torch.empty((m, n // 128), device="cuda"), 1)
    dh = nrp.fp8_linear_input_grad(dy.cuda(), w, codes=gq)
    dw, db = nrp.fp8_linear_weight_grad(dy.cuda(), hq, bias=True)
    dx, dgamma, dbeta = nrp.layer_norm_backward(dh, xq, mean, rstd, gamma.cuda())
    nrp.Context.default().check()
    wv, hv, xv, gv = values(w), values(hq), values(xq), values(gq)
    # each operator on the operands it was given
    ref = hv @ wv.t()
    close(y, ref + bias.double(), product_tol(hv, wv.t(), k, ref, torch.float32)
          + (ref + bias.double()).abs() * (2.0 ** -8 + U))
    close(dh, gv @ wv, product_tol(gv, wv, n, gv @ wv, torch.bfloat16))
    # the checkpoint is within one e4m3 rounding of h: 2^-4 of the value, or
    # half of the smallest step, 2^-10 of the block's scale
    hd = h.double().cpu()
    tiny = hq.scales.cpu().double().repeat_interleave(128, 1)[:, :k] * 2.0 ** -10
    assert ((hv - hd).abs() <= hd.abs() * 2.0 ** -4 + tiny).all()
    # end to end: the gradients of sum dy * linear(norm(x)) by differences, on
    # the exact chain with the quantised x and dy in place
    mu, rs = mean.double().cpu()[:, None], rstd.double().cpu()[:, None]
    u = (xv - mu) * rs
    dhd = dh.double().cpu()
    g = dhd * gamma.double()
    dx_ref = rs * (g - g.mean(1, keepdim=True) - u * (g * u).mean(1, keepdim=True))
    size = rs * (g.abs() + g.abs().mean(1, keepdim=True)
                 + u.abs() * (g * u).abs().mean(1, keepdim=True))
    close(dx, dx_ref, size * 40 * U + dx_ref.abs() * 2.0 ** -8)
    for got, want in ((dgamma, dhd * u), (dbeta, dhd)):
        close(got, want.sum(0), want.abs().sum(0) * 100 * U)
    d = dy.double()
    close(dw, d.t() @ hv, (d.abs().t() @ hv.abs()) * (m + m / 16 + 16) * 2.0 ** -23)
    close(db, d.sum(0), d.abs().sum(0) * (m + 16) * U)
