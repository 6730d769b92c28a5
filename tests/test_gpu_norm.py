"""LayerNorm forward and backward on the device against 64-bit forms.

Tolerances, u = 2^-24 (half a step of f32).  A row sum of C values is a chain
of n = ceil(C / 32) + 8 additions at most for rows held by a warp, and
ceil(C / 256) + 16 in the wide kernels: relative to the sum of magnitudes it is
off by n u.  The mean is off by dm = (n + 2) u mean|x|; rstd, from a sum of
squares, by dr = (n + 8) u relative.  y = (x - mean) rstd gamma + beta has
three more roundings.  The backward's u = (x - mean) rstd has two roundings of
the difference, its row means n additions.  dgamma and dbeta are chains of
rows / (8 parts) + 8 + parts / 8 + 8 additions, parts <= 296.  Outputs in bf16
add 2^-8 of the value."""
import math

import pytest

from __graft_entry__ import load_package

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SHAPES = [(1, 1), (1, 8), (3, 31), (5, 32), (14, 512), (7, 200), (9, 256), (33, 257), (8, 264),
          (40, 1000), (100, 1024), (3, 1025), (17, 2048), (5, 2056), (11, 5000), (749, 512),
          (2500, 80), (3000, 1024)]


@pytest.fixture(scope="module")
def nrp():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return load_package()


def rand(shape, seed, scale=1.0):
    import torch
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale


def close(got, ref, tol):
    d = (got.double().cpu() - ref).abs()
    bad = ~(d <= tol)
    assert not bad.any(), (int(bad.sum()), float((d / tol.clamp(min=1e-300)).max()))


def chain(cols):
    return -(-cols // 32) + 8 if cols <= 2048 else -(-cols // 256) + 16


def stats(x, eps=1e-5):
    mean = x.mean(1, keepdim=True)
    return mean, ((x - mean).square().mean(1, keepdim=True) + eps) ** -0.5


def inputs(rows, cols, dtype, offset=0.5):
    import torch
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    x = (rand((rows, cols), rows * 7 + cols) * torch.exp2(rand((rows, 1), 1)) + offset).to(dt)
    return x, 1 + 0.2 * rand((cols,), 2), 0.1 * rand((cols,), 3), dt


def forward_tol(x, gamma, beta, y, cols, dt):
    n = chain(cols)
    mean, rstd = stats(x)
    dm = (n + 2) * U * x.abs().mean(1, keepdim=True)
    u = (x - mean) * rstd
    return (gamma.abs() * (rstd * dm + u.abs() * (n + 12) * U) + (beta.abs() + y.abs()) * 2 * U
            + y.abs() * half_step(dt)), dm, (n + 8) * U


def half_step(dtype):
    import torch
    return torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(nrp, rows, cols, dtype):
    x, gamma, beta, dt = inputs(rows, cols, dtype)
    y, mean, rstd = nrp.layer_norm(x.cuda(), gamma.cuda(), beta.cuda())
    xd, g, b = x.double(), gamma.double(), beta.double()
    m, r = stats(xd)
    ref = (xd - m) * r * g + b
    tol, dm, dr = forward_tol(xd, g, b, ref, cols, dt)
    close(y, ref, tol)
    close(mean, m[:, 0], dm[:, 0])
    # a mean off by dm adds dm^2 to the variance
    close(rstd, r[:, 0], r[:, 0] * (dr + (r * dm).square()[:, 0]))
    z = x.cuda()  # in place
    assert nrp.layer_norm(z, gamma.cuda(), beta.cuda(), out=z)[0] is z
    assert (z == y).all()


@pytest.mark.parametrize("cols", [64, 200, 1024, 3001])
def test_forward_large_mean_and_constant_rows(nrp, cols):
    """A mean of 1000 spreads: the variance about the mean keeps its digits
    (sum of squares minus square of the sum would not); a constant row is
    beta; the largest and non-finite values stay in their rows."""
    import torch
    x = rand((6, cols), 1) + 1000
    x[1] = 4.0
    x[2, 0] = float("nan")
    x[3, 1] = float("inf")
    gamma, beta = 1 + 0.1 * rand((cols,), 2), rand((cols,), 3)
    y, mean, rstd = nrp.layer_norm(x.cuda(), gamma.cuda(), beta.cuda())
    assert torch.equal(y[1].cpu(), beta) and y[2].isnan().all() and y[3].isnan().all()
    for row in (0, 4, 5):
        xd = x[row:row + 1].double()
        m, r = stats(xd)
        ref = (xd - m) * r * gamma.double() + beta.double()
        tol, dm, dr = forward_tol(xd, gamma.double(), beta.double(), ref, cols, torch.float32)
        close(y[row:row + 1], ref, tol + gamma.double().abs() * (r * dm).square() * 4)


def grads(x, mean, rstd, dy, gamma):
    u = (x - mean) * rstd
    g = dy * gamma
    c1, c2 = g.mean(1, keepdim=True), (g * u).mean(1, keepdim=True)
    size = rstd * (g.abs() + g.abs().mean(1, keepdim=True)
                   + u.abs() * (g * u).abs().mean(1, keepdim=True))
    # u's own error: two roundings of |x - mean| and the subtraction's of |x|
    return rstd * (g - c1 - u * c2), (dy * u).sum(0), dy.sum(0), u, size


@pytest.mark.parametrize("kind", ["bf16", "f32", "fp8-bf16", "fp8-f32"])
@pytest.mark.parametrize("rows,cols", SHAPES + [(6, 16), (50, 144), (20, 4096)])
def test_backward(nrp, rows, cols, kind):
    import torch
    if kind.startswith("fp8") and cols % 16:
        pytest.skip("codes have rows of 16 bytes")
    x, gamma, _, dt = inputs(rows, cols, kind[-4:].lstrip("-"))
    dy = rand((rows, cols), 4, 1e-2).to(dt)
    _, mean, rstd = nrp.layer_norm(x.cuda(), gamma.cuda(), torch.zeros(cols).cuda())
    xin = x.cuda()
    xd = x.double()
    if kind.startswith("fp8"):
        xin = nrp.fp8_quantize(x.cuda())
        xd = nrp.fp8_dequantize(xin, torch.float32).cpu().double()
    guard = torch.full((rows + 1, cols), 9.0, dtype=dt, device="cuda")
    dx, dgamma, dbeta = nrp.layer_norm_backward(dy.cuda(), xin, mean, rstd, gamma.cuda(),
                                                out=guard[:rows])
    assert (guard[rows] == 9).all()
    m, r = mean.double().cpu()[:, None], rstd.double().cpu()[:, None]
    dxr, dgr, dbr, u, size = grads(xd, m, r, dy.double(), gamma.double())
    n = chain(cols)
    close(dx, dxr, size * (n + 12) * U + dxr.abs() * half_step(dt))
    parts = min(-(-rows // 8), 296)
    depth = -(-rows // (8 * parts)) + 8 + -(-parts // 8) + 8 + 4
    close(dgamma, dgr, (dy.double() * u).abs().sum(0) * depth * U)
    close(dbeta, dbr, dy.double().abs().sum(0) * depth * U)


@pytest.mark.parametrize("cols", [48, 100, 1500])
def test_backward_is_a_derivative(nrp, cols):
    """dx, dgamma and dbeta against central differences of sum dy * norm(x) in
    64 bits (step 1e-4: their own error is of the order 1e-8 of the change)."""
    import torch
    rows = 37
    x, gamma, beta, _ = inputs(rows, cols, "f32")
    dy = rand((rows, cols), 4)
    _, mean, rstd = nrp.layer_norm(x.cuda(), gamma.cuda(), beta.cuda())
    dx, dgamma, dbeta = nrp.layer_norm_backward(dy.cuda(), x.cuda(), mean, rstd, gamma.cuda())
    vx, vg, vb = (rand(t.shape, 10 + i).double() for i, t in enumerate((x, gamma, beta)))

    def loss(t):
        xd = x.double() + t * vx
        m, r = stats(xd)
        return (dy.double() * ((xd - m) * r * (gamma.double() + t * vg) + beta.double() + t * vb)).sum()

    h = 1e-4
    diff = float(loss(h) - loss(-h)) / (2 * h)
    got = sum(float((a.double().cpu() * b).sum()) for a, b in ((dx, vx), (dgamma, vg), (dbeta, vb)))
    size = sum(float((a.double().cpu() * b).abs().sum())
               for a, b in ((dx, vx), (dgamma, vg), (dbeta, vb)))
    assert abs(got - diff) <= 1e-5 * size


def test_unaligned_and_empty(nrp):
    """Views that start off 16 bytes take the element-wise kernels; no rows
    give zero dgamma and dbeta."""
    import torch
    rows, cols = 13, 64
    for dt in (torch.float32, torch.bfloat16):
        flat = rand((rows * cols + 1,), 1).to(dt).cuda()
        x = flat[1:].reshape(rows, cols)
        gamma, beta = rand((cols + 1,), 2).cuda()[1:], rand((cols,), 3).cuda()
        y, mean, rstd = nrp.layer_norm(x, gamma, beta)
        xd, g, b = x.double().cpu(), gamma.double().cpu(), beta.double().cpu()
        m, r = stats(xd)
        ref = (xd - m) * r * g + b
        close(y, ref, forward_tol(xd, g, b, ref, cols, dt)[0])
        a = nrp.layer_norm_backward(x, x, mean, rstd, gamma)
        b = nrp.layer_norm_backward(x.clone(), x.clone(), mean, rstd, gamma.clone())
        tol = a[0].double().abs().max() * 40 * U + a[0].double().abs() * half_step(dt)
        assert ((a[0].double() - b[0].double()).abs() <= 2 * tol).all()
    e = torch.zeros(0, cols, device="cuda")
    s = torch.zeros(0, device="cuda")
    assert nrp.layer_norm(e, gamma, beta)[0].shape == (0, cols)
    dx, dg, db = nrp.layer_norm_backward(e, e, s, s, gamma)
    assert dx.shape == (0, cols) and (dg == 0).all() and (db == 0).all()


def test_abi_without_parameter_gradients(nrp):
    """dgamma and dbeta NULL: dx alone, no workspace; mean and rstd NULL
    forward."""
    import torch
    rows, cols = 20, 96
    x, dy = rand((rows, cols), 1).cuda(), rand((rows, cols), 2).cuda()
    gamma, beta = rand((cols,), 3).cuda(), rand((cols,), 4).cuda()
    y, mean, rstd = nrp.layer_norm(x, gamma, beta)
    ctx, st = nrp.Context.default(), torch.cuda.current_stream().cuda_stream
    z = torch.empty_like(x)
    assert nrp.lib().nrp_layer_norm(ctx.handle, st, nrp.F32, x.data_ptr(), rows, cols,
                                    gamma.data_ptr(), beta.data_ptr(), 1e-5, z.data_ptr(), None,
                                    None) == 0
    assert torch.equal(y, z)
    dx = torch.empty_like(x)
    assert nrp.lib().nrp_layer_norm_backward(
        ctx.handle, st, nrp.F32, x.data_ptr(), None, dy.data_ptr(), mean.data_ptr(),
        rstd.data_ptr(), gamma.data_ptr(), rows, cols, dx.data_ptr(), None, None, None, 0) == 0
    assert torch.equal(dx, nrp.layer_norm_backward(dy, x, mean, rstd, gamma)[0])


def test_python_refusals_on_device(nrp):
    import torch
    x, v = torch.zeros(4, 64, device="cuda"), torch.ones(64, device="cuda")
    s = torch.ones(4, device="cuda")
    q = nrp.fp8_quantize(x)
    cases = [
        lambda: nrp.layer_norm(x, v[:63], v),
        lambda: nrp.layer_norm(x, v.bfloat16(), v),
        lambda: nrp.layer_norm(x, v, v.cpu()),
        lambda: nrp.layer_norm(x.half(), v, v),
        lambda: nrp.layer_norm(x[:, ::2], v[:32], v[:32]),
        lambda: nrp.layer_norm(x, v, v, eps=-1.0),
        lambda: nrp.layer_norm(x, v, v, out=x[:3]),
        lambda: nrp.layer_norm_backward(x, x.bfloat16(), s, s, v),
        lambda: nrp.layer_norm_backward(x, x[:3], s, s, v),
        lambda: nrp.layer_norm_backward(x, x, s[:3], s, v),
        lambda: nrp.layer_norm_backward(x, nrp.Fp8Tensor(q.codes, q.scales, 128), s, s, v),
    ]
    for i, c in enumerate(cases):
        with pytest.raises(nrp.NrpError):
            c()
            pytest.fail(f"case {i} was not refused")
