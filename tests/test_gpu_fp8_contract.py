"""What the 8-bit operators' and the LayerNorm's documentation allows beyond the
ordinary calls: the ends of the sizes, scales of every f32 value, rows of very
large values, profiling from several threads, autograd's view of the outputs.

u = 2^-24 is half a step of f32."""
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


def values(q):
    """float64 values of an Fp8Tensor on the CPU."""
    c, s = q.codes.cpu().double(), q.scales.cpu().double()
    s = s.repeat_interleave(q.block_rows, 0)[:c.shape[0]].repeat_interleave(128, 1)
    return c * s[:, :c.shape[1]]


def bf16(v):
    """float64 numpy values rounded once to bf16 (torch's conversion goes through
    f32), as float64."""
    _, e = np.frexp(v)
    step = np.exp2(np.maximum(e - 8, -133).astype(np.float64))
    return np.where(np.isfinite(v), np.round(v / step) * step, v)


def scales_on_ties():
    """Scales and codes whose product, rounded to f32 first, lands on a tie of bf16
    that it is not, with the other scales of the same draw."""
    g = np.random.default_rng(5)
    s = (g.integers(2 ** 23, 2 ** 24, 1 << 22) * 2.0 ** -30).astype(np.float32)
    found = []
    for c in (9.0, 11.0, 13.0, 15.0):
        v = s.astype(np.float64) * c
        off = bf16(v) != bf16(v.astype(np.float32).astype(np.float64))
        found += [(float(x), c) for x in s[off][:16]]
    assert len(found) == 64
    return found


def test_values_are_rounded_once(nrp):
    """Codes times scales of 24 bits in bf16, by fp8_dequantize and on the weight
    gradient's way into its products (dy the identity: dw is x^)."""
    import torch
    pairs = scales_on_ties()
    q = nrp.Fp8Tensor(codes((64, 128), 448.0, 1), torch.tensor([[s] for s, _ in pairs]).cuda(), 1)
    q.codes[:, 0] = torch.tensor([c for _, c in pairs]).to(torch.float8_e4m3fn).cuda()
    q.scales[5:9] *= -1
    want = torch.from_numpy(bf16(values(q).numpy()))
    assert not torch.equal(values(q).float().bfloat16().double(), want)  # (through f32)
    assert torch.equal(nrp.fp8_dequantize(q).double().cpu(), want)
    dw, _ = nrp.fp8_linear_weight_grad(torch.eye(64, device="cuda", dtype=torch.bfloat16), q)
    assert torch.equal(dw.double().cpu(), want)


@pytest.mark.parametrize("m,k,n", [(3, 16, 8), (70, 272, 264), (515, 400, 2000), (749, 1024, 1024),
                                   (2500, 256, 256), (5000, 560, 120), (1, 1040, 2504)])
def test_weight_gradient_of_any_scales(nrp, m, k, n):
    """Scales of any size and sign beside the quantiser's in one tile, a zero one, and
    a NaN code that reaches its column only: against the products of the values
    rounded to bf16, within (m + m/16 + 16) additions cut at 2^-23."""
    import torch
    g = torch.Generator().manual_seed(m)
    blocks = -(-k // 128)
    scales = torch.randn(m, blocks, generator=g) * torch.exp2(torch.randn(m, blocks, generator=g) * 6)
    tame = torch.rand(m, blocks, generator=g) < 0.5
    scales[tame] = torch.exp2(torch.randint(-20, 20, (m, blocks), generator=g).float())[tame]
    scales[m // 2] = 0.0
    q = nrp.Fp8Tensor(codes((m, k), 448.0, 2), scales.cuda(), 1)
    dy = (torch.randn(m, n, generator=g) * 1e-3).bfloat16()
    x, d = torch.from_numpy(bf16(values(q).numpy())), dy.double()
    ref, size = d.t() @ x, d.abs().t() @ x.abs()
    tol = size * (m + m / 16 + 16) * 2.0 ** -23
    for bias in (False, True):
        dw, _ = nrp.fp8_linear_weight_grad(dy.cuda(), q, bias=bias)
        assert ((dw.double().cpu() - ref).abs() <= tol + ref.abs() * U).all()
    q.codes.view(torch.uint8)[m - 1, k - 3] = 0xFF
    q.codes.view(torch.uint8)[m - 1, 1] = 0x7F
    dw = nrp.fp8_linear_weight_grad(dy.cuda(), q)[0].cpu()
    bad = torch.zeros(k, dtype=torch.bool)
    bad[[k - 3, 1]] = True
    assert dw[:, bad].isnan().all()
    assert ((dw[:, ~bad].double() - ref[:, ~bad]).abs() <= (tol + ref.abs() * U)[:, ~bad]).all()
    nrp.Context.default().check()


def codes(shape, top, seed):
    """e4m3 codes of magnitude up to `top`, an eighth of them zeros."""
    import torch
    g = torch.Generator().manual_seed(seed)
    v = (torch.rand(shape, generator=g) * 2 - 1) * top
    v[torch.rand(shape, generator=g) < 0.125] = 0
    return v.to(torch.float8_e4m3fn).cuda()


# (exponents of x's and the weight's scales, largest code): products of scales
# above and below f32's range whose block sums lie in it, and one of each kind in
# range
FAR = [(100, 30, 2.0 ** -7), (64, 66, 2.0 ** -7), (119, 119, 0.0), (-80, -70, 448.0),
       (-117, -20, 448.0), (-20, -117, 448.0), (-117, -117, 448.0), (119, -110, 448.0),
       (-110, 119, 448.0)]


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("m", [3, 20, 40, 300])
def test_products_of_far_scales(nrp, m, trans):
    """Rows and blocks whose scales' product leaves f32's range beside ordinary
    ones.  Tolerance: as for other products 132 additions cut at 2^-23 within a
    block, here two f32 roundings of a block's sum and its addition, and half of the
    smallest f32 number for each of those."""
    import torch
    red, cols = 256 + 16, 192
    blocks = 3
    for ex, ew, top in FAR:
        x = nrp.Fp8Tensor(codes((m, red), top, 1), torch.ones(m, blocks, device="cuda"), 1)
        wshape = (red, cols) if trans else (cols, red)
        w = nrp.Fp8Tensor(codes(wshape, top, 2),
                          torch.ones([-(-n // 128) for n in wshape], device="cuda"), 128)
        x.scales[:, 1] = 2.0 ** ex  # the middle block of the reduction
        if trans:
            w.scales[1] = 2.0 ** ew
        else:
            w.scales[:, 1] = -(2.0 ** ew)
        x.scales[m // 2, 1] = 2.0 ** -ew  # one row's product is 1
        xv, wv = values(x), values(w) if trans else values(w).t()
        if abs(ex + ew) > 100:  # the far block by itself
            for t in (x.scales, w.scales):
                t[torch.where(t == 1)] = 0.0
            xv, wv = values(x), values(w) if trans else values(w).t()
        ref, size = xv @ wv, xv.abs() @ wv.abs()
        assert (size < 3e38).all()
        call = nrp.fp8_linear_input_grad if trans else nrp.fp8_linear
        y = call(x, w, dtype=torch.float32).double().cpu()
        tol = size * (132 * 2.0 ** -23 + 8 * U) + 3 * blocks * 2.0 ** -149
        assert ((y - ref).abs() <= tol).all(), (ex, ew, float(((y - ref).abs() / tol).max()))


@pytest.mark.parametrize("m", [3, 300])
def test_zero_and_non_finite_scales(nrp, m):
    """A zero scale gives zeros whatever the other's size, an infinite or NaN one
    reaches its row (or its 128 features) only."""
    import torch
    x = nrp.fp8_quantize(torch.ones(m, 256, device="cuda"))
    w = nrp.fp8_quantize(torch.ones(256, 256, device="cuda"), 128)
    w.scales.fill_(2.0 ** 119)
    x.scales.zero_()
    assert (nrp.fp8_linear(x, w) == 0).all() and (nrp.fp8_linear_input_grad(x, w) == 0).all()
    w.scales.fill_(1.0)
    x.scales.fill_(1.0)
    x.scales[1, 1] = float("inf")
    x.scales[2, 0] = float("nan")
    y = nrp.fp8_linear(x, w, dtype=torch.float32)
    assert (y[1] == float("inf")).all() and y[2].isnan().all()
    rest = torch.cat([y[:1], y[3:]])
    assert rest.isfinite().all()
    x.scales.fill_(1.0)
    w.scales[1, 0] = float("nan")
    y = nrp.fp8_linear(x, w)
    assert y[:, 128:].isnan().all() and y[:, :128].isfinite().all()


def test_norm_gradient_of_a_billion_columns(nrp):
    """One row whose dgamma and dbeta are more than 2^31 values together.  With
    mean and rstd given, dgamma = dy u is two f32 roundings of u and one of the
    product off, dbeta = dy exact."""
    import torch
    torch.cuda.empty_cache()
    cols = 2 ** 30 + 24
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(1, cols, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    dy = torch.empty_like(x).normal_(generator=g)
    gamma = torch.ones(cols, device="cuda")
    mean, rstd = torch.full((1,), 0.25, device="cuda"), torch.full((1,), 1.5, device="cuda")
    dx, dgamma, dbeta = nrp.layer_norm_backward(dy, x, mean, rstd, gamma)
    for at in (slice(0, 1 << 20), slice(2 ** 29, 2 ** 29 + (1 << 20)), slice(cols - (1 << 20), cols)):
        d, u = dy[0, at].double(), (x[0, at].double() - 0.25) * 1.5
        assert ((dgamma[at].double() - d * u).abs() <= 4 * U * (d * u).abs()).all()
        assert torch.equal(dbeta[at], dy[0, at].float())
        assert dx[0, at].isfinite().all()
    del x, dy, gamma, dx, dgamma, dbeta
    torch.cuda.empty_cache()


def test_threads_with_profiling(nrp):
    """Four threads on one context with the launch timing on, and a fifth that
    reads it: every launch is counted once, and the results stay the same."""
    import threading
    import torch
    ctx = nrp.Context(0)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(40, 512, device="cuda", generator=g).bfloat16()
    gamma, beta = torch.rand(512, device="cuda"), torch.rand(512, device="cuda")
    w = nrp.fp8_quantize(torch.randn(256, 512, device="cuda", generator=g), 128)
    want = nrp.fp8_linear(nrp.layer_norm(x, gamma, beta)[0], w)
    torch.cuda.synchronize()
    turns, threads, wrong = 60, 4, []

    def work():
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(turns):
                y = nrp.fp8_linear(nrp.layer_norm(x, gamma, beta, ctx=ctx)[0], w, ctx=ctx)
                st.synchronize()
                if not torch.equal(y, want):
                    wrong.append(y)

    ctx.profile_reset()
    ctx.profile(True)
    ts = [threading.Thread(target=work) for _ in range(threads)]
    for t in ts:
        t.start()
    while any(t.is_alive() for t in ts):
        ctx.profile_read()
    for t in ts:
        t.join()
    ctx.profile(False)
    read = ctx.profile_read()
    assert not wrong
    assert {k: n for k, (n, _) in read.items()} == {
        "layernorm": turns * threads, "fp8_quant": turns * threads, "gemm_fp8": turns * threads}
    ctx.check()


@pytest.mark.parametrize("rows,cols", [(20, 512), (3000, 64), (700, 112), (2500, 1024), (600, 784),
                                       (300, 2048), (50, 4096), (40, 6000)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shift", [0, 16])
def test_norm_gradient_of_codes_far_from_zero(nrp, rows, cols, dtype, shift):
    """x in 8 bits, its mean up to a thousand spreads or so large that mean * rstd
    passes f32: u = (code * scale - mean) * rstd has two roundings of the difference
    in every kernel (not of the mean), which dgamma = dy u shows where one row alone
    has gradients.  Kernels by elements: x shifted `shift` bytes off the allocation,
    dy and dx by an element."""
    import torch
    dt = {"bf16": torch.bfloat16, "f32": torch.float32}[dtype]
    g = torch.Generator(device="cuda").manual_seed(cols)
    blocks, one = -(-cols // 128), rows - 3

    def off(t):
        held = torch.zeros(t.numel() + 1, device="cuda", dtype=t.dtype)
        v = held[1:].view(t.shape) if shift else held[:-1].view(t.shape)
        return v.copy_(t)

    q = nrp.Fp8Tensor(codes((rows, cols), 448.0, 1),
                      torch.randn(rows, blocks, device="cuda", generator=g), 1)
    mean = torch.randn(rows, device="cuda", generator=g)
    rstd = torch.exp2(torch.randn(rows, device="cuda", generator=g))
    dy = torch.zeros(rows, cols, device="cuda", dtype=dt)
    dy[one] = torch.randn(cols, device="cuda", generator=g)
    dy = off(dy)
    gamma = torch.randn(cols, device="cuda", generator=g)
    even = torch.arange(cols, device="cuda") % 2 == 0
    for top, scale, mu, r in ((448.0, 0.7, 0.7 * 448.4, 1.3), (448.0, 2.0 ** 91, 448 * 2.0 ** 91,
                                                              2.0 ** 40)):
        q.codes[one] = torch.where(even & (scale < 1), 416.0, top).to(torch.float8_e4m3fn)
        q.scales[one], mean[one], rstd[one] = scale, mu, r
        dx, dg, db = nrp.layer_norm_backward(dy, q, mean, rstd, gamma, out=off(dy))
        x = q.codes[one].double() * q.scales[one].double().repeat_interleave(128)[:cols]
        r = rstd[one].double()
        u = (x - mean[one].double()) * r
        d = dy[one].double()
        assert ((dg.double() - d * u).abs() <= 4 * U * (d * u).abs()).all()
        assert torch.equal(db.double(), d)
        w = d * gamma.double()
        ref = r * (w - w.mean() - u * (w * u).mean())
        size = r * (w.abs() + w.abs().mean() + u.abs() * (w * u).abs().mean())
        chain = cols / 32 + 20 if cols <= 2048 else cols / 256 + 20
        assert ((dx[one].double() - ref).abs() <= size * chain * U
                + ref.abs() * torch.finfo(dt).eps / 2).all()
        dx[one] = 0
        assert (dx == 0).all()


@pytest.mark.parametrize("rows,cols", [(14, 64), (37, 256), (23, 512), (50, 1024), (9, 2048),
                                       (40, 77), (11, 300), (21, 999), (13, 1999), (700, 512),
                                       (12, 4096), (8, 3001), (10, 6000), (9, 5001)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_norm_of_very_large_values(nrp, rows, cols, dtype):
    """Rows whose sum of squares, or sum, passes f32's range beside ordinary ones: the
    largest finite values of both signs, a single large one, a constant row, with NaN
    and infinities in others.  Tolerances in u = 2^-24: a row's sums are chains of
    n = cols / 32 + 8 additions (over 2048 columns cols / 256 + 16), the mean off by
    dm = (n + 2) u mean|x|, rstd by (n + 8) u, y by those and three roundings; rstd
    by half of the smallest f32 number too."""
    import torch
    dt = {"bf16": torch.bfloat16, "f32": torch.float32}[dtype]
    g = torch.Generator().manual_seed(cols)
    x = torch.randn(rows, cols, generator=g).double()
    top = torch.finfo(dt).max
    x[1] *= 1e20
    x[2] = (torch.rand(cols, generator=g) * 2 - 1).double() * top
    x[3] *= 1e-3
    x[3, cols // 2] = 1e38
    x[4] = top
    x[5] = x[5] * 1e18 + 1e22
    x[6, 1] = float("inf")
    x[7, 0] = float("nan")
    x = x.to(dt)
    gamma, beta = 1 + 0.2 * torch.randn(cols, generator=g), 0.1 * torch.randn(cols, generator=g)
    y, mean, rstd = (t.double().cpu() for t in nrp.layer_norm(x.cuda(), gamma.cuda(), beta.cuda()))
    assert y[6:8].isnan().all() and mean[7].isnan() and rstd[7].isnan()
    keep = [r for r in range(rows) if r not in (6, 7)]
    xd, ga, be = x.double()[keep], gamma.double(), beta.double()
    m = xd.mean(1, keepdim=True)
    r = ((xd - m).square().mean(1, keepdim=True) + float(torch.tensor(1e-5))) ** -0.5
    n = cols / 32 + 8 if cols <= 2048 else cols / 256 + 16
    dm = (n + 2) * U * xd.abs().mean(1, keepdim=True)
    u = (xd - m) * r
    ref = u * ga + be
    dr = (n + 8) * U + (r * dm).square()
    assert ((mean[keep][:, None] - m).abs() <= dm).all()
    assert ((rstd[keep][:, None] - r).abs() <= r * dr + 2.0 ** -149).all()
    tol = (ga.abs() * (r * dm + u.abs() * ((n + 12) * U + dr)) + (be.abs() + ref.abs()) * 2 * U
           + ref.abs() * torch.finfo(dt).eps / 2)
    assert ((y[keep] - ref).abs() <= tol).all()
    z = x.cuda()  # in place
    nrp.layer_norm(z, gamma.cuda(), beta.cuda(), out=z)
    assert torch.equal(z.double().cpu()[keep], y[keep])
    # the gradients take such a row's statistics (within +-2^126 of its mean)
    s = [1, 3, 5]
    dy = torch.randn(3, cols, generator=g).to(dt)
    _, mean, rstd = nrp.layer_norm(x[s].cuda(), gamma.cuda(), beta.cuda())
    dg = nrp.layer_norm_backward(dy.cuda(), x[s].cuda(), mean, rstd, gamma.cuda())[1]
    u = (x[s].double() - mean.double().cpu()[:, None]) * rstd.double().cpu()[:, None]
    assert ((dg.double().cpu() - (dy.double() * u).sum(0)).abs()
            <= 23 * U * (dy.double() * u).abs().sum(0)).all()


def test_outputs_raise_their_version(nrp):
    """Every output of the caller's counts as written in place: autograd refuses a
    gradient that needs the value which was there."""
    import torch
    x = torch.randn(20, 256, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    v = torch.ones(256, device="cuda")
    w = nrp.fp8_quantize(torch.randn(128, 256, device="cuda"), 128)
    q = nrp.fp8_quantize(x)
    dy = torch.zeros(20, 128, device="cuda", dtype=torch.bfloat16)
    y = nrp.fp8_linear(x, w)
    _, mean, rstd = nrp.layer_norm(x, v, v)
    dw, db = nrp.fp8_linear_weight_grad(dy, q, bias=True)
    calls = [
        ([*q[:2]], lambda: nrp.fp8_quantize(x, out=q)),
        ([x], lambda: nrp.fp8_dequantize(q, torch.float32, out=x)),
        ([y, *q[:2]], lambda: nrp.fp8_linear(x, w, out=y, codes=q)),
        ([x], lambda: nrp.fp8_linear_input_grad(nrp.fp8_quantize(y), w, dtype=torch.float32, out=x)),
        ([dw, db], lambda: nrp.fp8_linear_weight_grad(dy, q, out=dw, bias_out=db)),
        ([x], lambda: nrp.layer_norm(x, v, v, out=x)),
        ([x], lambda: nrp.layer_norm_backward(torch.ones_like(x), q, mean, rstd, v, out=x)),
    ]
    for i, (outs, call) in enumerate(calls):
        before = [t._version for t in outs]
        call()
        assert [t._version for t in outs] == [n + 1 for n in before], i
    p = torch.ones(20, 256, device="cuda", requires_grad=True)
    loss = (p * x).sum()  # keeps x
    nrp.layer_norm(x, v, v, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():  # no version there
        z = torch.empty_like(x)
    assert nrp.layer_norm(x, v, v, out=z)[0] is z


def test_results_have_storages_of_their_own(nrp):
    """Codes and scales, mean and rstd, dgamma and dbeta: growing one in place leaves
    the other, and none holds more memory than its values."""
    import torch
    x = torch.randn(16, 256, device="cuda")
    v = torch.ones(256, device="cuda")
    q = nrp.fp8_quantize(x)
    _, mean, rstd = nrp.layer_norm(x, v, v)
    _, dg, db = nrp.layer_norm_backward(x, x, mean, rstd, v)
    for first, second in ((q.codes, q.scales), (mean, rstd), (dg, db)):
        for t in (first, second):
            assert t.storage_offset() == 0
            assert t.untyped_storage().nbytes() == t.numel() * t.element_size()
        keep = second.clone()
        n = first.numel()
        first.resize_(2 * n).view(torch.uint8)[n * first.element_size():] = 7
        assert torch.equal(second, keep)


@pytest.mark.parametrize("block_rows", [0, -1, 2, 2 ** 40, 2 ** 70, -2 ** 70, 1.0, None, "1"])
def test_block_rows_of_any_kind_are_refused(nrp, block_rows):
    """With the library's own error, also for an int past 64 bits."""
    import torch
    x = torch.zeros(4, 64, device="cuda")
    q = nrp.fp8_quantize(x)
    for call in (lambda: nrp.fp8_quantize(x, block_rows),
                 lambda: nrp.fp8_dequantize(q._replace(block_rows=block_rows))):
        with pytest.raises(nrp.NrpError):
            call()


@pytest.mark.parametrize("m,k,n", [(16000, 1024, 4096), (12500, 512, 1024), (4000, 1024, 1024),
                                   (16000, 144, 256), (8192, 400, 200)])
def test_weight_gradient_precision(nrp, m, k, n):
    """The gradients of many tokens as a whole.  A tensor-core addition is cut off by
    up to 2^-23 of the sum, 2^-24 on average and always towards zero; over a segment
    of 64 additions, whose partial sums grow like sqrt(j), these add up to 64 * 2/3 *
    2^-24 of the segment's sum, and segments, added with rounding, are independent:
    2.6e-6 of the norm.  (One chain of m / 16 additions is off by 8e-6 at 16000
    tokens.)  dbias: chains of m / 32 rounded additions, sqrt(m / 32 / 6) 2^-24 of
    the norm on average; twice that and eight more for the joins."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(m + n)
    q = nrp.fp8_quantize(torch.randn(m, k, device="cuda", generator=g))
    dy = torch.randn(m, n, device="cuda", generator=g).bfloat16()
    dw, db = nrp.fp8_linear_weight_grad(dy, q, bias=True)
    x = q.codes.double() * q.scales.double().repeat_interleave(128, 1)[:, :k]
    ref, d = dy.double().t() @ x, dy.double().sum(0)
    assert (dw.double() - ref).norm() <= 64 * 2 / 3 * U * ref.norm()
    assert (db.double() - d).norm() <= (2 * (m / 192) ** 0.5 + 8) * U * d.norm()


@pytest.mark.parametrize("rows,cols", [(20, 512), (3000, 64), (2500, 1024), (600, 784), (50, 4096),
                                       (40, 6000)])
def test_norm_gradient_of_a_nan_code(nrp, rows, cols):
    """A NaN code, or an infinite scale's block, reaches its row of dx and its columns
    of dgamma only."""
    import torch
    q = nrp.Fp8Tensor(codes((rows, cols), 448.0, 1),
                      torch.ones(rows, -(-cols // 128), device="cuda"), 1)
    g = torch.Generator(device="cuda").manual_seed(rows)
    dy = torch.randn(rows, cols, device="cuda", generator=g).bfloat16()
    mean = torch.randn(rows, device="cuda", generator=g)
    rstd = torch.rand(rows, device="cuda", generator=g) + 0.5
    gamma = torch.randn(cols, device="cuda", generator=g)
    q.codes.view(torch.uint8)[7, 5] = 0x7F
    q.codes.view(torch.uint8)[rows - 1, cols - 1] = 0xFF
    dx, dg, db = nrp.layer_norm_backward(dy, q, mean, rstd, gamma)
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[[7, rows - 1]] = True
    assert dx[bad].isnan().all() and dx[~bad].isfinite().all()
    bad = torch.zeros(cols, dtype=torch.bool, device="cuda")
    bad[[5, cols - 1]] = True
    assert dg[bad].isnan().all() and dg[~bad].isfinite().all() and db.isfinite().all()


def test_too_many_columns_are_refused_from_python(nrp):
    """With the code of an unsupported size, whichever call inside sees it first."""
    import torch
    torch.cuda.empty_cache()
    cols = 2 ** 31 - 1
    x = torch.empty(1, cols, device="cuda", dtype=torch.bfloat16)
    v = torch.empty(cols, device="cuda")
    s = torch.ones(1, device="cuda")
    for call in (lambda: nrp.layer_norm(x, v, v), lambda: nrp.layer_norm_backward(x, x, s, s, v)):
        with pytest.raises(nrp.NrpError, match="size") as e:
            call()
        assert e.value.code == nrp.NRP_ERR_UNSUPPORTED
    del x, v
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,cols", [(20, 64), (20, 77), (300, 77), (3000, 64), (700, 300),
                                       (600, 999), (600, 1000), (300, 1999), (50, 3001), (40, 6001)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_norm_gradient_of_constant_large_rows(nrp, rows, cols, dtype):
    """Rows of one large value, whose mean times rstd = eps^-1/2 passes f32's range:
    u is 0 in them, also where a row ends inside a strip.  Row sums are chains of
    cols / 32 + 20 additions (over 2048 columns cols / 256 + 20)."""
    import torch
    dt = {"bf16": torch.bfloat16, "f32": torch.float32}[dtype]
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.full((rows, cols), 2.0 ** 122, device="cuda", dtype=dt)
    mean = torch.full((rows,), 2.0 ** 122, device="cuda")
    rstd = torch.full((rows,), 1e-5 ** -0.5, device="cuda")
    dy = torch.randn(rows, cols, device="cuda", generator=g).to(dt)
    gamma = torch.randn(cols, device="cuda", generator=g)
    dx, dg, db = nrp.layer_norm_backward(dy, x, mean, rstd, gamma)
    w = dy.double() * gamma.double()
    ref = rstd.double()[:, None] * (w - w.mean(1, keepdim=True))
    size = rstd.double()[:, None] * (w.abs() + w.abs().mean(1, keepdim=True))
    chain = cols / 32 + 20 if cols <= 2048 else cols / 256 + 20
    assert ((dx.double() - ref).abs() <= size * chain * U
            + ref.abs() * torch.finfo(dt).eps / 2).all()
    assert (dg == 0).all()
    d = dy.double()
    assert ((db.double() - d.sum(0)).abs() <= (rows + 16) * U * d.abs().sum(0)).all()


@pytest.mark.parametrize("trans", [False, True])
def test_shared_reduction_of_far_scales(nrp, trans):
    """Scales of 2^100 by 2^30 (products of codes at most 2^-14: sums in range) where
    several CTAs share a tile's reduction of 32 blocks; tolerance as above."""
    import torch
    m, red, cols = 64, 4096, 256
    x = nrp.Fp8Tensor(codes((m, red), 2.0 ** -7, 1), torch.full((m, 32), 2.0 ** 100).cuda(), 1)
    wshape = (red, cols) if trans else (cols, red)
    w = nrp.Fp8Tensor(codes(wshape, 2.0 ** -7, 2),
                      torch.full([n // 128 for n in wshape], -2.0 ** 30).cuda(), 128)
    x.scales[:, ::2] = 2.0 ** -110
    x.scales[5] = 1.0
    xv, wv = values(x), values(w) if trans else values(w).t()
    ref, size = xv @ wv, xv.abs() @ wv.abs()
    call = nrp.fp8_linear_input_grad if trans else nrp.fp8_linear
    y = call(x, w, dtype=torch.float32).double().cpu()
    assert ((y - ref).abs() <= size * (132 * 2.0 ** -23 + 40 * U) + 96 * 2.0 ** -149).all()
