"""The 8-bit linears and the LayerNorm in the calls around the ordinary ones:
several streams and threads at once, first calls inside a capture, views off
the 16-byte boundaries, offsets past 32 bits.

What runs twice has to give the same bits (every kernel adds in a fixed
order), so most of these compare with a plain call of the same operator, which
the other tests hold against 64-bit forms."""
import math
import subprocess
import sys
import threading

import pytest

from __graft_entry__ import load_package

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nrp():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return load_package()


# rows, in and out columns: the few-row kernel, shared reductions, narrow and
# wide tiles
SIZES = [(14, 1024, 1024), (64, 2048, 1024), (300, 512, 512), (896, 1024, 2048),
         (2500, 1024, 1024)]


def operands(nrp, m, k, n, seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    return {"x": r(m, k).bfloat16(), "dy": r(m, n).mul_(0.01).bfloat16(), "bias": r(n).bfloat16(),
            "w": nrp.fp8_quantize(r(n, k) / math.sqrt(k), 128), "gamma": r(k), "beta": r(k)}


def step(nrp, o):
    """Every operator once, as a training step uses them."""
    h, mean, rstd = nrp.layer_norm(o["x"], o["gamma"], o["beta"])
    hq = nrp.fp8_quantize(h)
    y = nrp.fp8_linear(hq, o["w"], o["bias"])
    y2 = nrp.fp8_linear(h, o["w"], o["bias"])
    dh = nrp.fp8_linear_input_grad(o["dy"], o["w"])
    dw, db = nrp.fp8_linear_weight_grad(o["dy"], hq, bias=True)
    xq = nrp.fp8_quantize(o["x"])
    dx, dg, dbeta = nrp.layer_norm_backward(dh, xq, mean, rstd, o["gamma"])
    dx2 = nrp.layer_norm_backward(dh, o["x"], mean, rstd, o["gamma"])[0]
    back = nrp.fp8_dequantize(xq)
    return [h, mean, rstd, hq.codes.float(), hq.scales, y, y2, dh, dw, db, dx, dg, dbeta, dx2, back]


def same(a, b):
    import torch
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_streams_at_once(nrp):
    """Steps of different sizes queued on four streams at the same time."""
    import torch
    sets = [operands(nrp, *SIZES[i % len(SIZES)], seed=i) for i in range(4)]
    alone = [step(nrp, o) for o in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    runs = [[] for _ in sets]
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                runs[i].append(step(nrp, sets[i]))
    torch.cuda.synchronize()
    nrp.Context.default().check()
    assert all(same(r, alone[i]) for i in range(4) for r in runs[i])


def test_threads(nrp):
    import torch
    sets = [operands(nrp, *s, seed=9) for s in SIZES[:3]]
    alone = [step(nrp, o) for o in sets]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(8):
                got = step(nrp, sets[i])
                st.synchronize()
                if not same(got, alone[i]):
                    wrong.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(len(sets))]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not wrong


def test_graphs_of_several_streams(nrp):
    """Two captured steps replayed at once on two streams, between eager calls,
    with their inputs changed in place."""
    import torch
    sets = [operands(nrp, *s, seed=3) for s in ((64, 2048, 1024), (896, 1024, 2048))]
    graphs, outs = [], []
    for o in sets:
        step(nrp, o)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(nrp, o))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in sets]
    for turn in range(4):
        for o in sets:
            o["x"].mul_(-0.5)
            o["dy"].mul_(2.0)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        eager = [step(nrp, o) for o in sets]
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(outs, eager)), turn
    nrp.Context.default().check()


FIRST = """
import sys
sys.path.insert(0, {root!r})
import torch
from __graft_entry__ import load_package
import tests.test_gpu_fp8_edges as t
nrp = load_package()
ctx = nrp.Context.default()
sizes = t.SIZES + [(749, 1024, 1024), (40, 5008, 272)]
sets = [t.operands(nrp, *s) for s in sizes]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = [t.step(nrp, o) for o in sets]
graph.replay()
torch.cuda.synchronize()
ctx.check()
assert all(t.same(a, t.step(nrp, o)) for a, o in zip(got, sets))
print("fine")
"""


def test_first_calls_inside_a_capture(nrp):
    """A process whose first call of each kernel is captured (attributes and
    occupancy are asked for there)."""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST.format(root=root)], capture_output=True,
                       text=True, timeout=300, cwd=root)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("m,k,n", SIZES + [(37, 336, 208)])
def test_views_off_the_boundary(nrp, m, k, n):
    """Outputs, biases and parameters one element past a 16-byte boundary,
    and nothing written around them."""
    import torch
    o = operands(nrp, m, k, n, seed=5)
    plain = step(nrp, o)

    def off(shape, dtype):
        held = torch.full((math.prod(shape) + 2,), 3.0, device="cuda", dtype=dtype)
        return held, held[1:-1].view(shape)

    def moved(t):
        held, v = off(t.shape, t.dtype)
        v.copy_(t)
        return v

    bf, f32 = torch.bfloat16, torch.float32
    h, mean, rstd, y, dh, dw, db, dx, dg, dbeta, dx2 = (plain[i] for i in
                                                       (0, 1, 2, 5, 7, 8, 9, 10, 11, 12, 13))
    hq, xq = nrp.fp8_quantize(h), nrp.fp8_quantize(o["x"])
    gamma, beta, bias = moved(o["gamma"]), moved(o["beta"]), moved(o["bias"])
    outs = {name: off(t.shape, t.dtype) for name, t in
            {"h": h, "y": y, "dh": dh, "dw": dw, "db": db, "dx": dx, "dx2": dx2}.items()}
    nrp.fp8_linear(hq, o["w"], bias, out=outs["y"][1])
    nrp.fp8_linear_input_grad(o["dy"], o["w"], out=outs["dh"][1])
    nrp.fp8_linear_weight_grad(o["dy"], hq, out=outs["dw"][1], bias_out=outs["db"][1])
    for name, want in (("y", y), ("dh", dh), ("dw", dw), ("db", db)):
        assert torch.equal(outs[name][1], want), name
    # The norms take other kernels for such views, with other orders of the sums.
    # Either's sums over a row (of unit scale) are within chain 2^-24 of the exact
    # ones; u, gamma and dh stay below 8 here, so no value moves by more than 64
    # times the sums of both do; in bf16 a rounding may fall the other way, one
    # step (2^-7 relative).  A sum over rows has a chain of m + 16.
    off_f32 = 64 * 2 * (k / 8 + 16) * 2.0 ** -24
    mean2, rstd2 = moved(mean), moved(rstd)
    got, m2, r2 = nrp.layer_norm(moved(o["x"]), gamma, beta, out=outs["h"][1])
    a = nrp.layer_norm_backward(moved(dh), xq, mean2, rstd2, gamma, out=outs["dx"][1])
    b = nrp.layer_norm_backward(moved(dh), moved(o["x"]), mean2, rstd2, gamma, out=outs["dx2"][1])
    for got, want in ((got, h), (m2, mean), (r2, rstd), (a[0], dx), (b[0], dx2)):
        step_of = 2.0 ** -7 * want.double().abs() if want.dtype == bf else 0.0
        assert ((got.double() - want.double()).abs() <= off_f32 + step_of).all()
    d = dh.double().abs()
    u = ((nrp.fp8_dequantize(xq, f32).double() - mean[:, None]) * rstd[:, None]).abs()
    assert ((a[1].double() - dg.double()).abs()
            <= (m + 16) * 2.0 ** -23 * (d * (u + 1)).sum(0)).all()
    assert ((a[2].double() - dbeta.double()).abs() <= (m + 16) * 2.0 ** -23 * d.sum(0)).all()
    for name, (held, _) in outs.items():
        assert held[0] == 3 and held[-1] == 3, name


def test_offsets_past_32_bits(nrp):
    """More than 2^32 elements: the last rows are what the same rows give by
    themselves."""
    import torch
    torch.cuda.empty_cache()
    m, k, n = 4_200_000, 1024, 16
    tail = 300
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(m, k, device="cuda", dtype=torch.bfloat16)
    for i in range(0, m, 600_000):
        x[i:i + 600_000].normal_(generator=g)
    gamma, beta = torch.ones(k, device="cuda"), torch.zeros(k, device="cuda")
    xq = nrp.fp8_quantize(x)
    last = nrp.fp8_quantize(x[-tail:])
    assert torch.equal(xq.codes[-tail:].float(), last.codes.float())
    assert torch.equal(xq.scales[-tail:], last.scales)
    assert torch.equal(nrp.fp8_dequantize(xq)[-tail:], nrp.fp8_dequantize(last))
    w = nrp.fp8_quantize(torch.randn(n, k, device="cuda", generator=g), 128)
    # (few rows share their reductions: another order of the block sums, so
    # against 64 bits: 132 additions cut at 2^-23 in a block, then k / 128)
    xv, wv = (nrp.fp8_dequantize(q, torch.float32).double() for q in (last, w))
    ref, size = xv @ wv.t(), xv.abs() @ wv.t().abs()
    off = (nrp.fp8_linear(xq, w, dtype=torch.float32)[-tail:].double() - ref).abs()
    assert (off <= size * (132 * 2.0 ** -23 + (k // 128 + 1) * 2.0 ** -24)).all()
    # dw of a dy that is zero but for the last rows
    dy = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)
    dy[-tail:].normal_(generator=g)
    dw, db = nrp.fp8_linear_weight_grad(dy, xq, bias=True)
    ref = dy[-tail:].double().t() @ nrp.fp8_dequantize(last).double()
    size = dy[-tail:].double().abs().t() @ nrp.fp8_dequantize(last).double().abs()
    assert ((dw.double() - ref).abs() <= size * (tail + 64) * 2.0 ** -23).all()
    assert ((db.double() - dy[-tail:].double().sum(0)).abs()
            <= dy[-tail:].double().abs().sum(0) * (tail + 16) * 2.0 ** -24).all()
    del dy
    h, mean, rstd = nrp.layer_norm(x, gamma, beta)
    h2, mean2, rstd2 = nrp.layer_norm(x[-tail:], gamma, beta)
    assert torch.equal(h[-tail:], h2) and torch.equal(mean[-tail:], mean2)
    dx = nrp.layer_norm_backward(h, xq, mean, rstd, gamma)[0]
    assert torch.equal(dx[-tail:], nrp.layer_norm_backward(h2, last, mean2, rstd2, gamma)[0])
    nrp.Context.default().check()
    # the products' outputs past 2^32 elements
    del h, dx, x
    torch.cuda.empty_cache()
    g8 = nrp.fp8_quantize(torch.randn(m, n, device="cuda", generator=g).bfloat16())
    wide = nrp.fp8_linear_input_grad(g8, w)
    few = nrp.Fp8Tensor(g8.codes[-tail:], g8.scales[-tail:], 1)
    assert torch.equal(wide[-tail:], nrp.fp8_linear_input_grad(few, w))
    del wide
    torch.cuda.empty_cache()


def test_statistics_and_sums_are_tensors_of_their_own(nrp):
    """mean and rstd, dgamma and dbeta: their values stay when the other of the
    pair is written or goes away, also for no rows, and autograd takes them."""
    import torch
    o = operands(nrp, 33, 256, 256, seed=2)
    y, mean, rstd = nrp.layer_norm(o["x"].view(3, 11, 256), o["gamma"], o["beta"])
    assert mean.shape == rstd.shape == (3, 11) and mean.is_contiguous() and rstd.is_contiguous()
    keep = rstd.clone()
    mean.zero_()
    del mean
    torch.full((4096,), 5.0, device="cuda")
    assert torch.equal(rstd, keep)
    dx, dg, db = nrp.layer_norm_backward(y, o["x"].view(3, 11, 256), rstd * 0, rstd, o["gamma"])
    assert dg.shape == db.shape == (256,)
    keep = db.clone()
    dg.add_(1)
    assert torch.equal(db, keep)
    p = torch.ones(256, device="cuda", requires_grad=True)
    (p * db).sum().backward()
    assert torch.equal(p.grad, db)
    e, mean, rstd = nrp.layer_norm(o["x"][:0], o["gamma"], o["beta"])
    assert mean.shape == rstd.shape == (0,) and e.shape == (0, 256)
    q = nrp.fp8_quantize(o["x"].view(3, 11, 256)[:, :, :80].contiguous())
    assert q.codes.shape == (3, 11, 80) and q.scales.shape == (33, 1)
    codes = q.codes.float()
    q.scales.mul_(2)
    assert torch.equal(q.codes.float(), codes) and q.codes.is_contiguous()
    assert nrp.fp8_quantize(o["x"][:0], 128).scales.shape == (0, 2)


@pytest.mark.parametrize("rows,cols", [(128, 512), (129, 512), (32, 2048), (33, 2048), (256, 200),
                                       (257, 200), (86, 768), (4097, 8), (3, 2056), (5000, 1),
                                       (5001, 16), (4999, 77), (3000, 128), (3001, 127),
                                       (300, 129), (70, 4096), (33, 3001), (50, 6000),
                                       (50, 6001), (120, 8200)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_norm_gradient_on_both_sides_of_one_launch(nrp, rows, cols, dtype):
    """Where one cluster takes all rows and where two launches do, with the
    workspace that the size asks for, and rows of half a warp: all gradients
    against 64 bits."""
    import ctypes as C
    import torch
    dt = {"bf16": torch.bfloat16, "f32": torch.float32}[dtype]
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, cols, device="cuda", generator=g).to(dt)
    dy = torch.randn(rows, cols, device="cuda", generator=g).to(dt)
    gamma = torch.randn(cols, device="cuda", generator=g)
    _, mean, rstd = nrp.layer_norm(x, gamma, gamma)
    size = C.c_int64()
    assert nrp.lib().nrp_layer_norm_backward_workspace(rows, cols, C.byref(size)) == 0
    assert (size.value == 0) == (cols <= 2048 and rows * (-(-cols // 256) * 256) <= 65536)
    dx, dg, db = nrp.layer_norm_backward(dy, x, mean, rstd, gamma)
    u = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    d = dy.double()
    w = d * gamma.double()
    c2 = (w * u).mean(1, keepdim=True)
    ref = rstd.double()[:, None] * (w - w.mean(1, keepdim=True) - u * c2)
    size = rstd.double()[:, None] * (w.abs() + w.abs().mean(1, keepdim=True)
                                     + u.abs() * (w * u).abs().mean(1, keepdim=True))
    # row sums: chains of cols / 32 + 16 at most, in rows over 2048 of cols / 256 + 16
    half = 2.0 ** -8 if dt == torch.bfloat16 else 2.0 ** -24
    assert ((dx.double() - ref).abs() <= size * (cols / 32 + 20) * 2.0 ** -24
            + ref.abs() * half + 2.0 ** -30).all()
    # u takes two roundings, dy u one, a column's chain rows + 16
    assert ((dg.double() - (d * u).sum(0)).abs()
            <= (rows + 20) * 2.0 ** -24 * (d * u).abs().sum(0) + 2.0 ** -30).all()
    assert ((db.double() - d.sum(0)).abs() <= (rows + 16) * 2.0 ** -24 * d.abs().sum(0)).all()


@pytest.mark.parametrize("rows,cols", [(700, 129), (701, 777), (600, 130), (900, 255), (1300, 1023),
                                       (333, 2047), (2000, 1001)])
@pytest.mark.parametrize("off", [0, 1, 2])
def test_norm_gradient_of_odd_rows(nrp, rows, cols, off):
    """bf16 rows of odd columns and of tensors off a word: all gradients, and
    nothing written around dx."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(cols)

    def view(fill=None):
        held = torch.full((rows * cols + off + 8,), 9.0, device="cuda", dtype=torch.bfloat16)
        v = held[off:off + rows * cols].view(rows, cols)
        if fill is not None:
            v.copy_(fill)
        return held, v

    x = view(torch.randn(rows, cols, device="cuda", generator=g) + 0.5)[1]
    dy = view(torch.randn(rows, cols, device="cuda", generator=g))[1]
    gamma = torch.randn(cols, device="cuda", generator=g)
    _, mean, rstd = nrp.layer_norm(x, gamma, gamma)
    held, out = view()
    dx, dg, db = nrp.layer_norm_backward(dy, x, mean, rstd, gamma, out=out)
    assert (held[:off] == 9).all() and (held[off + rows * cols:] == 9).all()
    d, u = dy.double(), (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    w = d * gamma.double()
    c1, c2 = w.mean(1, keepdim=True), (w * u).mean(1, keepdim=True)
    ref = rstd.double()[:, None] * (w - c1 - u * c2)
    # row sums: chains of cols / 32 + 16 at most in f32, u's two roundings
    chain = (cols / 32 + 20) * 2.0 ** -24
    size = rstd.double()[:, None] * (w.abs() + w.abs().mean(1, keepdim=True)
                                     + u.abs() * (w * u).abs().mean(1, keepdim=True))
    assert ((dx.double() - ref).abs() <= size * chain + ref.abs() * 2.0 ** -8).all()
    assert ((dg.double() - (d * u).sum(0)).abs()
            <= (rows + 20) * 2.0 ** -24 * (d * u).abs().sum(0) + 2.0 ** -30).all()
    assert ((db.double() - d.sum(0)).abs() <= (rows + 16) * 2.0 ** -24 * d.abs().sum(0)).all()


@pytest.mark.parametrize("rows,cols", [(20, 512), (5000, 64), (5000, 1024), (3000, 777), (40, 6001),
                                       (700, 2048), (50, 4096), (90, 8192)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_norm_gradient_without_parameters(nrp, rows, cols, dtype):
    """dgamma, dbeta and workspace NULL: the same dx, in every kernel."""
    import torch
    dt = {"bf16": torch.bfloat16, "f32": torch.float32}[dtype]
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, cols, device="cuda", generator=g).to(dt)
    dy = torch.randn(rows, cols, device="cuda", generator=g).to(dt)
    gamma = torch.randn(cols, device="cuda", generator=g)
    _, mean, rstd = nrp.layer_norm(x, gamma, gamma)
    want = nrp.layer_norm_backward(dy, x, mean, rstd, gamma)[0]
    ctx, st = nrp.Context.default(), torch.cuda.current_stream().cuda_stream
    dx = torch.empty_like(x)
    code = nrp.BF16 if dt == torch.bfloat16 else nrp.F32
    assert nrp.lib().nrp_layer_norm_backward(
        ctx.handle, st, code, x.data_ptr(), None, dy.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
        gamma.data_ptr(), rows, cols, dx.data_ptr(), None, None, None, 0) == 0
    assert torch.equal(dx, want)
