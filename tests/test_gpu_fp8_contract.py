"""What the 8-bit operators' and the LayerNorm's documentation allows beyond the
ordinary calls: the ends of the sizes, scales of every f32 value, rows of very
large values, profiling from several threads, autograd's view of the outputs.

u = 2^-24 is half a step of f32."""
import math

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
