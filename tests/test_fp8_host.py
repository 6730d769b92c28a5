"""Refusals of the 8-bit linears' and the LayerNorm's C ABI without a GPU:
every argument is checked before the device is touched, so a zeroed stand-in
for the context is enough."""
import ctypes as C

import pytest

from __graft_entry__ import load_package

INVALID, UNSUPPORTED = -1, -3
F32, BF16 = 0, 1


@pytest.fixture(scope="module")
def nrp():
    from __graft_entry__ import _load_build_script
    _load_build_script().build()
    return load_package()


@pytest.fixture(scope="module")
def mem():
    buf = C.create_string_buffer(8192)
    return (C.addressof(buf) + 255) // 256 * 256, buf


def refused(nrp, code, fn, *args):
    assert getattr(nrp.lib(), fn)(*args) == code
    assert nrp.lib().nrp_last_error().decode()


def test_quantize_refusals(nrp, mem):
    p, _ = mem
    good = [p, None, BF16, p, 4, 64, 1, p, p]

    def bad(code, **kw):
        a = list(good)
        for k, v in kw.items():
            a[int(k[1:])] = v
        refused(nrp, code, "nrp_fp8_quantize", *a)

    bad(INVALID, _0=None)
    bad(INVALID, _3=None)
    bad(INVALID, _4=-1)
    bad(INVALID, _5=0)
    bad(INVALID, _7=None)
    bad(INVALID, _8=None)
    bad(UNSUPPORTED, _2=2)
    bad(UNSUPPORTED, _5=72)
    bad(UNSUPPORTED, _6=64)
    bad(INVALID, _3=p + 8)
    bad(INVALID, _7=p + 8)
    bad(INVALID, _8=p + 2)
    refused(nrp, UNSUPPORTED, "nrp_fp8_dequantize", p, None, p, p, 4, 60, 1, BF16, p)
    refused(nrp, UNSUPPORTED, "nrp_fp8_dequantize", p, None, p, p, 4, 64, 2, BF16, p)
    refused(nrp, UNSUPPORTED, "nrp_fp8_dequantize", p, None, p, p, 4, 64, 1, 7, p)
    refused(nrp, INVALID, "nrp_fp8_dequantize", p, None, p, p, 4, 64, 1, BF16, p + 4)
    refused(nrp, INVALID, "nrp_fp8_dequantize", p, None, None, p, 4, 64, 1, BF16, p)


@pytest.mark.parametrize("fn", ["nrp_fp8_linear", "nrp_fp8_linear_input_grad"])
def test_product_refusals(nrp, mem, fn):
    p, _ = mem
    # ctx, stream, dtype, x, xq, xs, M, red, wq, ws, out, (bias,) y
    good = [p, None, BF16, None, p, p, 4, 64, p, p, 32]
    good += [None, p] if fn == "nrp_fp8_linear" else [p]

    def bad(code, **kw):
        a = list(good)
        for k, v in kw.items():
            a[int(k[1:])] = v
        refused(nrp, code, fn, *a)

    bad(INVALID, _0=None)
    bad(INVALID, _4=None)
    bad(INVALID, _5=None)
    bad(INVALID, _8=None)
    bad(INVALID, _9=None)
    bad(INVALID, **{f"_{len(good) - 1}": None})
    bad(INVALID, _6=-1)
    bad(INVALID, _7=0)
    bad(INVALID, _10=0)
    bad(UNSUPPORTED, _2=3)
    bad(UNSUPPORTED, _7=65)
    bad(INVALID, _3=p + 4)   # an input to quantise, unaligned
    bad(INVALID, _4=p + 1)
    bad(INVALID, _8=p + 1)
    if fn.endswith("input_grad"):
        bad(UNSUPPORTED, _10=33)


def test_weight_grad_refusals(nrp, mem):
    p, _ = mem
    # ctx, stream, dy, xq, xs, M, N, K, dtype, dw, db
    good = [p, None, p, p, p, 4, 32, 64, F32, p, None]

    def bad(code, **kw):
        a = list(good)
        for k, v in kw.items():
            a[int(k[1:])] = v
        refused(nrp, code, "nrp_fp8_linear_weight_grad", *a)

    for i in (0, 2, 3, 4, 9):
        bad(INVALID, **{f"_{i}": None})
    bad(INVALID, _5=-1)
    bad(INVALID, _6=0)
    bad(INVALID, _7=0)
    bad(UNSUPPORTED, _6=36)
    bad(UNSUPPORTED, _7=72)
    bad(UNSUPPORTED, _8=2)
    bad(INVALID, _2=p + 2)
    bad(INVALID, _3=p + 2)


def test_layer_norm_refusals(nrp, mem):
    p, _ = mem
    good = [p, None, F32, p, 4, 33, p, p, 1e-5, p, p, p]

    def bad(code, **kw):
        a = list(good)
        for k, v in kw.items():
            a[int(k[1:])] = v
        refused(nrp, code, "nrp_layer_norm", *a)

    for i in (0, 3, 6, 7, 9):
        bad(INVALID, **{f"_{i}": None})
    bad(INVALID, _10=None)  # mean without rstd
    bad(INVALID, _11=None)
    bad(INVALID, _4=-1)
    bad(INVALID, _5=0)
    bad(INVALID, _8=-1.0)
    bad(INVALID, _8=float("nan"))
    bad(UNSUPPORTED, _2=2)


def test_layer_norm_backward_refusals(nrp, mem):
    p, _ = mem
    n = C.c_int64(-1)
    assert nrp.lib().nrp_layer_norm_backward_workspace(9, 33, C.byref(n)) == 0
    need = n.value
    assert need == 0  # few rows: none
    assert nrp.lib().nrp_layer_norm_backward_workspace(3000, 33, C.byref(n)) == 0
    need = n.value
    assert need > 0
    # ctx, stream, dtype, x, xs, dy, mean, rstd, gamma, rows, cols, dx, dg, db, ws, bytes
    good = [p, None, F32, p, None, p, p, p, p, 3000, 33, p, p, p, p, need]

    def bad(code, **kw):
        a = list(good)
        for k, v in kw.items():
            a[int(k[1:])] = v
        refused(nrp, code, "nrp_layer_norm_backward", *a)

    for i in (0, 3, 5, 6, 7, 8, 11):
        bad(INVALID, **{f"_{i}": None})
    bad(INVALID, _12=None)  # dgamma without dbeta
    bad(INVALID, _13=None)
    bad(INVALID, _9=-1)
    bad(INVALID, _10=0)
    bad(UNSUPPORTED, _2=9)
    bad(UNSUPPORTED, _4=p)  # codes of 33 columns
    bad(INVALID, _14=None)
    bad(INVALID, _15=need - 1)
    bad(INVALID, _14=p + 4)
    assert nrp.lib().nrp_layer_norm_backward_workspace(-1, 33, C.byref(n)) == INVALID
    assert nrp.lib().nrp_layer_norm_backward_workspace(9, 0, C.byref(n)) == INVALID
    assert nrp.lib().nrp_layer_norm_backward_workspace(9, 33, None) == INVALID


def test_python_refusals(nrp):
    """The torch layer refuses what the C ABI cannot see."""
    import torch
    x = torch.zeros(4, 64)
    with pytest.raises(nrp.NrpError):
        nrp.fp8_quantize(x)  # not on a CUDA device
    with pytest.raises(nrp.NrpError):
        nrp.layer_norm(x, torch.ones(64), torch.zeros(64))
    with pytest.raises(nrp.NrpError):
        nrp.fp8_linear(x, (x, x, 128))  # not an Fp8Tensor


# Arguments far apart, named by their place in the call: (function, arguments,
# outputs, inputs, element size of each).
AT = [0x10000000 * i for i in range(1, 12)]
CALLS = {
    "quantize": ("nrp_fp8_quantize", lambda a, p: [p, None, BF16, a["x"], 64, 256, 1, a["codes"],
                                                   a["scales"]],
                 {"codes": 16, "scales": 4}, {"x": 16}),
    "dequantize": ("nrp_fp8_dequantize", lambda a, p: [p, None, a["codes"], a["scales"], 64, 256, 1,
                                                       F32, a["x"]],
                   {"x": 16}, {"codes": 16, "scales": 4}),
    "linear": ("nrp_fp8_linear", lambda a, p: [p, None, BF16, a["x"], a["xq"], a["xs"], 64, 256,
                                               a["wq"], a["ws"], 512, a["bias"], a["y"]],
               {"y": 2, "xq": 16, "xs": 4}, {"x": 16, "wq": 16, "ws": 4, "bias": 2}),
    "linear of codes": ("nrp_fp8_linear", lambda a, p: [p, None, F32, None, a["xq"], a["xs"], 64,
                                                        256, a["wq"], a["ws"], 512, a["bias"],
                                                        a["y"]],
                        {"y": 4}, {"xq": 16, "xs": 4, "wq": 16, "ws": 4, "bias": 4}),
    "input gradient": ("nrp_fp8_linear_input_grad",
                       lambda a, p: [p, None, BF16, a["x"], a["xq"], a["xs"], 64, 256, a["wq"],
                                     a["ws"], 512, a["y"]],
                       {"y": 2, "xq": 16, "xs": 4}, {"x": 16, "wq": 16, "ws": 4}),
    "weight gradient": ("nrp_fp8_linear_weight_grad",
                        lambda a, p: [p, None, a["dy"], a["xq"], a["xs"], 64, 256, 512, F32,
                                      a["dw"], a["db"]],
                        {"dw": 4, "db": 4}, {"dy": 16, "xq": 16, "xs": 4}),
    "norm": ("nrp_layer_norm", lambda a, p: [p, None, BF16, a["x"], 64, 256, a["gamma"], a["beta"],
                                             C.c_float(1e-5), a["y"], a["mean"], a["rstd"]],
             {"y": 2, "mean": 4, "rstd": 4}, {"x": 2, "gamma": 4, "beta": 4}),
    "norm backward": ("nrp_layer_norm_backward",
                      lambda a, p: [p, None, BF16, a["x"], None, a["dy"], a["mean"], a["rstd"],
                                    a["gamma"], 1000, 256, a["dx"], a["dg"], a["db"], a["ws"],
                                    1 << 24],
                      {"dx": 2, "dg": 4, "db": 4, "ws": 16},
                      {"x": 2, "dy": 2, "mean": 4, "rstd": 4, "gamma": 4}),
    "norm backward of codes": ("nrp_layer_norm_backward",
                               lambda a, p: [p, None, F32, a["x"], a["xs"], a["dy"], a["mean"],
                                             a["rstd"], a["gamma"], 64, 256, a["dx"], a["dg"],
                                             a["db"], None, 0],
                               {"dx": 4, "dg": 4, "db": 4},
                               {"x": 16, "xs": 4, "dy": 4, "mean": 4, "rstd": 4, "gamma": 4}),
}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_overlaps_and_alignment(nrp, mem, name):
    """An output at the place of an input or of another output, and any argument
    off its alignment, is refused."""
    p, _ = mem
    fn, call, outs, ins = CALLS[name]
    place = dict(zip(list(outs) + list(ins), AT))
    for o in outs:
        for other in list(outs) + list(ins):
            if other == o:
                continue
            if name == "norm" and (o, other) == ("y", "x"):  # in place, but not shifted
                refused(nrp, INVALID, fn, *call(dict(place, y=place["x"] + 16), p))
            else:
                refused(nrp, INVALID, fn, *call(dict(place, **{o: place[other]}), p))
                assert "overlap" in nrp.lib().nrp_last_error().decode()
    for arg, align in {**outs, **ins}.items():
        refused(nrp, INVALID, fn, *call(dict(place, **{arg: place[arg] + align // 2}), p))
        assert "aligned" in nrp.lib().nrp_last_error().decode()
