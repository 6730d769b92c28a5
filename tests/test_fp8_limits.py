"""The ends of the 8-bit operators' and the LayerNorm's argument ranges without
a GPU: what the kernels' 32-bit indices cannot take is refused before the device
is touched."""
import ctypes as C

import pytest

from __graft_entry__ import load_package

INVALID, UNSUPPORTED = -1, -3
F32, BF16 = 0, 1
MOST = 2 ** 31 - 4096  # the largest size of a product

# pointers far enough apart that no argument of any size meets another
AT = [(i + 1) << 52 for i in range(10)]


@pytest.fixture(scope="module")
def nrp():
    from __graft_entry__ import _load_build_script
    _load_build_script().build()
    return load_package()


@pytest.fixture(scope="module")
def ctx():
    buf = C.create_string_buffer(8192)
    return (C.addressof(buf) + 255) // 256 * 256, buf


def status(nrp, fn, *args):
    rc = getattr(nrp.lib(), fn)(*args)
    return rc, nrp.lib().nrp_last_error().decode()


def product(fn, ctx, m, red, cols):
    x, xq, xs, wq, ws, y = AT[:6]
    a = [ctx, None, BF16, None, xq, xs, m, red, wq, ws, cols]
    return a + ([None, y] if fn == "nrp_fp8_linear" else [y])


@pytest.mark.parametrize("fn", ["nrp_fp8_linear", "nrp_fp8_linear_input_grad"])
@pytest.mark.parametrize("sizes", [(2 ** 31 - 1, 16, 16), (MOST + 1, 16, 16), (16, 2 ** 31 - 16, 16),
                                   (16, 16, 2 ** 31 - 16)])
def test_product_sizes(nrp, ctx, fn, sizes):
    rc, msg = status(nrp, fn, *product(fn, ctx[0], *sizes))
    assert rc == UNSUPPORTED and "size" in msg


@pytest.mark.parametrize("m,n,k", [(2 ** 31 - 1, 8, 16), (2 ** 31 - 63, 8, 16), (MOST + 1, 8, 16),
                                   (64, 2 ** 31 - 8, 16), (64, 8, 2 ** 31 - 16)])
def test_weight_gradient_sizes(nrp, ctx, m, n, k):
    """From 2^31 - 63 rows on the count of 64-token steps would be negative."""
    rc, msg = status(nrp, "nrp_fp8_linear_weight_grad", ctx[0], None, AT[0], AT[1], AT[2], m, n, k,
                     F32, AT[3], AT[4])
    assert rc == UNSUPPORTED and "size" in msg


@pytest.mark.parametrize("cols", [MOST + 1, 2 ** 31 - 2048, 2 ** 31 - 1])
def test_norm_columns(nrp, ctx, cols):
    """The last columns' indices would pass 2^31 and come back negative."""
    p = ctx[0]
    rc, msg = status(nrp, "nrp_layer_norm", p, None, BF16, AT[0], 1, cols, AT[1], AT[2], 1e-5, AT[3],
                     AT[4], AT[5])
    assert rc == UNSUPPORTED and "size" in msg
    n = C.c_int64()
    rc, msg = status(nrp, "nrp_layer_norm_backward_workspace", 1, cols, C.byref(n))
    assert rc == UNSUPPORTED and "size" in msg
    rc, msg = status(nrp, "nrp_layer_norm_backward", p, None, BF16, AT[0], None, AT[1], AT[2], AT[3],
                     AT[4], 1, cols, AT[5], AT[6], AT[7], AT[8], 1 << 40)
    assert rc == UNSUPPORTED and "size" in msg


def test_default_context_of_threads(nrp, monkeypatch):
    """Threads that ask for a device's default context at once get the same one
    (its making releases the GIL)."""
    import threading
    import time
    made = []

    def slow(self, device=0):
        time.sleep(0.05)
        self.handle, self.device = None, device
        made.append(self)

    monkeypatch.setattr(nrp.Context, "__init__", slow)
    monkeypatch.setattr(nrp.Context, "_default", {})
    got = []
    ts = [threading.Thread(target=lambda: got.append(nrp.Context.default(3))) for _ in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert len(made) == 1 and all(c is made[0] for c in got) and len(got) == 4


@pytest.mark.parametrize("off", [None, 1])
def test_pointers_of_no_rows(nrp, ctx, off):
    """A matrix without rows: its pointers may be null or anything.  What is asked
    for is then nothing, or (without a device) the device."""
    p, n = ctx[0], 0
    q = None if off is None else AT[0] + off
    g = AT[1]
    calls = [
        ("nrp_fp8_quantize", p, None, BF16, q, n, 64, 1, q, q),
        ("nrp_fp8_quantize", p, None, F32, q, n, 64, 128, q, q),
        ("nrp_fp8_dequantize", p, None, q, q, n, 64, 1, F32, q),
        ("nrp_fp8_linear", p, None, BF16, None, q, q, n, 64, g, g, 32, None, q),
        ("nrp_fp8_linear", p, None, BF16, q, q, q, n, 64, g, g, 32, None, q),
        ("nrp_fp8_linear_input_grad", p, None, BF16, q, q, q, n, 64, g, g, 32, q),
        ("nrp_layer_norm", p, None, F32, q, n, 64, g, g, 1e-5, q, q, q),
        ("nrp_layer_norm_backward", p, None, F32, q, None, q, q, q, g, n, 64, q, None, None, None, 0),
        ("nrp_layer_norm_backward", p, None, F32, q, g, q, q, q, g, n, 64, q, None, None, None, 0),
    ]
    for fn, *args in calls:
        rc, msg = status(nrp, fn, *args)
        assert rc in (0, -2), (fn, msg)
