"""CPU check of the Python layer's scales of the e4m3 layers: tensors that hold enough elements in another order are refused
before the library, which counts bytes, is called."""
import ctypes as C
import types

import pytest

torch = pytest.importorskip("torch")

from strix_trellis import runtime  # noqa: E402

E4M3 = torch.float8_e4m3fn


class Called(Exception):
    pass


class Library:
    """Any entry point of it says that it was called."""

    def __getattr__(self, name):
        def call(*args):
            raise Called(name)
        call.__name__ = name
        return call


CTX = types.SimpleNamespace(lib=Library(), handle=C.c_void_p(1))
LAYER = types.SimpleNamespace(ctx=CTX, lib=CTX.lib, handle=C.c_void_p(2))
STREAM = types.SimpleNamespace(cuda_stream=0)


def tensor(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def weights(scales, up_scales=None, N=300, I=640):
    w = tensor(N, I, dtype=E4M3)
    runtime.Fp8Weights(CTX, w, scales, up=None if up_scales is None else w, up_scales=up_scales, stream=STREAM)


@pytest.mark.parametrize("shape", [(5, 3), (15,), (3, 6), (4, 5), (3, 5, 2), (1, 15)])
def test_weights(shape):
    """[ceil(300 / 128), ceil(640 / 128)] is [3, 5]."""
    with pytest.raises(ValueError, match=r"^scales must be \[3, 5\]"):
        weights(tensor(*shape))
    with pytest.raises(ValueError, match=r"^up_scales must be \[3, 5\]"):
        weights(tensor(3, 5), tensor(*shape))


@pytest.mark.parametrize("shape", [(5, 7), (35,), (7, 6), (8, 5)])
def test_rows(shape):
    """Rows [7, 640] have scales [7, 5], hidden rows [7, 640] too."""
    x, y, wide = tensor(7, 640, dtype=E4M3), tensor(7, 300), tensor(7, 640, dtype=E4M3)
    for call in (runtime.fp8_linear, runtime.Fp8LinearPlan, runtime.fp8_gated, runtime.Fp8GatedPlan,
                 runtime.fp8_linear_workspace_bytes, runtime.fp8_gated_workspace_bytes):
        with pytest.raises(ValueError, match=r"^x_scales must be \[7, 5\]"):
            call(LAYER, x, y, x_scales=tensor(*shape))
    for call in (runtime.fp8_gated, runtime.Fp8GatedPlan, runtime.fp8_gated_workspace_bytes):
        with pytest.raises(ValueError, match=r"^y_scales must be \[7, 5\]"):
            call(LAYER, y, wide, y_scales=tensor(*shape))


def test_what_reaches_the_library():
    """The documented shapes, with dimensions of one left out or put in, and what is too short, which the library refuses."""
    for scales in (tensor(3, 5), tensor(3, 1, 5), None, tensor(2, 5), tensor(14)):
        with pytest.raises(Called):
            weights(scales)
    for scales in (tensor(1, 5), tensor(5), tensor(5, 1)):
        with pytest.raises(Called):
            weights(scales, N=128)
    x, y = tensor(7, 640, dtype=E4M3), tensor(7, 300)
    for scales in (tensor(7, 5), tensor(7, 5, 1), tensor(7, 4), None):
        with pytest.raises(Called):
            runtime.fp8_linear(LAYER, x, y, x_scales=scales)
    with pytest.raises(Called):
        runtime.fp8_linear(LAYER, x[:1], y[:1], x_scales=tensor(5))
    with pytest.raises(Called):
        runtime.fp8_linear(LAYER, x[:0], y[:0], x_scales=tensor(0, 5))
