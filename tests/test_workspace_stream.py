"""Workspaces that a call or a plan allocates itself lie on the stream that uses them.

A caching allocator's block may still be in use by work that its last owner left enqueued on the current stream; work
on another stream would write into it ahead of that.  Checked on the CPU with a library and streams that only record
(the operators' direct calls and plans, the linear calls and plans), and on the GPU with work left enqueued.
"""
import contextlib
import ctypes as C
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")

from strix_trellis import abi, runtime  # noqa: E402

NEED = 4096


class _Stream:
    """Taken for a torch stream: by its type's module."""

    def __init__(self, handle):
        self.cuda_stream = handle


_Stream.__module__ = "torch.cuda.streams"


class _Library:
    """Every entry point succeeds; queries answer NEED bytes, creations a handle."""

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("_bytes"):
                args[-1]._obj.value = NEED
            elif name.endswith("_create"):
                args[-1]._obj.value = 1
            return 0
        call.__name__ = name
        return call


@pytest.fixture
def recorded(monkeypatch):
    """(context, weights, the current stream at each allocation of a workspace)."""
    state = SimpleNamespace(current=_Stream(1), seen=[])

    @contextlib.contextmanager
    def switch(stream):
        before, state.current = state.current, stream
        yield
        state.current = before

    allocate = runtime.alloc_workspace

    def record(*args):
        state.seen.append(state.current)
        return allocate(*args)

    monkeypatch.setattr(torch.cuda, "stream", switch)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: state.current)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle, device=None: _Stream(handle))
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: _Stream(0))
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, stream: None)
    monkeypatch.setattr(runtime, "alloc_workspace", record)
    lib = _Library()
    ctx = SimpleNamespace(handle=C.c_void_p(1), lib=lib, device=0)
    weights = SimpleNamespace(handle=C.c_void_p(2), ctx=ctx, lib=lib, input=64, output=32)
    return ctx, weights, state


def _calls(ctx, weights):
    x, y = torch.zeros(20, 64), torch.zeros(20, 32)
    e = torch.zeros(20)
    return {
        "int8 call": lambda s: runtime.int8_linear(weights, x, y, stream=s),
        "int8 plan": lambda s: runtime.Int8LinearPlan(weights, x, y, stream=s),
        "log probabilities call": lambda s: runtime.token_logprobs(ctx, x, entropy=e, stream=s),
        "log probabilities plan": lambda s: runtime.TokenLogprobsPlan(ctx, x, entropy=e, stream=s),
        "gemm call": lambda s: runtime.gemm(weights, x, y, stream=s),
        "linear plan": lambda s: runtime.LinearPlan(weights, x, y, stream=s, operation="gemm"),
    }


@pytest.mark.parametrize("what", ["int8 call", "int8 plan", "log probabilities call", "log probabilities plan", "gemm call",
                                  "linear plan"])
def test_workspaces_lie_on_their_stream(recorded, what):
    ctx, weights, state = recorded
    call, current = _calls(ctx, weights)[what], state.current
    call(None)
    call(_Stream(7))
    call(SimpleNamespace(cuda_stream=9))      # a HIP stream of the caller's
    call(SimpleNamespace(cuda_stream=0))      # the device's default stream
    assert [s.cuda_stream for s in state.seen] == [1, 7, 9, 0]
    assert state.current is current


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["torch", "hip"])
def test_memory_still_in_use_on_the_current_stream(kind):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from strix_trellis import device
    ctx = runtime.Context(0)
    g = torch.Generator().manual_seed(1)
    weights = runtime.Int8Weights(ctx, torch.randint(-127, 128, (300, 4096), generator=g, dtype=torch.int8).cuda(),
                                  torch.ones(300, device="cuda"))
    x, y, want = torch.randn(1000, 4096, device="cuda"), torch.zeros(1000, 300, device="cuda"), torch.zeros(1000, 300, device="cuda")
    side = torch.cuda.Stream() if kind == "torch" else device.Stream(0)
    runtime.int8_linear(weights, x, want)
    need = runtime.int8_linear_workspace_bytes(weights, x, y)
    assert need > 1 << 20
    out = torch.zeros(need, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for _ in range(3):
        torch.cuda.empty_cache()
        held = torch.full((need,), 77, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        torch.cuda._sleep(20_000_000)         # work ahead of the copy, some milliseconds
        out.copy_(held)
        del held                              # its memory is free for the next allocation on this stream
        runtime.int8_linear(weights, x, y, stream=side)
        torch.cuda.synchronize()
        assert bool((out == 77).all())
        assert torch.equal(y, want)
        out.zero_()
        y.zero_()
    weights.destroy()
    if kind == "hip":
        side.destroy()
