"""Which stream the binding's calls go to, and whose tensors they take: host arithmetic, with a library that records what it is given."""
import types

import pytest
import torch

import sepal_runner_b200 as sb
from sepal_runner_b200 import lib as binding

DEVICE = -1  # what a CPU tensor answers to get_device(): these calls pass for calls on the context's device


@pytest.fixture()
def recorded(monkeypatch):
    """A Context without a device, and the arguments of its C calls."""
    calls = []

    class Library:
        here = staticmethod(lambda: None)

        def __getattr__(self, name):
            return lambda *args: calls.append((name, args, self.here())) or 0

    context = sb.Context.__new__(sb.Context)
    context._lib, context._h, context.device = Library(), None, DEVICE
    binding._torch()
    monkeypatch.setattr(binding, "_RAW_STREAM", lambda device: 7000 + device)  # the current stream of a device

    def other_device(*_):
        raise AssertionError("asked for the current device")

    monkeypatch.setattr(torch.cuda, "current_device", other_device)

    class Device:
        """torch.cuda.device, writing down the device that a call is made on."""

        here = None

        def __init__(self, device):
            self.device = device

        def __enter__(self):
            Device.here = self.device

        def __exit__(self, *_):
            Device.here = None

    monkeypatch.setattr(torch.cuda, "device", Device)
    context._lib.here = lambda: Device.here
    return context, calls


def every_call(ctx, stream=None):
    """Each launching call of the binding once; yields (position of the stream in the C call, counted from its end)."""
    h = lambda *shape: torch.zeros(shape, dtype=torch.float16)  # noqa: E731
    f = lambda *shape: torch.zeros(shape)  # noqa: E731
    b = lambda *shape: torch.zeros(shape, dtype=torch.int8)  # noqa: E731
    kw = {"stream": stream}
    ctx.gemm_f16(h(4, 128), h(8, 128), **kw)
    yield -1
    q, s = ctx.quantize_group_s8(f(128, 128), **kw)
    yield -1
    placed = ctx.prepare_w8g(q, s, **kw)
    yield -1
    ctx.gemm_w8g(h(4, 128), placed, **kw)
    yield -1
    q, s = ctx.quantize_rows_s8(h(8, 128), **kw)
    yield -1
    ctx.gemm_w8r(h(4, 128), q, s, **kw)
    yield -1
    ctx.rms_norm_s8(f(4, 128), f(128), **kw)
    yield -1
    ctx.quantize_tokens_s8(h(4, 128), **kw)
    yield -1
    ctx.gemm_s8(b(4, 128), f(4), b(8, 128), f(8), **kw)
    yield -1
    ctx.pack_gate_up(h(128, 64), **kw)
    yield -1
    ctx.float_to_half(f(64), **kw)
    yield -1
    ctx.status(**kw)
    yield 1
    ctx.debug_leave_status(0, **kw)
    yield 1
    shape = sb.AttentionShape(heads=2, kv_heads=1, head_dim=128, rotary_dims=32, rope_theta=1e4, eps=1e-6)
    rows = [(0, 4, 0, 0)]
    sb.attention_prepare(ctx, shape, rows, h(4, 512), h(4, 128), h(4, 128), f(128), f(128), h(4, 256), h(16, 128), h(16, 128), **kw)
    yield -1
    sb.attention(ctx, shape, rows, h(4, 256), h(16, 128), h(16, 128), h(4, 256), h(4, 256), **kw)
    yield -1
    shape = sb.DeltaNetShape(key_heads=1, value_heads=1, head_dim=128, conv_kernel=4, eps=1e-6)
    sb.deltanet(ctx, shape, rows, h(4, 384), h(4, 128), h(4, 1), h(4, 1), f(384, 4), f(1), f(1), f(128), f(1, 1, 128, 128), f(1, 3, 384), h(4, 128), **kw)
    yield -1


def test_calls_go_to_the_current_stream_of_the_contexts_device(recorded):
    """... whichever device is the current one."""
    ctx, calls = recorded
    without_context = {"quantize_group_s8", "prepare_w8g_scales", "quantize_rows_s8", "pack_gate_up", "float_to_half"}  # these run on the current device
    for at in every_call(ctx):
        name, args, here = calls[-1]
        assert args[at] == 7000 + DEVICE, name
        assert (here == DEVICE) == (name.replace("sepal_b200_", "") in without_context), name
    assert len({name for name, *_ in calls}) == 16


def test_a_stream_of_another_device_is_refused(recorded):
    ctx, calls = recorded
    wrong = types.SimpleNamespace(cuda_stream=5, device=types.SimpleNamespace(index=3))
    for call in (lambda: ctx.gemm_s8(torch.zeros((4, 16), dtype=torch.int8), torch.ones(4), torch.zeros((8, 16), dtype=torch.int8), torch.ones(8),
                                     torch.zeros(4, 8), stream=wrong),
                 lambda: ctx.status(stream=wrong), lambda: ctx.gemm_f16(torch.zeros((4, 16)).half(), torch.zeros((8, 16)).half(), torch.zeros(4, 8), stream=wrong)):
        with pytest.raises(ValueError, match="the context is on"):
            call()
    assert calls == []


def test_tensors_of_another_device_are_refused(recorded, monkeypatch):
    """Every launching call with tensors that are not on the context's device: an address that its kernel could not read."""
    ctx, calls = recorded
    calls_here = []
    for _ in every_call(ctx):
        calls_here.append(calls[-1][0])
    ctx.device = 0
    calls.clear()
    h, f, b = (lambda *shape, d=d: torch.zeros(shape, dtype=d) for d in (torch.float16, torch.float32, torch.int8))
    placed = sb.W8gWeight(q=b(8, 128), scales=f(8, 1), scales_t=h(1, 256), descale=f(2))
    attention = sb.AttentionShape(heads=2, kv_heads=1, head_dim=128, rotary_dims=32, rope_theta=1e4, eps=1e-6)
    deltanet = sb.DeltaNetShape(key_heads=1, value_heads=1, head_dim=128, conv_kernel=4, eps=1e-6)
    rows = [(0, 4, 0, 0)]
    for call in (lambda: ctx.gemm_f16(h(4, 128), h(8, 128)), lambda: ctx.quantize_group_s8(f(128, 128)), lambda: ctx.prepare_w8g(b(8, 128), f(8, 1)),
                 lambda: ctx.gemm_w8g(h(4, 128), placed), lambda: ctx.quantize_rows_s8(h(8, 128)), lambda: ctx.gemm_w8r(h(4, 128), b(8, 128), f(8)),
                 lambda: ctx.rms_norm_s8(f(4, 128), f(128)), lambda: ctx.quantize_tokens_s8(h(4, 128)), lambda: ctx.gemm_s8(b(4, 128), f(4), b(8, 128), f(8)),
                 lambda: ctx.pack_gate_up(h(128, 64)), lambda: ctx.float_to_half(f(64)),
                 lambda: sb.attention_prepare(ctx, attention, rows, h(4, 512), h(4, 128), h(4, 128), f(128), f(128), h(4, 256), h(16, 128), h(16, 128)),
                 lambda: sb.attention(ctx, attention, rows, h(4, 256), h(16, 128), h(16, 128), h(4, 256), h(4, 256)),
                 lambda: sb.deltanet(ctx, deltanet, rows, h(4, 384), h(4, 128), h(4, 1), h(4, 1), f(384, 4), f(1), f(1), f(128), f(1, 1, 128, 128), f(1, 3, 384), h(4, 128))):
        with pytest.raises(ValueError, match="cuda:0"):
            call()
    assert calls == [] and len(calls_here) == 16
    # the call without a context, which runs on the current device
    monkeypatch.setattr(binding, "library", lambda: ctx._lib)
    with pytest.raises(ValueError, match="this call runs on the current device"):
        sb.gemm_f16_noalloc(h(4, 128), h(8, 128), f(4, 8), stream=types.SimpleNamespace(cuda_stream=0), wait=False)
    assert calls == []
    ctx.device = DEVICE
    for bad in (torch.zeros(8, dtype=torch.float16), torch.zeros(4, 4).t()[:2]):
        with pytest.raises(AssertionError):
            ctx.float_to_half(bad)
    assert calls == []
