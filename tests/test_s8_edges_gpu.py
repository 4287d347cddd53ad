"""Activations in 8 bits where a range, a promise or a stream ends."""
import pytest
import torch

import sepal_runner_b200 as sb

pytestmark = pytest.mark.gpu


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(gen, *shape, std=1.0):
    return torch.randn(shape, generator=gen, device="cuda") * std


# (the vector kernel's narrow and wide blocks, rows it reads twice, and the kernel of single values)
@pytest.mark.parametrize("cols", [256, 12288, 12292, 255])
@pytest.mark.parametrize("delta", [None, torch.float16, torch.float32])
def test_a_normed_row_that_overflows(ctx, cols, delta):
    """x (1 + w) is finite and its quotient by the root mean square is not: a NaN scale, zero bytes and NaN values; the other rows as alone."""
    gen = generator(cols)
    x = randn(gen, 6, cols)
    w = torch.zeros(cols, device="cuda")
    w[cols // 2] = 2.0**127
    x[:, cols // 2] = 0.0  # the ordinary rows do not meet the large gain
    x[1, cols // 2] = 0.125  # u = 2^124, and the row's root mean square is 2^-6 ..
    x[1] *= 2.0**-4          # .. (below): v = 2^120 * 2^9 or so
    x[1, : cols // 2] *= 2.0**-6
    x[1, cols // 2 + 1 :] *= 2.0**-6
    d = None if delta is None else torch.zeros((6, cols), device="cuda").to(delta)
    u = x[1].double() * (1 + w.double())
    v = u / (x[1].double().square().mean() + 1e-6).sqrt()
    assert u.abs().max() < 3.4e38 < v.abs().max() / 2
    values = torch.full((6, cols), 9.0, dtype=torch.float16, device="cuda")
    q, s = ctx.rms_norm_s8(x.clone(), w, delta=d, values=values)
    assert torch.isnan(s).tolist() == [False, True, False, False, False, False]
    assert (q[1] == 0).all() and torch.isnan(values[1]).all()
    rest = [0, 2, 3, 4, 5]
    q0, s0 = ctx.rms_norm_s8(x[rest].clone(), w)
    assert torch.equal(q[rest], q0) and torch.equal(s[rest], s0)
    # the largest v that float32 holds is still a number
    x[1] = 0.0
    x[1, 0] = 1.0
    w.zero_()
    smooth = torch.full((cols,), float(torch.finfo(torch.float32).max) / 2 / cols**0.5, device="cuda")
    q, s = ctx.rms_norm_s8(x[1:2].clone(), w, col_scale=smooth, delta=None if d is None else d[:1])
    assert torch.isfinite(s).all() and q[0, 0] == 127 and (q[0, 1:] == 0).all()


def test_products_that_overflow_before_the_division(ctx):
    """An infinity in x (1 + w) is one, though its quotient would fit."""
    x = torch.full((2, 64), 1e10, device="cuda")
    x[1] = 1.0
    w = torch.zeros(64, device="cuda")
    w[3] = 1e30
    q, s = ctx.rms_norm_s8(x, w)
    assert torch.isnan(s).tolist() == [True, False] and (q[0] == 0).all() and q[1, 3] == 127


def test_rows_that_the_weights_quantiser_treats_otherwise(ctx):
    """The two quantisers on binary16: the same bytes on finite rows, down to products of 2^-121; here a row that is not finite is marked."""
    gen = generator(4)
    x = randn(gen, 4, 64).half()
    x[0] = 0
    x[1, 0] = 6e-8
    for factor in (1.0, 2.0**-110):
        smooth = torch.full((64,), factor, device="cuda")
        assert (x[2].float().abs().max() * factor) >= 2.0**-121
        q, s = ctx.quantize_tokens_s8(x, col_scale=smooth)
        want, want_s = ctx.quantize_rows_s8(x, smooth)
        assert torch.equal(q, want) and torch.equal(s, want_s)
    x[2, 3], x[3, 5] = float("nan"), float("inf")
    q, s = ctx.quantize_tokens_s8(x)
    assert torch.isnan(s).tolist() == [False, False, True, True] and (q[2:] == 0).all()


def test_a_context_before_torch_has_touched_the_gpu():
    """The stream of a call is found in a process whose torch has not initialised CUDA yet."""
    import os
    import subprocess
    import sys

    code = "import sepal_runner_b200 as sb; c = sb.Context(0); assert c.status() == 0; c.debug_leave_status(5); assert c.status() == 5 and c.status() == 0; c.close()"
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def stream_of(tensor):
    """The stream that torch's allocator has a tensor's memory down for."""
    for segment in torch.cuda.memory_snapshot():
        if segment["address"] <= tensor.data_ptr() < segment["address"] + segment["total_size"]:
            return segment["stream"]
    raise AssertionError("not memory of torch's allocator")


def test_results_belong_to_the_stream_of_the_call(ctx):
    """What a call with `stream=` allocates is that stream's: memory of the current stream may still be in use there, and would be handed
    out again there while the call's own stream writes it."""
    side = torch.cuda.Stream()
    gen = generator(12)
    x16, x32, w16 = randn(gen, 40, 256).half(), randn(gen, 40, 256), randn(gen, 128, 256).half()
    gain, stacked = torch.zeros(256, device="cuda"), randn(gen, 128, 256).half()
    torch.cuda.synchronize()
    for stream, number in ((side, side.cuda_stream), (None, torch.cuda.current_stream().cuda_stream)):
        q, s = ctx.rms_norm_s8(x32, gain, stream=stream)
        q2, s2 = ctx.quantize_tokens_s8(x16, stream=stream)
        wq, sw = ctx.quantize_rows_s8(w16, stream=stream)
        gq, gs = ctx.quantize_group_s8(x32, stream=stream)
        placed = ctx.prepare_w8g(gq, gs, stream=stream)
        results = [q, s, q2, s2, wq, sw, gq, gs, placed.scales_t, placed.descale, ctx.gemm_s8(q, s, wq, sw, stream=stream), ctx.gemm_f16(x16, w16, stream=stream),
                   ctx.gemm_w8r(x16, wq, sw, stream=stream), ctx.gemm_w8g(x16, placed, stream=stream), ctx.pack_gate_up(stacked, stream=stream),
                   ctx.float_to_half(x32, stream=stream)]
        assert [stream_of(r) for r in results] == [number] * len(results)
        torch.cuda.synchronize()
    ctx.check_status()


def test_results_on_another_stream_over_busy_memory(ctx):
    """A result is not placed over memory that the current stream's work still reads."""
    side = torch.cuda.Stream()
    gen = generator(13)
    x = randn(gen, 4096, 4096)
    gain = torch.zeros(4096, device="cuda")
    want_q, want_s = ctx.rms_norm_s8(x, gain)
    source = torch.randint(0, 100, (4096, 4096), generator=gen, device="cuda", dtype=torch.int8)
    total = source.long().sum().item()
    matrix = randn(gen, 4096, 4096)
    torch.cuda.synchronize()
    for _ in range(5):
        busy = source.clone()
        torch.cuda.synchronize()
        for _ in range(4):
            matrix @ matrix  # the current stream works for a while before it reads `busy`
        late = busy.long().sum()
        del busy
        q, s = ctx.rms_norm_s8(x, gain, stream=side)
        torch.cuda.synchronize()
        assert late.item() == total and torch.equal(q, want_q) and torch.equal(s, want_s)


# (few rows of a long k: the few-rows kernel with its parts of k; many: pairs. Both request weights ahead of the kernel before them.)
@pytest.mark.parametrize("t,hidden,inner", [(1, 1024, 4096), (29, 1024, 4096), (200, 1024, 4096), (700, 512, 640)])
def test_weights_requested_early_change_no_bits(t, hidden, inner):
    """A layer's MLP many times over, back to back: as dependents and in plain order, with and without the promise of static weights."""
    gen = generator(t)
    start, delta, gain = randn(gen, t, hidden, std=2.0), randn(gen, t, hidden, std=0.1).half(), randn(gen, hidden, std=0.2)
    c = sb.Context(0)
    gate_up, gate_up_s = c.quantize_rows_s8(randn(gen, 2 * inner, hidden, std=0.02).half())
    down, down_s = c.quantize_rows_s8(randn(gen, hidden, inner, std=0.02).half())
    c.close()
    torch.cuda.synchronize()
    results = []
    for overlap in (1, 0):
        for static in (False, True):
            sb.library().sepal_b200_set_launch_overlap(overlap)
            c = sb.Context(0)
            c.set_static_weights(static)
            x = start.clone()
            torch.cuda.synchronize()
            for _ in range(12):
                q, s = c.rms_norm_s8(x, gain, delta=delta)
                a = c.gemm_s8(q, s, gate_up, gate_up_s, epilogue=sb.SWIGLU)
                q, s = c.quantize_tokens_s8(a)
                c.gemm_s8(q, s, down, down_s, x, epilogue=sb.ADD)
            c.check_status()
            results.append(x)
            c.close()
    assert torch.isfinite(results[0]).all() and not torch.equal(results[0], start)
    assert all(torch.equal(r, results[0]) for r in results[1:])
