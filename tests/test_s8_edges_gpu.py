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


@pytest.mark.parametrize("t,n,k", [(20, 256, 256), (200, 256, 384)])
def test_residual_updates_at_the_ends_of_float32(ctx, t, n, k):
    """Old values and products that are subnormal, zeros of either sign, infinities and NaN: every schedule and alignment of Y adds them as one
    IEEE addition does, the TMA's reductions too."""
    gen = generator(t)
    x = torch.randint(-127, 128, (t, k), generator=gen, device="cuda", dtype=torch.int8)
    w = torch.randint(-127, 128, (n, k), generator=gen, device="cuda", dtype=torch.int8)
    sx, sw = torch.ones(t, device="cuda"), torch.ones(n, device="cuda")
    sx[::2] = 0.0        # products of zero, of either sign
    sx[1::4] = 1e-43     # subnormal products
    sx[3::4] = 3e-39     # .. and around the smallest normal number
    old = randn(gen, t, n) * 1e-38
    old[:, 0], old[:, 1], old[:, 2], old[:, 3], old[:, 4] = -0.0, 0.0, float("inf"), float("-inf"), float("nan")
    old[:, 5:8] = 2.0**-149
    old[:, 8] = -(2.0**-126)
    old[:, 9:12] = 3e38
    sw[9] = float("inf")  # an infinite scale: NaN where the token's is zero
    sums = (x.double() @ w.double().T).float() * sx[:, None] * sw
    want = old + sums
    for config in (-1, 512 + 32, 512 + 96, 512 + 256, 1024 + 1, 1024 + 3, 1024 + 16 + 2):
        if 1024 <= config < 1040 and t > 128:
            continue
        for offset in (0, 1):
            y = torch.zeros((t, n + 8), device="cuda")[:, offset : offset + n]
            y.copy_(old)
            ctx.gemm_s8(x, sx, w, sw, y, epilogue=sb.ADD, config=config)
            number = ~torch.isnan(want)
            assert torch.equal(torch.isnan(y), ~number), (config, offset)
            assert torch.equal(y[number].view(torch.int32), want[number].view(torch.int32)), (config, offset)
    ctx.check_status()


@pytest.mark.parametrize("t,c", [(1, 1024), (29, 3584), (900, 2560), (901, 4096), (300, 2563)])
def test_bytes_are_the_float32_formulas(ctx, t, c):
    """Bytes and scales to the bit as IEEE float32 arithmetic gives them on the host: one division 127 / max and one product a value. (The norm's
    scale depends on the order of its sum.)"""
    import numpy as np

    gen = generator(t)
    x = randn(gen, t, c, std=3.0)
    x[:, :: c // 8] *= 12.0
    w, smooth, delta = randn(gen, c, std=0.2), torch.exp(randn(gen, c, std=0.3)), randn(gen, t, c).half()

    def host(u):
        top = np.abs(u).max(1, keepdims=True)
        return np.rint(u * (np.float32(127) / top)).astype(np.int8), (top / np.float32(127))[:, 0]

    for kind in (torch.float16, torch.float32):
        rows = x.to(kind)
        for col_scale in (None, smooth):
            u = rows.float().cpu().numpy()
            if col_scale is not None:
                u = u * col_scale.cpu().numpy()
            want_q, want_s = host(u)
            for _ in range(3):
                q, s = ctx.quantize_tokens_s8(rows, col_scale=col_scale)
                assert np.array_equal(q.cpu().numpy(), want_q) and np.array_equal(s.cpu().numpy(), want_s)
    stream = x.cpu().numpy() + delta.float().cpu().numpy()
    gain = np.float32(1) + w.cpu().numpy()
    for col_scale in (None, smooth):
        want_q, _ = host(stream * (gain if col_scale is None else gain * col_scale.cpu().numpy()))
        first = None
        for _ in range(3):
            q, s = ctx.rms_norm_s8(x.clone(), w, delta=delta, col_scale=col_scale)
            first = s if first is None else first
            assert np.array_equal(q.cpu().numpy(), want_q) and torch.equal(s, first)


def mlp_and_its_error(x, gain, gate, up, down, sx, s_gate, s_up, sa, s_down, eps=1e-6):
    """An MLP in 64 bits on the weights as they were, the variance of each output's error when the rows of its operands are rounded in steps
    sx, s_gate, .. (first order, the rounding errors independent, each with a twelfth of its step's square), and the part of the gate's that
    the rounded activations alone have."""
    x, gain, gate, up, down, sx, s_gate, s_up, sa, s_down = (v.double() for v in (x, gain, gate, up, down, sx, s_gate, s_up, sa, s_down))
    v = x / (x.square().mean(1, keepdim=True) + eps).sqrt() * (1 + gain)
    g, u = v @ gate.T, v @ up.T
    step, energy = sx[:, None].square() / 12, v.square().sum(1, keepdim=True)
    from_x = step * gate.square().sum(1)
    var_g, var_u = from_x + s_gate.square() / 12 * energy, step * up.square().sum(1) + s_up.square() / 12 * energy
    sig = torch.sigmoid(g)
    a = g * sig * u
    var_a = (sig * (1 + g * (1 - sig)) * u).square() * var_g + (g * sig).square() * var_u + sa[:, None].square() / 12
    return v, g, from_x, a @ down.T, var_a @ down.square().T + s_down.square() / 12 * a.square().sum(1, keepdim=True)


def layer_weights(ctx, gen, hidden, inner, std=0.02):
    stacked, down = randn(gen, 2 * inner, hidden, std=std).half(), randn(gen, hidden, inner, std=std).half()
    gate_up, packed_s = ctx.quantize_rows_s8(ctx.pack_gate_up(stacked))
    source = torch.tensor([sb.pack_gate_up_source(p, inner) for p in range(2 * inner)], device="cuda")
    stacked_s = torch.empty_like(packed_s)
    stacked_s[source] = packed_s
    return stacked, down, gate_up, packed_s, stacked_s, *ctx.quantize_rows_s8(down)


# The sum of the squared errors of t rows of outputs that share a row's activations: its expectation is the sum of the variances, and its relative
# spread at most sqrt(2 / t) (the rows are independent, the outputs of a row may not be). Half as much again in the norm is 2.25 in the sum: more
# than 7 spreads at 64 rows. What binary16 and float32 round on the way (the SwiGLU's 2^-11, the weights' none) is under a hundredth of it.
ERROR = 1.5


def test_an_mlps_error_is_that_of_its_roundings(ctx):
    """Against the same weights and activations in 64 bits: the error of the 8-bit MLP is what rounding its operands to bytes makes, no more,
    and at these distributions about three hundredths of its output."""
    t, hidden, inner = 64, 1024, 3584
    gen = generator(31)
    x, gain = randn(gen, t, hidden, std=2.0), randn(gen, hidden, std=0.2)
    stacked, down, gate_up, packed_s, stacked_s, dq, ds = layer_weights(ctx, gen, hidden, inner)
    q, s = ctx.rms_norm_s8(x, gain)
    a = ctx.gemm_s8(q, s, gate_up, packed_s, epilogue=sb.SWIGLU)
    aq, sa = ctx.quantize_tokens_s8(a)
    y = ctx.gemm_s8(aq, sa, dq, ds, y_half=False)
    ctx.check_status()
    *_, want, variance = mlp_and_its_error(x, gain, stacked[:inner], stacked[inner:], down, s, stacked_s[:inner], stacked_s[inner:], sa, ds)
    error = (y.double() - want).norm()
    assert error <= ERROR * variance.sum().sqrt()
    assert error <= 0.05 * want.norm()  # (the sum of the variances is 0.03 to 0.04 squared here: steps of 4 / 127 of a row's root mean square)


def test_the_values_of_the_bytes_show_the_activations_share_of_the_error(ctx):
    """`values` through a multiply that takes binary16: what rounding the activations alone would cost a layer whose weights are not in 8 bits."""
    t, hidden, inner = 64, 1024, 1792
    gen = generator(32)
    x, gain = randn(gen, t, hidden, std=2.0), randn(gen, hidden, std=0.2)
    stacked, down, _, _, stacked_s, _, ds = layer_weights(ctx, gen, hidden, inner)
    values = torch.empty((t, hidden), dtype=torch.float16, device="cuda")
    q, s = ctx.rms_norm_s8(x, gain, values=values)
    got = ctx.gemm_f16(values, stacked[:inner], y_half=False)
    ctx.check_status()
    v, g, from_x, _, _ = mlp_and_its_error(x, gain, stacked[:inner], stacked[inner:], down, s, stacked_s[:inner], stacked_s[inner:], torch.ones(t, device="cuda"), ds)
    expected = from_x.sum().sqrt()
    assert expected / ERROR <= (got.double() - g).norm() <= ERROR * expected


def test_a_trunk_in_eight_bits_beside_the_same_trunk_in_binary16():
    """One layer of random weights, stored both ways: the hidden states differ by the MLP's rounding errors alone."""
    import numpy as np

    base = dict(layers=1, hidden=512, intermediate=1792, vocab=500, attn_q=512, attn_kv=64, dn_in=1024, dn_v_offset=512, dn_v=256, max_call_tokens=300, eps=1e-6, seed=23)
    half, eight = sb.Trunk(0, sb.TrunkConfig(mlp_int8=0, **base)), sb.Trunk(0, sb.TrunkConfig(mlp_int8=2, **base))
    hidden, inner = base["hidden"], base["intermediate"]
    for name in ("embedding", "norm_in", "mix_in", "mix_out", "norm_post"):
        assert np.array_equal(half.weight(name), eight.weight(name))
    tokens = np.random.default_rng(1).integers(0, base["vocab"], 96).astype(np.uint32)
    want, got = (torch.from_numpy(trunk.run(tokens, want_all=True)[1]).double().cuda() for trunk in (half, eight))
    # the stream ahead of the MLP, from the public calls
    ctx = sb.Context(0)
    weight = lambda name, *shape: torch.from_numpy(half.weight(name).copy()).cuda().view(*shape)  # noqa: E731
    x = weight("embedding", base["vocab"], hidden)[torch.from_numpy(tokens.astype(np.int64)).cuda()].float()
    normed = (x / (x.square().mean(1, keepdim=True) + 1e-6).sqrt() * (1 + weight("norm_in", hidden))).half()
    mixed = ctx.gemm_f16(normed, weight("mix_in", base["dn_in"], hidden))
    ctx.gemm_f16(mixed[:, 512:768], weight("mix_out", hidden, 256), x, epilogue=sb.ADD)
    gain = weight("norm_post", hidden)
    q, s = ctx.rms_norm_s8(x, gain)
    scales = torch.from_numpy(eight.weight("gate_up_scales").copy()).cuda()
    a = ctx.gemm_s8(q, s, torch.from_numpy(eight.weight("gate_up").copy()).cuda().view(2 * inner, hidden), scales, epilogue=sb.SWIGLU)
    _, sa = ctx.quantize_tokens_s8(a)
    ctx.check_status()
    packed = weight("gate_up", inner // 64, 2, 64, hidden)
    gate, up = packed[:, 0].reshape(inner, hidden), packed[:, 1].reshape(inner, hidden)
    by_block = scales.view(inner // 64, 2, 64)
    *_, mlp, variance = mlp_and_its_error(x, gain, gate, up, weight("down", hidden, inner), s, by_block[:, 0].reshape(-1), by_block[:, 1].reshape(-1), sa,
                                          torch.from_numpy(eight.weight("down_scales").copy()).cuda())
    expected = variance.sum().sqrt()
    assert (got - want).norm() <= ERROR * expected + 2.0**-9 * mlp.norm()  # (binary16's own roundings in the other trunk)
    assert (got - want).norm() >= expected / ERROR - 2.0**-9 * mlp.norm()
    ctx.close()
