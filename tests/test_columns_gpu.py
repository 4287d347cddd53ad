"""Results that are bands of a wider matrix, as narrow as the calls allow (any even number of columns): the columns behind a row are not
written, whichever kernel runs. The TMA drops what lies past a matrix in units of 16 bytes only, so rows that are not whole units must
leave another way."""
import pytest
import torch

import sepal_runner_b200 as sb

pytestmark = pytest.mark.gpu


def band(t, n, dtype, fill=None):
    """[t, n] columns of 16-byte aligned rows, between rows and columns of -0 (which a store of zeros and an addition of zeros both change)."""
    buffer = torch.full((t + 2, (n + 7) // 8 * 8 + 16), -0.0, dtype=dtype, device="cuda")
    y = buffer[1 : t + 1, :n]
    if fill is not None:
        y.copy_(fill)

    def untouched():
        bits = buffer.view(torch.int16 if dtype == torch.float16 else torch.int32).clone()
        expected = bits[0, 0].clone()
        bits[1 : t + 1, :n] = expected
        return bool((bits == expected).all()) and expected.item() < 0

    return y, untouched


CONFIGS = {"f16": [-1, 0, 2, 192, 258, 194, 512 + 64, 512 + 192, 512 + 256, 1024 + 2], "w8g": [-1, 0, 2, 258, 512 + 96, 512 + 192, 512 + 320, 1024 + 2],
           "w8r": [-1, 258, 512 + 160, 1024 + 3]}


@pytest.mark.parametrize("weights", ["f16", "w8g", "w8r"])
@pytest.mark.parametrize("t,n,k", [(129, 2, 128), (150, 130, 256), (200, 258, 1280), (256, 1002, 512), (130, 1004, 512), (200, 1006, 256)])
def test_the_columns_behind_a_row_are_not_written(ctx, weights, t, n, k):
    gen = torch.Generator(device="cuda").manual_seed(t + n)
    x = torch.randn((t, k), generator=gen, device="cuda").half()
    w = torch.randn((n, k), generator=gen, device="cuda") * 0.05
    if weights == "f16":
        w = w.half()
        multiply = lambda **kw: ctx.gemm_f16(x, w, **kw)  # noqa: E731
    elif weights == "w8g":
        placed = ctx.prepare_w8g(*ctx.quantize_group_s8(w))
        multiply = lambda **kw: ctx.gemm_w8g(x, placed, **kw)  # noqa: E731
    else:
        q, sw = ctx.quantize_rows_s8(w.half())
        multiply = lambda **kw: ctx.gemm_w8r(x, q, sw, **kw)  # noqa: E731
    old = torch.randn((t, n), generator=gen, device="cuda")
    for config in CONFIGS[weights]:
        for dtype in (torch.float16, torch.float32):
            plain = multiply(y_half=dtype == torch.float16, config=config)
            y, untouched = band(t, n, dtype)
            multiply(y=y, config=config)
            assert untouched(), (config, dtype)
            assert torch.equal(y, plain), (config, dtype)
            y, untouched = band(t, n, dtype, old)
            multiply(y=y, epilogue=sb.ADD, config=config)
            assert untouched(), (config, dtype)
            added = old.to(dtype).clone()
            multiply(y=added, epilogue=sb.ADD, config=config)
            assert torch.equal(y, added), (config, dtype)
    ctx.check_status()


@pytest.mark.parametrize("t,n,k", [(300, 514, 9728), (1500, 2562, 4096)])
def test_residual_updates_that_would_share_tiles(ctx, t, n, k):
    """Sizes at which the automatic schedule shares tiles between CTA pairs through the TMA's additions, with rows that the TMA does not take."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    x, w = torch.randn((t, k), generator=gen, device="cuda").half(), (torch.randn((n, k), generator=gen, device="cuda") * 0.02).half()
    old = torch.randn((t, n), generator=gen, device="cuda")
    placed = ctx.prepare_w8g(*ctx.quantize_group_s8(w.float()))
    for multiply, weights in ((ctx.gemm_f16, w), (ctx.gemm_w8g, placed)):
        product = multiply(x, weights, y_half=False, config=258)
        y, untouched = band(t, n, torch.float32, old)
        multiply(x, weights, y, epilogue=sb.ADD)
        ctx.check_status()
        assert untouched()
        # two float32 sums of the same k products in different orders: each is off by at most k halves of a step of the sum of magnitudes
        # (the int8 weights' conversion to binary16 moves that by 2^-10 at most), and the addition rounds once more; a part of a tile that
        # is missing or added twice is far beyond it
        dense = w.double() if weights is w else (placed.q.double().view(n, -1, 128) * placed.scales.double()[:, :, None]).view(n, k)
        magnitudes = x.double().abs() @ dense.abs().T
        assert ((y.double() - old.double() - product.double()).abs() <= 2.002 * k * 2.0**-24 * magnitudes + 2.0**-24 * (old.double().abs() + 1.01 * magnitudes)).all()
    with pytest.raises(sb.SepalB200Error, match="whole 16-byte units"):
        ctx.gemm_w8g(x, placed, band(t, n, torch.float32)[0], epilogue=sb.ADD, config=512 + 97)
