"""What a trunk's configuration is refused for before a device is touched (so these need none)."""
import numpy as np
import pytest

import sepal_runner_b200 as sb


def config(**kw):
    base = dict(layers=1, hidden=256, intermediate=384, vocab=500, attn_q=256, attn_kv=64, dn_in=512, dn_v_offset=256, dn_v=128, max_call_tokens=300, seed=11)
    base.update(kw)
    return sb.TrunkConfig(**base)


@pytest.mark.parametrize("value", [3, 4, 255, 2**32 - 1])
def test_a_storage_that_does_not_exist(value):
    with pytest.raises(sb.SepalB200Error, match="mlp_int8 is 0"):
        sb.Trunk(0, config(mlp_int8=value))


@pytest.mark.parametrize("eps", [0.0, -1e-6, 1e-31, float("inf"), float("nan")])
def test_an_eps_that_the_norm_to_bytes_does_not_take(eps):
    with pytest.raises(sb.SepalB200Error, match="eps must be a positive number"):
        sb.Trunk(0, config(mlp_int8=2, eps=eps))


def test_widths_whose_sums_do_not_fit():
    for bad in (dict(hidden=1 << 17), dict(intermediate=1 << 17)):
        with pytest.raises(sb.SepalB200Error, match="at most 131071"):
            sb.Trunk(0, config(mlp_int8=2, **bad))


def test_widths():
    for bad in (dict(hidden=200), dict(hidden=0), dict(intermediate=100), dict(intermediate=0), dict(dn_v=64), dict(layers=0), dict(dn_v_offset=448), dict(dn_value_heads=1, dn_key_heads=1)):
        with pytest.raises(sb.SepalB200Error, match="widths must be multiples of 128"):
            sb.Trunk(0, config(**bad))


def test_the_same_with_a_checkpoint(tmp_path):
    path = str(tmp_path / "one.safetensors")
    sb.write_tensor_file(path, {"embed_tokens.weight": np.zeros((500, 256), np.float32)})
    with pytest.raises(sb.SepalB200Error, match="mlp_int8 is 0"):
        sb.Trunk(0, config(mlp_int8=3), sb.Checkpoint(path))
