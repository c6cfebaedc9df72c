"""The attention layer's parameters and buffers, without a GPU: what it holds through conversions."""
import copy

import pytest
import torch


def _layer():
    from CudaGaussianVoxelizer import PyGaussianAttention
    return PyGaussianAttention(96, 6, 2, wavelengths=(0.8, 40.0), device="cpu")


@pytest.mark.parametrize("convert", [
    lambda m: m.bfloat16(), lambda m: m.to(torch.bfloat16), lambda m: m.half().float(), lambda m: m.double(),
    lambda m: torch.nn.Sequential(m).to(device="cpu", dtype=torch.bfloat16)[0], lambda m: copy.deepcopy(m).bfloat16(),
], ids=["bfloat16", "to", "half_float", "double", "parent", "copy"])
def test_the_table_of_angles_keeps_its_values(convert):
    """A table rounded to 8 bits would turn a token 40 m away by tenths of a radian: it stays float32, bit for bit, while the
    weights follow the conversion."""
    layer = _layer()
    table = layer.freqs.clone()
    converted = convert(layer)
    assert converted.freqs.dtype == torch.float32 and torch.equal(converted.freqs, table)
    assert converted.to_q.weight.dtype == converted.q_weight.dtype
    assert "freqs" in dict(converted.named_buffers()) and "freqs" not in converted.state_dict()


def test_the_table_follows_the_device():
    layer = _layer().to("meta")
    assert layer.freqs.device.type == "meta" and layer.freqs.dtype == torch.float32
    assert layer.bfloat16().freqs.dtype == torch.float32
