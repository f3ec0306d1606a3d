"""Which modules packed_layers replaces (no GPU needed)."""
import pytest

torch = pytest.importorskip("torch")

from f2cgt_amd import pipeline  # noqa: E402


def test_a_norm_or_a_layer_itself():
    norm = pipeline.LayerNorm(8)
    assert pipeline.packed_layers(norm) is norm and norm.packed
    layer = torch.nn.Linear(8, 4)
    packed = pipeline.packed_layers(layer)
    assert type(packed) is pipeline.PackedLinear and packed.weight is layer.weight and packed.bias is layer.bias
    assert pipeline.packed_layers(packed) is packed


def test_a_layer_under_several_names_stays_one():
    layer = torch.nn.Linear(8, 8)
    net = torch.nn.Sequential(layer, torch.nn.ReLU(), layer, torch.nn.Sequential(layer, pipeline.LayerNorm(8)))
    pipeline.packed_layers(net)
    assert type(net[0]) is pipeline.PackedLinear and net[2] is net[0] and net[3][0] is net[0] and net[3][1].packed
    assert net[0].weight is layer.weight and len(list(net.parameters())) == 4


def test_what_is_no_plain_layer_stays():
    hooked = torch.nn.Linear(4, 4)
    hooked.register_forward_hook(lambda *_: None)
    net = torch.nn.Sequential(hooked, torch.nn.Bilinear(4, 4, 4))
    net.register_module("none", None)
    assert pipeline.packed_layers(net)[0] is hooked and type(net[1]) is torch.nn.Bilinear
