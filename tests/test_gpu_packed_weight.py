"""What may happen to a packed layer's weight between the passes."""
import pytest

torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    import f2cgt_amd
    from f2cgt_amd import pipeline

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def test_a_weight_may_change_where_only_its_own_gradient_is_made():
    """nn.Linear keeps its weight for the input's gradient alone: behind given features it may take a step between the passes."""
    lib = f2cgt_amd.load()
    g = torch.Generator(device="cuda").manual_seed(4)
    x, seed = torch.randn((50, 40), generator=g, device="cuda"), torch.randn((50, 8), generator=g, device="cuda")
    for layer in (torch.nn.Linear(40, 8, device="cuda"), pipeline.PackedLinear(40, 8, device="cuda")):
        out = layer(x)
        with torch.no_grad():
            layer.weight.mul_(2.0)
        out.backward(seed)
    values = lib.unpack_activations(*lib.pack_activations(x)).double()
    # exact products, sixteen rows to an instruction and three planes: a few roundings each
    by = 4 * (3 * 4 + 64) * U * (seed.double().abs().t() @ values.abs())
    assert bool(((layer.weight.grad.double() - seed.double().t() @ values).abs() <= by).all())
    leaf = x.clone().requires_grad_()
    out = layer(leaf)
    with torch.no_grad():
        layer.weight.mul_(2.0)
    with pytest.raises(RuntimeError, match="inplace"):
        out.backward(seed)
