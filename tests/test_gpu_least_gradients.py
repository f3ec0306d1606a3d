"""The smallest gradients that an 8-bit checkpoint is multiplied with: what is lost of them, and what is not."""
import pytest

torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    import f2cgt_amd

pytestmark = pytest.mark.gpu

LEAST = 2.0 ** -133                                         # bf16's least number: a subnormal one


def _weights(grad, value):
    """dweight [n, 32] of rows of gradients, each against a value of its own in one column."""
    m = grad.shape[0]
    assert m <= 32
    return f2cgt_amd.load().packed_linear_grad(grad, *f2cgt_amd.load().pack_activations(value * torch.eye(32, device="cuda")[:m]))[0][:, :m]


@pytest.mark.parametrize("value", [1.0, 2.0 ** 20])
def test_bits_of_fp32_gradients_from_the_least_bf16_on_are_kept(value):
    """24 bits of a gradient from 2^-110 on reach down to 2^-133; of smaller ones the bits below that are cut off."""
    g = torch.Generator(device="cuda").manual_seed(1)
    bits = torch.randint(1, 1 << 23, (32, 64), generator=g, device="cuda", dtype=torch.int32)
    large = torch.randint(127 - 110, 127 - 90, (32, 64), generator=g, device="cuda", dtype=torch.int32)
    grad = (large << 23 | bits).view(torch.float32)
    assert torch.equal(_weights(grad, value), grad.t() * value)
    small = torch.randint(0, 127 - 110, (32, 64), generator=g, device="cuda", dtype=torch.int32)
    grad = (small << 23 | bits).view(torch.float32)
    lost = grad.t().double() - _weights(grad, value).double() / value
    assert bool((lost >= 0).all()) and bool((lost < LEAST).all()) and bool((lost > 0).any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_subnormal_16_bit_gradients_are_kept(dtype):
    g = torch.Generator(device="cuda").manual_seed(2)
    most = 1 << (7 if dtype == torch.bfloat16 else 10)
    bits = torch.randint(1, most, (32, 64), generator=g, device="cuda", dtype=torch.int16).view(dtype)
    grad = torch.where(torch.rand((32, 64), generator=g, device="cuda") < 0.5, -bits, bits)
    assert torch.equal(_weights(grad, 1.0), grad.t().float())
