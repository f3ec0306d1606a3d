"""The bias' gradient of a layer without inputs, over many rows."""
import pytest

torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    import f2cgt_amd

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _bias(grad):
    lib = f2cgt_amd.load()
    m = grad.shape[0]
    codes, exponents = (torch.empty((m, 0), dtype=t, device="cuda") for t in (torch.int8, torch.uint8))
    return lib.packed_linear_grad(grad, codes, exponents, True)[1]


@pytest.mark.parametrize("m", [(1 << 24) + 4096, 40000000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_columns_of_equal_values_grow_beyond_24_bits(m, dtype):
    """2^24 ones and one more are 2^24 in fp32 when they are added one after the other."""
    grad = torch.ones((m, 2), device="cuda", dtype=dtype)
    grad[:, 1] = -0.5
    # (parts of up to 2^24 are exact, and so are their sums, multiples of 32 below 2^29)
    assert _bias(grad).tolist() == [float(m), -0.5 * m]


@pytest.mark.parametrize("m,n", [(0, 3), (1, 1), (15, 70), (16, 64), (17, 65), (4095, 5), (4097, 130), (70001, 9)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_column_sums(m, n, dtype):
    g = torch.Generator(device="cuda").manual_seed(m + n)
    grad = torch.randn((m, n + 2), generator=g, device="cuda").to(dtype)[:, 1:n + 1]
    want, size = grad.double().sum(0), grad.double().abs().sum(0)
    got = _bias(grad)
    assert torch.equal(got, _bias(grad.contiguous()))
    # each addition is off by half a step of a sum that the sizes bound; m of them at most
    assert bool(((got.double() - want).abs() <= m * U * size).all())
