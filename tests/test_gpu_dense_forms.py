"""Every tile and form that the dense operators choose by size, with values: a shape for each that no other test takes."""
import pytest

torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    import f2cgt_amd

from test_gpu_muon_rounding import check  # noqa: E402

pytestmark = pytest.mark.gpu

FORMS = [
    (1, 20, 300),           # up to 32 rows, two column strips a wave
    (1, 50, 400),           # a workgroup each, 33 to 64 rows, two column strips a wave
    (1, 1500, 1500),        # symmetric products in 64 x 64 tiles without groups of waves
    (1, 2048, 2048),        # and updates in 64 x 128
    (4, 2048, 512),         # a batch; with groups, updates in 64 x 128
    (1, 3200, 3200),        # symmetric products in 128 x 128 tiles
    (1, 3970, 4100),        # in 192 x 192; updates in 128 x 128
    (2, 4100, 3970),        # a batch in 128 x 128, turned
]


@pytest.mark.parametrize("count,rows,cols", FORMS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_updates(count, rows, cols, dtype):
    lib = f2cgt_amd.load()
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    rank = max(1, min(rows, cols) // 8)
    u = torch.stack([torch.randn((rows, rank), generator=g, device="cuda") @ torch.randn((rank, cols), generator=g, device="cuda") +
                     1e-2 * torch.randn((rows, cols), generator=g, device="cuda") for _ in range(count)]).to(dtype)
    got = lib.orthogonalize(u)
    for i in {0, count - 1}:
        check(got[i], u[i], where="cuda")


def _whole(rows, columns, g):
    """Codes below 41, of which no sum of these sizes goes beyond 2^24."""
    return torch.randint(-40, 41, (rows, (columns + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.int8)[:, :columns]


@pytest.mark.parametrize("m,k,n", [(4099, 4096, 4096),      # the rows left over in a launch of their own
                                   (4111, 4100, 4093), (5, 1000, 8200), (16, 2048, 16385)])     # few tokens, 32 outputs a workgroup
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_products(m, k, n, dtype):
    lib = f2cgt_amd.load()
    g = torch.Generator(device="cuda").manual_seed(m + n)
    codes, weight = _whole(m, k, g), _whole(n, k, g)
    scales = 2.0 ** torch.randint(-3, 4, (m,), generator=g, device="cuda").float()
    weight_scales = 2.0 ** torch.randint(-3, 4, (n,), generator=g, device="cuda").float()
    bias = torch.randint(-9, 10, (n,), generator=g, device="cuda").float()
    out = lib.int8_linear(codes, scales, weight, weight_scales, bias, False, dtype)
    product = (codes.double() @ weight.double().t().contiguous()) * (scales.double()[:, None] * weight_scales.double())
    # (scales are powers of two: the product is exact, the bias' addition rounded to float32)
    assert torch.equal(out, (product.float() + bias).to(dtype))


@pytest.mark.parametrize("m,k,n", [(300, 200, 130), (17, 129, 256), (1000, 256, 33)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_rows_of_two_lines_coded_where_they_are_multiplied(m, k, n, dtype):
    lib = f2cgt_amd.load()
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    x = torch.randn((m, k), generator=g, device="cuda").to(dtype)
    weight, weight_scales = lib.quantize_rows(torch.randn((n, k), generator=g, device="cuda"))
    codes, scales = lib.quantize_rows(x)
    got = lib.quantized_linear(x, weight, weight_scales)
    # whole sums below 2^23 times a product of scales, in float32
    want = (codes.double() @ weight.double().t().contiguous()).float() * (scales[:, None] * weight_scales)
    assert torch.equal(got, want.to(dtype))
