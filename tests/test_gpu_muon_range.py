"""Orthogonalised updates with coefficients near the ends of what is taken: in range in every form."""
import pytest

torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    import f2cgt_amd

from test_gpu_muon_rounding import check  # noqa: E402

pytestmark = pytest.mark.gpu


def _two_lengths(rows, cols, square):
    """An update of two singular values, the squares of which are `square` and 1 - square of the norm's."""
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    left, _ = torch.linalg.qr(torch.randn((rows, 2), generator=g, device="cuda", dtype=torch.float64).cpu())
    right, _ = torch.linalg.qr(torch.randn((cols, 2), generator=g, device="cuda", dtype=torch.float64).cpu())
    # (rows nearly of their own, so that entries of the products are as large as their singular values)
    left = 0.02 * left
    left[0, 0] = left[rows - 1, 1] = 1.0
    lengths = torch.tensor([square, 1 - square], dtype=torch.float64).sqrt()
    return ((left * lengths) @ right.t()).float().cuda()


@pytest.mark.parametrize("rows,cols", [(20, 40), (33, 40), (40, 33), (100, 128), (128, 256), (90, 2800), (200, 333), (600, 700)])
@pytest.mark.parametrize("coefficients", [(7.0, -9.0, 0.0), (7.4, -35.0, 29.1667), (-7.0, 9.0, 0.0)])
def test_a_step_that_turns_directions_round(rows, cols, coefficients):
    """b t + c t^2, of which the product with X is made, is beyond 8 here, and a + b t + c t^2 below 7.5."""
    lib = f2cgt_amd.load()
    for square in (1.0, 0.6):
        u = _two_lengths(rows, cols, square)
        for dtype in (torch.float32, torch.bfloat16):
            x = u.to(dtype)
            got = lib.orthogonalize(x, 1, coefficients)
            assert bool(got.isfinite().all())
            check(got, x, 1, coefficients)
    weight = torch.zeros((rows, cols), device="cuda")
    lib.muon_step([weight], [u], [torch.zeros_like(u)], -1.0, 0.0, 0.0, False, 1, coefficients)
    check(weight, u, 1, coefficients)
