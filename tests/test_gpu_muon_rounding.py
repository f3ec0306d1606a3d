"""Orthogonalised updates: what a result adds to its own rounding, for updates of every structure, numbers of steps and
coefficients."""
import pytest

torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    import f2cgt_amd

pytestmark = pytest.mark.gpu

DEFAULT = (3.4445, -4.7750, 2.0315)
STEEP = (3.9505, -6.3029, 2.6377)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _two_planes(x):
    """An operand of the products: two fp16 numbers, times 4096."""
    x = x.float() * 4096
    hi = x.half().float()
    return (hi.double() + (x - hi).half().double()) / 4096


def _iterate(u, steps, coefficients, operand=lambda x: x, dtype=torch.float64, where="cpu"):
    """The definition in `dtype`; `operand` is done to what goes into a product."""
    a, b, c = coefficients
    x = u.detach().to(where).to(dtype)
    turned = x.shape[0] > x.shape[1]
    x = x.t() if turned else x
    x = x / (x.norm() + 1e-7)
    for _ in range(steps):
        z = operand(x)
        gram = z @ z.t()
        y = operand(gram)
        x = a * z + operand(b * y + c * y @ y) @ z
    return x.t() if turned else x


def check(got, u, steps=5, coefficients=DEFAULT, where="cpu"):
    """Operands of two planes cost `far`, and as much for the products' fourth part, which is left out.  Each product's fp32 sum is
    off too, and later steps multiply that as they do in a float32 evaluation, which adds its own; four times its distance
    `single` is what the other tests of these results take: E = 2 far + 4 single + 2^-20 of the norm.  A rounded y is as near to
    `want` as the rounded `want`, but for 2 |y - want|, value by value (it is rounded otherwise only where `want` is as near to the
    middle of two neighbours): E twice beside the result's own rounding."""
    want = _iterate(u, steps, coefficients, where=where)
    norm = float(want.norm())
    far = float((_iterate(u, steps, coefficients, _two_planes, where=where) - want).norm())
    single = float((_iterate(u, steps, coefficients, dtype=torch.float32, where=where).double() - want).norm())
    error = 2 * far + 4 * single + 2.0 ** -20 * norm
    own = float((want.to(got.dtype).double() - want).norm())
    off = float((got.to(where).double() - want).norm())
    assert off <= own + 2 * error, (off / norm, own / norm, error / norm)


def _update(rows, cols, kind):
    g = _gen(rows + 3 * cols)
    if kind == "noise":
        return torch.randn((rows, cols), generator=g, device="cuda")
    if kind == "low":
        rank = max(1, min(rows, cols) // 8)
        u = torch.randn((rows, rank), generator=g, device="cuda") @ torch.randn((rank, cols), generator=g, device="cuda")
        return u + 1e-2 * torch.randn((rows, cols), generator=g, device="cuda")
    whole = lambda n, top: torch.randint(1, top, (n,), generator=g, device="cuda").float()    # noqa: E731
    if kind == "outer":                     # few different values: their roundings do not average out
        return whole(rows, 4)[:, None] * whole(cols, 6)[None, :]
    u = torch.zeros((rows, cols), device="cuda")
    if kind == "column":
        u[:, cols // 2] = whole(rows, 8)
    else:
        u[rows // 3] = whole(cols, 8)
    return u


@pytest.mark.parametrize("rows,cols", [(20, 50), (50, 40), (64, 64), (64, 200), (50, 400), (128, 128), (130, 130), (500, 500), (90, 2800), (300, 700)])
@pytest.mark.parametrize("kind", ["noise", "low", "outer", "column", "row"])
def test_results_are_their_own_rounding(rows, cols, kind):
    lib = f2cgt_amd.load()
    u = _update(rows, cols, kind)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = u.to(dtype)
        check(lib.orthogonalize(x), x)


@pytest.mark.parametrize("rows,cols", [(64, 200), (30, 60), (300, 500)])
@pytest.mark.parametrize("steps,coefficients", [(1, DEFAULT), (10, DEFAULT), (30, DEFAULT), (5, STEEP), (10, STEEP), (8, (1.5, -0.5, 0.0))])
def test_other_steps_and_coefficients(rows, cols, steps, coefficients):
    lib = f2cgt_amd.load()
    for kind in ("noise", "low"):
        u = _update(rows, cols, kind)
        for dtype in (torch.bfloat16, torch.float16, torch.float32):
            x = u.to(dtype)
            check(lib.orthogonalize(x, steps, coefficients), x, steps, coefficients)
