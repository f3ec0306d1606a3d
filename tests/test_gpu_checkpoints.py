"""Activations in 8 bits: the codes and values of the definition, and gradients that are made with them, against float64."""
import pytest

torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    import f2cgt_amd
    from f2cgt_amd import pipeline

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}     # half a unit in the last place
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _two_to(e):
    """2^e in float64 of whole numbers, from its bits (torch.pow is off in the last place for some)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _definition(x):
    """(codes, exponents) of x [m, k] by the definition, in float64 on the CPU."""
    x = x.double().cpu()
    m, k = x.shape
    codes, exponents = torch.zeros((m, k), dtype=torch.int8), torch.zeros((m, (k + 31) // 32), dtype=torch.uint8)
    for j in range(exponents.shape[1]):
        part = x[:, 32 * j:32 * j + 32]
        most = part.abs().amax(1)
        bad = ~torch.isfinite(part).all(1)
        most[bad] = 0
        fraction, power = torch.frexp(most)
        e = torch.clamp(torch.where(fraction > 127 / 128, power - 6, power - 7), min=-126)
        e[most == 0] = -126
        step = _two_to(e)
        code = torch.round(part.nan_to_num(0, 0, 0) / step[:, None])
        limit = torch.where(e == 122, 63.0, 127.0).double()[:, None]
        code = torch.minimum(torch.maximum(code, -limit), limit)
        code[bad] = 0
        codes[:, 32 * j:32 * j + 32] = code.to(torch.int8)
        exponents[:, j] = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return codes, exponents


def _decoded(codes, exponents):
    """The values in float64, on the GPU."""
    step = _two_to(exponents.long() - 127)
    step[exponents == 255] = float("nan")
    return codes.double() * step.repeat_interleave(32, -1)[..., :codes.shape[-1]]


def _same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


SHAPES = [(1, 1), (3, 3), (2, 31), (5, 32), (7, 33), (300, 100), (65, 128), (40, 602), (4, 4099), (1, 16384), (1000, 8), (2, 70000)]


@pytest.mark.parametrize("m,k", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_codes_are_the_definitions(m, k, dtype):
    lib = f2cgt_amd.load()
    g = _gen(m + k)
    x = (torch.randn((m, k), generator=g, device="cuda") * torch.exp(3 * torch.randn((m, k), generator=g, device="cuda"))).to(dtype)
    x[torch.rand((m, k), generator=g, device="cuda") < 0.2] = 0
    codes, ex = lib.pack_activations(x)
    want, want_ex = _definition(x)
    assert torch.equal(codes.cpu(), want) and torch.equal(ex.cpu(), want_ex)
    assert codes.stride(0) % 16 == 0 or m == 1
    values = _decoded(codes, ex)
    for out in TYPES:
        got = lib.unpack_activations(codes, ex, out)
        held = values.clamp(-65504, 65504) if out == torch.float16 else values
        assert got.dtype == out and _same(got, held.to(out))     # (fp16 inputs have infinities among them: NaN)
    if dtype != torch.float16:                                   # every value is a bf16
        assert torch.equal(lib.unpack_activations(codes, ex, torch.bfloat16).double(), values)
    # half a step at most, and a step is at most 1/63.5 of the largest (unless it is the least one)
    step = _two_to(ex.long() - 127).repeat_interleave(32, -1)[:, :k]
    assert bool(((values - x.double()).abs() <= 0.5 * step)[~torch.isnan(values)].all())


def test_borders_of_the_steps():
    lib = f2cgt_amd.load()
    x = torch.zeros((400, 64))
    g = torch.Generator().manual_seed(1)
    edge = 127 * 2.0 ** torch.arange(-140, 121, dtype=torch.float64)
    for r, top in enumerate(edge.tolist()):                      # a group's largest value just below, at and just above 127 steps
        x[r, 0] = torch.tensor(top, dtype=torch.float64).float()
        x[r, 1:32] = torch.rand(31, generator=g) * x[r, 0]
        x[r, 32] = torch.nextafter(x[r, 0], torch.tensor(float("inf")))
        x[r, 33:] = (torch.rand(31, generator=g) - 0.5) * x[r, 0]
    x[300, 0], x[301, 0], x[302, 5] = 3.4028234e38, -3.4028234e38, 3.38e38       # fp32's top
    x[303, 0], x[304, 0], x[305, 40] = 2.0 ** -149, 2.0 ** -127, -(2.0 ** -126)   # its end
    x[306, :32] = (torch.arange(32) - 16 + 0.5) * 2.0 ** -3                        # ties go to even codes
    x[306, 0] = 127 * 2.0 ** -3
    x = x.cuda()
    codes, ex = lib.pack_activations(x)
    want, want_ex = _definition(x)
    assert torch.equal(codes.cpu(), want) and torch.equal(ex.cpu(), want_ex)
    assert bool(torch.isfinite(lib.unpack_activations(codes, ex)).all())
    assert bool(torch.isfinite(lib.unpack_activations(codes, ex, torch.bfloat16)).all())
    half = torch.tensor([[65504.0, -65504.0, 6e-8, 0.0]], device="cuda").half()
    back = lib.unpack_activations(*lib.pack_activations(half), torch.float16)
    assert back.tolist() == [[65504.0, -65504.0, 0.0, 0.0]]


@pytest.mark.parametrize("dtype", TYPES)
def test_groups_that_hold_no_numbers(dtype):
    lib = f2cgt_amd.load()
    x = torch.randn((6, 100), generator=_gen(2), device="cuda").to(dtype)
    clean, clean_ex = lib.pack_activations(x)
    x[1, 40], x[2, 99], x[4, 0] = float("nan"), float("inf"), float("-inf")
    codes, ex = lib.pack_activations(x)
    back = lib.unpack_activations(codes, ex, dtype)
    bad = torch.zeros((6, 100), dtype=torch.bool, device="cuda")
    bad[1, 32:64] = bad[2, 96:] = bad[4, :32] = True
    assert torch.equal(torch.isnan(back), bad) and not codes[bad].any()
    assert torch.equal(back[~bad], lib.unpack_activations(clean, clean_ex, dtype)[~bad])


def _gradient_case(m, n, k, g, dtype, whole=False):
    if whole:
        codes = torch.randint(-15, 16, (m, (k + 15) // 16 * 16 + 16), generator=g, device="cuda", dtype=torch.int8)[:, :k]
        ex = torch.randint(126, 129, (m, (k + 31) // 32), generator=g, device="cuda").to(torch.uint8)
        return torch.randint(-8, 9, (m, n), generator=g, device="cuda").to(dtype), codes, ex
    x = torch.relu(torch.randn((m, k), generator=g, device="cuda")) * torch.exp(torch.randn((1, k), generator=g, device="cuda"))
    grad = torch.randn((m, n), generator=g, device="cuda") * torch.exp(2 * torch.randn((m, 1), generator=g, device="cuda")) * 1e-2
    return grad.to(dtype), *f2cgt_amd.load().pack_activations(x)


def _check_gradient(grad, codes, ex, out_type):
    lib = f2cgt_amd.load()
    m = grad.shape[0]
    dw, db = lib.packed_linear_grad(grad, codes, ex, True, out_type)
    values, wide = _decoded(codes, ex), grad.double()
    want, size = torch.mm(wide.t(), values), torch.mm(wide.abs().t(), values.abs())
    # products are exact; sixteen rows are added by an instruction, to each of up to three planes one after the other: an error of a few roundings each
    steps = 4 * (3 * ((m + 15) // 16) + 64)
    for got, exact, by in ((dw, want, steps * U * size), (db, wide.sum(0), (m + 64) * U * wide.abs().sum(0))):
        bound = by + HALF[out_type] * (exact.abs() + by) + LEAST[out_type]
        assert got.dtype == out_type and bool(((got.double() - exact).abs() <= bound).all()), float(((got.double() - exact).abs() - bound).max())
    only, none = lib.packed_linear_grad(grad, codes, ex, False, out_type)
    assert none is None and torch.equal(only, dw)


# a row and an output, fewer columns than a piece, whole tiles of each size and one more or less, long sums for few outputs
PRODUCTS = [(1, 1, 1), (1, 8, 40), (2, 7, 100), (31, 9, 33), (32, 64, 64), (33, 65, 63), (64, 128, 128), (65, 129, 130), (100, 40, 602), (127, 602, 16),
            (1000, 47, 128), (1024, 256, 128), (4099, 128, 602), (20011, 16, 100), (300, 1000, 515), (513, 4096, 4100), (130, 4100, 4200)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("dtype", TYPES)
def test_weight_gradients(m, n, k, dtype):
    g = _gen(m + 3 * n + 7 * k)
    grad, codes, ex = _gradient_case(m, n, k, g, dtype)
    _check_gradient(grad, codes, ex, torch.float32)
    _check_gradient(grad, codes, ex, dtype)
    # whole numbers come out as they are
    grad, codes, ex = _gradient_case(m, n, k, g, dtype, whole=True)
    lib = f2cgt_amd.load()
    dw, db = lib.packed_linear_grad(grad, codes, ex, True)
    if m <= 30000:                                               # (15 * 2 * 8 * m, in halves, stays below 2^24)
        assert torch.equal(dw.double(), torch.mm(grad.double().t(), _decoded(codes, ex))) and torch.equal(db.double(), grad.double().sum(0))


def test_planes_of_fp32_gradients_are_exact():
    """A gradient whose value needs 24 bits, once, against a code of one: it comes back with every bit, unless the last of its planes,
    2^-23 of it, is below 2^-126, where matrix instructions take bf16 for zero: two planes at most are lost then."""
    lib = f2cgt_amd.load()
    bits = torch.randint(1 << 23, 250 << 23, (64, 64), generator=_gen(9), device="cuda", dtype=torch.int32)
    grad = torch.zeros((4096, 64), device="cuda")
    grad[::64] = bits.view(torch.float32)
    for row in range(0, 4096, 64 * 7):
        x = torch.zeros((4096, 70), device="cuda")
        x[row] = 1.0
        codes, ex = lib.pack_activations(x)
        got, want = lib.packed_linear_grad(grad, codes, ex)[0], grad[row][:, None].expand(64, 70)
        whole = want >= 2.0 ** -103
        assert torch.equal(got[whole], want[whole]) and int(whole.sum()) > 1000
        assert bool(((got.double() - want.double()).abs()[~whole] <= 2 * 2.0 ** -126).all())


def test_gradients_at_views_and_of_nothing():
    lib = f2cgt_amd.load()
    g = _gen(4)
    room = torch.randn((500, 3, 90), generator=g, device="cuda")
    grad = room[:, 1, 5:75]                                      # rows 270 apart
    codes, ex = lib.pack_activations(room[:, 0, 1:])
    want = lib.packed_linear_grad(grad.contiguous(), codes, ex, True)
    odd = torch.zeros((500, 91), dtype=torch.int8, device="cuda")
    odd[:, 1:90] = codes
    for c in (codes, codes.contiguous(), odd[:, 1:90], codes.t().contiguous().t()):
        for gr in (grad, grad.t().contiguous().t()):
            assert all(torch.equal(a, b) for a, b in zip(lib.packed_linear_grad(gr, c, ex, True), want))
        assert torch.equal(lib.unpack_activations(c, ex), lib.unpack_activations(codes, ex))
    cube = lib.packed_linear_grad(grad.reshape(5, 100, 70), codes.contiguous().view(5, 100, 89), ex.view(5, 100, 3), True)
    assert all(torch.equal(a, b) for a, b in zip(cube, want))
    empty = torch.empty((0, 70), device="cuda")
    dw, db = lib.packed_linear_grad(empty, *lib.pack_activations(torch.empty((0, 89), device="cuda")), True)
    assert dw.shape == (70, 89) and not dw.any() and not db.any()
    none, ex0 = lib.pack_activations(torch.empty((500, 0), device="cuda"))
    dw, db = lib.packed_linear_grad(grad, none, ex0, True)
    # (no columns: another order of the same 500 additions, each off by half a step of a sum that Σ|g| bounds)
    assert dw.shape == (70, 0) and bool(((db - want[1]).double().abs() <= 2 * 500 * U * grad.double().abs().sum(0)).all())
    assert lib.packed_linear_grad(empty.new_empty((500, 0)), codes, ex, True)[0].shape == (0, 89)
    assert lib.unpack_activations(none, ex0).shape == (500, 0)


def test_gradients_that_are_no_numbers_stay_in_their_row():
    lib = f2cgt_amd.load()
    g = _gen(6)
    grad, codes, ex = _gradient_case(700, 70, 200, g, torch.float32)
    want = lib.packed_linear_grad(grad, codes, ex, True)
    bad = grad.clone()
    bad[3, 5], bad[699, 69] = float("nan"), float("inf")
    dw, db = lib.packed_linear_grad(bad, codes, ex, True)
    rows = torch.tensor([i for i in range(70) if i not in (5, 69)], device="cuda")
    assert torch.equal(dw[rows], want[0][rows]) and torch.equal(db[rows], want[1][rows])
    assert bool(torch.isnan(dw[5]).all()) and bool(torch.isnan(dw[69]).all())
    ex[698, 1] = 255                                             # a group of no numbers: its columns alone
    codes[698, 32:64] = 0
    dw, _ = lib.packed_linear_grad(grad, codes, ex)
    columns = torch.tensor([j for j in range(200) if not 32 <= j < 64], device="cuda")
    assert torch.equal(dw[:, columns], want[0][:, columns]) and bool(torch.isnan(dw[:, 32:64]).all())


def test_refusals():
    lib = f2cgt_amd.load()
    x = torch.randn(6, 40, device="cuda")
    codes, ex = lib.pack_activations(x)
    for call in (lambda: lib.pack_activations(x.double()), lambda: lib.pack_activations(torch.ones((), device="cuda")),
                 lambda: lib.unpack_activations(codes.int(), ex), lambda: lib.unpack_activations(codes, ex[:, :1]),
                 lambda: lib.unpack_activations(codes, ex.int()), lambda: lib.unpack_activations(codes, ex, torch.float64),
                 lambda: lib.packed_linear_grad(x[:5], codes, ex), lambda: lib.packed_linear_grad(x.double(), codes, ex),
                 lambda: lib.packed_linear_grad(x, codes, ex, False, torch.int32), lambda: lib.packed_linear_grad(x.cpu(), codes, ex)):
        with pytest.raises(RuntimeError):
            call()
    leaf = x.clone().requires_grad_()
    for call in (lambda: lib.pack_activations(leaf), lambda: lib.packed_linear_grad(leaf, codes, ex)):
        with pytest.raises(RuntimeError, match="no_grad"):
            call()


def test_offsets_beyond_32_bits():
    lib = f2cgt_amd.load()
    m, k = 4300000, 520                                          # 2.2e9 codes
    g = _gen(8)
    x = torch.zeros((m, k), device="cuda", dtype=torch.bfloat16)
    tail = torch.randn((100, k), generator=g, device="cuda").to(torch.bfloat16)
    x[-100:] = tail
    codes, ex = lib.pack_activations(x)
    want, want_ex = lib.pack_activations(tail)
    assert torch.equal(codes[-100:], want) and torch.equal(ex[-100:], want_ex) and not codes[:-100].any()
    assert torch.equal(lib.unpack_activations(codes, ex, torch.bfloat16)[-100:], lib.unpack_activations(want, want_ex, torch.bfloat16))
    grad = torch.ones((m, 520), device="cuda", dtype=torch.bfloat16)
    whole = torch.randint(-9, 10, (100, 520), generator=g, device="cuda")
    grad[-100:] = whole.to(torch.bfloat16)
    back = lib.unpack_activations(want, want_ex).double()
    size = torch.mm(whole.double().abs().t(), back.abs())
    dw, _ = lib.packed_linear_grad(grad, codes, ex)
    assert bool(((dw.double() - torch.mm(whole.double().t(), back)).abs() <= 4 * (7 + 64) * U * size).all())


def test_layers_keep_codes_and_train():
    """Outputs and input gradients are nn.Linear's, the weight's gradient is the one at the decoded input."""
    lib = f2cgt_amd.load()
    g = _gen(10)
    x = torch.randn((5, 60, 100), generator=g, device="cuda")
    plain = torch.nn.Linear(100, 70, device="cuda")
    packed = pipeline.PackedLinear.of(plain)
    leaf, other = x.clone().requires_grad_(), x.clone().requires_grad_()
    out, want = packed(leaf), plain(other)
    assert torch.equal(out, want)
    seed = torch.randn(out.shape, generator=g, device="cuda")
    held = [t.dtype for t in out.grad_fn.saved_tensors]
    assert torch.int8 in held and sum(t.numel() for t in out.grad_fn.saved_tensors if t.is_floating_point()) == 7000      # (the weight)
    want_x, = torch.autograd.grad(want, other, seed)
    dx, dw, db = torch.autograd.grad(out, (leaf, packed.weight, packed.bias), seed)
    assert torch.equal(dx, want_x)
    values, flat = lib.unpack_activations(*lib.pack_activations(x)).double().view(300, 100), seed.double().view(300, 70)
    assert bool(((dw.double() - flat.t() @ values).abs() <= 4 * (57 + 65) * U * (flat.abs().t() @ values.abs())).all())
    assert bool(((db.double() - flat.sum(0)).abs() <= 400 * U * flat.abs().sum(0)).all())
    with torch.no_grad():
        assert packed(x).grad_fn is None
    frozen = pipeline.PackedLinear(100, 70, device="cuda")
    frozen.weight.requires_grad_(False)
    frozen(leaf).sum().backward()
    assert frozen.bias.grad is not None and leaf.grad is not None
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = packed(leaf)
    assert out.dtype == torch.bfloat16
    out.float().square().sum().backward()
    assert packed.weight.grad.dtype == torch.float32 and bool(torch.isfinite(packed.weight.grad).all())
    with pytest.raises(RuntimeError):
        first, = torch.autograd.grad(packed(leaf).square().sum(), leaf, create_graph=True)
        first.sum().backward()
    served = pipeline.int8_layers(torch.nn.Sequential(packed))
    assert type(served[0]) is pipeline.Int8Linear


@pytest.mark.parametrize("m,n,k", [(1024, 256, 128), (5000, 128, 602), (300, 2000, 1500)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_graphs(m, n, k, dtype):
    lib = f2cgt_amd.load()
    g = _gen(m)
    x, grad = torch.randn((m, k), generator=g, device="cuda").to(dtype), torch.randn((m, n), generator=g, device="cuda").to(dtype)

    def both():
        codes, ex = lib.pack_activations(x)
        return (lib.unpack_activations(codes, ex, dtype),) + lib.packed_linear_grad(grad, codes, ex, True, dtype)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = both()
    torch.cuda.current_stream().wait_stream(side)
    graphs, held = [], []
    for _ in range(2):                                            # two graphs whose workspaces are their own
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(both())
    for i in range(4):
        x.mul_(1 - 2 * (i % 2))
        grad.add_(0.125 * i)
        want = both()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for h in held for a, b in zip(h, want))
        if i == 0:
            assert all(torch.equal(a, b) for a, b in zip(first, want))
