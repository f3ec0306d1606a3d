"""Orthogonalised updates and the optimiser's step: against float64, and what is refused."""
import pytest

torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    import f2cgt_amd
    from f2cgt_amd import pipeline

pytestmark = pytest.mark.gpu

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _iterate(u, dtype, steps=5, coefficients=COEFFICIENTS):
    """The definition in `dtype`, on the host."""
    a, b, c = coefficients
    x = u.detach().cpu().to(dtype)
    turned = x.shape[0] > x.shape[1]
    x = x.t() if turned else x
    x = x / (x.norm() + 1e-7)
    for _ in range(steps):
        gram = x @ x.t()
        x = a * x + (b * gram + c * gram @ gram) @ x
    return (x.t() if turned else x).cuda()


def _update(rows, cols, kind, g):
    if kind == "noise":
        return torch.randn((rows, cols), generator=g, device="cuda")
    rank = max(1, min(rows, cols) // 8)
    u = torch.randn((rows, rank), generator=g, device="cuda") @ torch.randn((rank, cols), generator=g, device="cuda")
    return u + 1e-2 * torch.randn((rows, cols), generator=g, device="cuda")


def _check(got, u, dtype, steps=5, coefficients=COEFFICIENTS):
    """Operands of 22 bits instead of the 24 of a float32 evaluation: four times its distance from float64, in the norm; the
    result's own rounding besides."""
    want, single = _iterate(u, torch.float64, steps, coefficients), _iterate(u, torch.float32, steps, coefficients)
    far = float((single.double() - want).norm())
    bound = 4 * far + (2.0 ** -21 + HALF[dtype]) * float(want.norm())
    off = float((got.double() - want).norm())
    assert off <= bound, (off / float(want.norm()), bound / float(want.norm()))


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 2), (3, 40), (16, 16), (31, 33), (32, 32), (33, 31), (47, 256), (64, 64), (65, 65), (64, 200), (100, 128),
          (128, 128), (128, 256), (256, 128), (129, 130), (200, 77), (256, 256), (300, 1000), (1000, 70), (513, 511), (600, 600),
          (20, 4000), (99, 2721), (2100, 64), (200, 1800)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("kind", ["noise", "low"])
def test_one_matrix_against_float64(rows, cols, kind):
    lib = f2cgt_amd.load()
    u = _update(rows, cols, kind, _gen(rows + 3 * cols))
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = u.to(dtype)
        before = x.clone()
        got = lib.orthogonalize(x)
        assert got.shape == x.shape and got.dtype == dtype and torch.equal(x, before)
        _check(got, x, dtype)


@pytest.mark.parametrize("rows,cols", [(1024, 1024), (700, 2100), (2300, 500)])
def test_larger_matrices(rows, cols):
    lib = f2cgt_amd.load()
    u = _update(rows, cols, "low", _gen(rows))
    _check(lib.orthogonalize(u), u, torch.float32)
    _check(lib.orthogonalize(u.bfloat16()), u.bfloat16(), torch.bfloat16)


@pytest.mark.parametrize("rows,cols", [(3970, 4100), (4333, 4000)])
def test_the_largest_tiles(rows, cols):
    # (both references on the device: float64 products of this size take the host minutes)
    lib = f2cgt_amd.load()
    u = _update(rows, cols, "low", _gen(rows))

    def iterate(dtype):
        a, b, c = COEFFICIENTS
        x = u.to(dtype) if rows <= cols else u.t().to(dtype).contiguous()
        x = x / (x.norm() + 1e-7)
        for _ in range(5):
            gram = torch.mm(x, x.t())
            x = a * x + torch.mm(b * gram + c * torch.mm(gram, gram), x)
        return x if rows <= cols else x.t()

    want, single = iterate(torch.float64), iterate(torch.float32)
    got = lib.orthogonalize(u)
    bound = 4 * float((single.double() - want).norm()) + (2.0 ** -21 + HALF[torch.float32]) * float(want.norm())
    assert float((got.double() - want).norm()) <= bound


@pytest.mark.parametrize("count,rows,cols", [(1, 20, 30), (3, 128, 128), (5, 64, 96), (70, 33, 17), (130, 8, 8), (3, 200, 300), (2, 400, 150)])
def test_a_batch_is_its_matrices(count, rows, cols):
    lib = f2cgt_amd.load()
    g = _gen(count)
    u = torch.stack([_update(rows, cols, "low", g) for _ in range(count)])
    got = lib.orthogonalize(u)
    for i in range(count):
        assert torch.equal(got[i], lib.orthogonalize(u[i]))
    _check(got[-1], u[-1], torch.float32)
    two = u[:1].expand(2, rows, cols).reshape(2, 1, rows, cols)
    assert torch.equal(lib.orthogonalize(two)[1, 0], got[0])
    assert torch.equal(lib.orthogonalize(u.mT)[0], lib.orthogonalize(u[0].t().contiguous()))


@pytest.mark.parametrize("steps", [1, 2, 3, 6, 10])
def test_other_numbers_of_steps_and_coefficients(steps):
    lib = f2cgt_amd.load()
    for rows, cols in ((40, 100), (150, 260)):
        u = _update(rows, cols, "noise", _gen(steps))
        _check(lib.orthogonalize(u, steps), u, torch.float32, steps)
        cubic = (1.5, -0.5, 0.0)
        _check(lib.orthogonalize(u, steps, cubic), u, torch.float32, steps, cubic)


def test_sizes_of_updates():
    lib = f2cgt_amd.load()
    for rows, cols in ((30, 50), (140, 300)):
        u = _update(rows, cols, "noise", _gen(2))
        for size in (1e-5, 1e-3, 1e4, 1e18, 1e30):
            _check(lib.orthogonalize(u * size), u.double() * size, torch.float32)
        assert bool((lib.orthogonalize(torch.zeros_like(u)) == 0).all())
        for bad in (float("nan"), float("inf")):
            v = torch.stack([u, u])
            v[1, 3, 4] = bad
            got = lib.orthogonalize(v)
            assert bool(got[1].isnan().all()) and bool(got[0].isfinite().all())
    assert lib.orthogonalize(torch.empty((0, 5), device="cuda")).shape == (0, 5)
    assert lib.orthogonalize(torch.empty((3, 5, 0), device="cuda")).shape == (3, 5, 0)
    assert lib.orthogonalize(torch.empty((0, 5, 6), device="cuda")).shape == (0, 5, 6)


def _step(w, g, v, size, decay, momentum, nesterov, dtype):
    w, g, v = (t.detach().cpu().to(dtype) for t in (w, g, v))
    v = momentum * v + (1 - momentum) * g
    u = momentum * v + (1 - momentum) * g if nesterov else v
    return ((1 - decay) * w - size * _iterate(u, dtype).cpu()).cuda(), v.cuda()


@pytest.mark.parametrize("rows,cols,count", [(1, 1, 1), (256, 128, 2), (47, 256, 3), (100, 128, 2), (300, 200, 2), (65, 1000, 1), (12, 12, 70), (600, 130, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nesterov", [True, False])
def test_the_step_against_float64(rows, cols, count, dtype, nesterov):
    lib = f2cgt_amd.load()
    g = _gen(rows + cols + count)
    weights = [torch.randn((rows, cols), generator=g, device="cuda").to(dtype) for _ in range(count)]
    grads = [_update(rows, cols, "low", g).to(dtype) for _ in range(count)]
    momenta = [torch.randn((rows, cols), generator=g, device="cuda") * 0.1 for _ in range(count)]
    before = [(w.clone(), d.clone(), v.clone()) for w, d, v in zip(weights, grads, momenta)]
    lib.muon_step(weights, grads, momenta, 0.5, 0.1, 0.9, nesterov)
    for i in {0, count // 2, count - 1}:
        w0, g0, v0 = before[i]
        assert torch.equal(grads[i], g0)
        want, held = _step(w0, g0, v0, 0.5, 0.1, 0.9, nesterov, torch.float64)
        single, _ = _step(w0, g0, v0, 0.5, 0.1, 0.9, nesterov, torch.float32)
        # the momentum: two products and a sum, and its factors rounded to float32
        assert bool(((momenta[i].double() - held).abs() <= 5 * 2.0 ** -24 * (v0.double().abs() + g0.double().abs())).all())
        far = float((single.double() - want).norm())
        bound = 4 * far + (2.0 ** -21 + HALF[dtype]) * float(want.norm())
        assert float((weights[i].double() - want).norm()) <= bound


def test_layouts_of_lists_and_versions():
    lib = f2cgt_amd.load()
    g = _gen(4)
    w, d, v = (torch.randn((40, 60), generator=g, device="cuda") for _ in range(3))
    want_w, want_v = w.clone(), v.clone()
    lib.muon_step([want_w], [d], [want_v], 0.1)
    other = [t.t().contiguous().t() for t in (w, d, v)]                  # columns after one another
    lib.muon_step([other[0]], [other[1]], [other[2]], 0.1)
    assert torch.equal(other[0], want_w) and torch.equal(other[2], want_v)
    p = torch.nn.Parameter(w.clone())
    product = (p * p).sum()
    lib.muon_step([p], [d], [v], 0.1)
    assert torch.equal(p.detach(), want_w)
    with pytest.raises(RuntimeError):                                   # the weight that was kept has changed since
        product.backward()
    lib.muon_step([], [], [], 0.1)


@pytest.mark.parametrize("rows,cols", [(30, 40), (100, 128), (70, 3000), (300, 500)])
def test_replayed_in_a_graph(rows, cols):
    lib = f2cgt_amd.load()
    g = _gen(rows)
    w, d, v = (torch.randn((rows, cols), generator=g, device="cuda") for _ in range(3))
    lib.muon_step([w], [d], [v], 0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lib.muon_step([w], [d], [v], 0.1)
    for _ in range(3):
        d.copy_(torch.randn((rows, cols), generator=g, device="cuda"))
        want_w, want_v = w.clone(), v.clone()
        lib.muon_step([want_w], [d], [want_v], 0.1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w, want_w) and torch.equal(v, want_v)


def test_what_is_refused():
    lib = f2cgt_amd.load()
    m = lambda *s: torch.randn(s, device="cuda")    # noqa: E731
    w, d, v = m(4, 5), m(4, 5), m(4, 5)
    for call in (lambda: lib.orthogonalize(w.cpu()), lambda: lib.orthogonalize(w.double()), lambda: lib.orthogonalize(w[0]),
                 lambda: lib.orthogonalize(w, 0), lambda: lib.orthogonalize(w, 101), lambda: lib.orthogonalize(w, 5, (30.0, 0.0, 0.0)),
                 lambda: lib.orthogonalize(w, 5, (float("nan"), 0.0, 0.0)), lambda: lib.orthogonalize(w.clone().requires_grad_()),
                 lambda: lib.orthogonalize(m(65537, 1)),
                 lambda: lib.muon_step([w], [d], [], 0.1), lambda: lib.muon_step([w], [d[:3]], [v], 0.1),
                 lambda: lib.muon_step([w], [d], [v.bfloat16()], 0.1), lambda: lib.muon_step([w, w], [d, d], [v, v.clone()], 0.1),
                 lambda: lib.muon_step([w, m(5, 4)], [d, m(5, 4)], [v, m(5, 4)], 0.1), lambda: lib.muon_step([w[0]], [d[0]], [v[0]], 0.1),
                 lambda: lib.muon_step([w], [d.double()], [v], 0.1), lambda: lib.muon_step([w], [d], [v], 0.1, 1.5),
                 lambda: lib.muon_step([w], [d], [v], 0.1, 0.0, 1.0), lambda: lib.muon_step([w], [d], [v], 0.1, 0.0, 0.9, True, 0)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        pipeline.Muon([torch.nn.Parameter(m(4))])
    with pytest.raises(ValueError):
        pipeline.Muon([torch.nn.Parameter(w)], scale="other")


@pytest.mark.parametrize("scale", ["spectral", "rms"])
def test_the_optimiser_takes_the_steps(scale):
    g = _gen(8)
    shapes = [(30, 20), (20, 30), (30, 20)]
    params = [torch.nn.Parameter(torch.randn(s, generator=g, device="cuda")) for s in shapes]
    opt = pipeline.Muon(params, lr=0.1, momentum=0.8, weight_decay=0.05, scale=scale)
    mirror = [(p.detach().double(), torch.zeros_like(p, dtype=torch.float64)) for p in params]
    for it in range(3):
        for i, p in enumerate(params):
            p.grad = None if (it, i) == (1, 1) else torch.randn(p.shape, generator=g, device="cuda")
            if p.grad is not None:
                size = (max(1.0, p.shape[0] / p.shape[1])) ** 0.5 if scale == "spectral" else 0.2 * max(p.shape) ** 0.5
                mirror[i] = _step(mirror[i][0], p.grad, mirror[i][1], 0.1 * size, 0.1 * 0.05, 0.8, True, torch.float64)
        if it == 2:                         # from a saved state
            saved = {k: v for k, v in opt.state_dict().items()}
            opt = pipeline.Muon(params, lr=0.1, momentum=0.8, weight_decay=0.05, scale=scale)
            opt.load_state_dict(saved)
        opt.step()
    for p, (w, v) in zip(params, mirror):
        # three steps of relative error 1e-4 at most in updates of about one unit of length per singular value
        assert float((p.detach().double() - w).norm() / w.norm()) <= 3e-4
        assert torch.allclose(opt.state[p]["momentum"].double(), v, rtol=1e-5, atol=1e-6)
    half = torch.nn.Parameter(torch.randn((8, 8), generator=g, device="cuda").bfloat16())
    half.grad = torch.randn((8, 8), generator=g, device="cuda").bfloat16()
    opt = pipeline.Muon([half])
    opt.step()
    fresh = pipeline.Muon([half])
    fresh.load_state_dict(opt.state_dict())
    held = fresh.state[half]["momentum"]
    assert held.dtype == torch.float32 and torch.equal(held, opt.state[half]["momentum"])


def test_train_and_serve():
    from f2cgt_amd import train_and_serve
    full, few, equal, losses = train_and_serve.run(nodes=5000, steps=30)
    assert float(losses[-5:].mean()) < 0.5 * float(losses[0])
    assert full > 0.8 and few > full - 0.02 and equal > 0.95


@pytest.mark.parametrize("rows,cols", [(33, 40), (100, 128), (128, 256), (90, 2800), (700, 650)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_special_values_in_every_form(rows, cols, dtype):
    lib = f2cgt_amd.load()
    u = torch.randn((2, rows, cols), generator=_gen(rows), device="cuda").to(dtype)
    assert bool((lib.orthogonalize(torch.zeros_like(u)) == 0).all())
    alone = lib.orthogonalize(u[:1])
    for bad in (float("nan"), float("inf"), -float("inf")):
        v = u.clone()
        v[1, rows - 1, cols - 1] = bad
        got = lib.orthogonalize(v)
        assert bool(got[1].isnan().all()) and bool(got[0].isfinite().all())
        off = float((got[0].double() - alone[0].double()).norm() / alone[0].double().norm())
        assert off <= 2.0 ** -18 + 2 * HALF[dtype] * (2 if dtype == torch.bfloat16 else 1)     # (a batch may be tiled otherwise)
