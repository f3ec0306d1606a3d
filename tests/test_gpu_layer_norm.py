"""Layer norm and its gradients against the formulas in float64."""
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
# one value, rows shorter than a piece, every number of lanes to a row, whole and ragged, rows that a workgroup shares and longer ones
SHAPES = [(1, 1), (5, 3), (9, 7), (33, 8), (70, 31), (257, 33), (130, 64), (1000, 100), (515, 128), (64, 250), (40, 256), (300, 515), (61, 602),
          (1, 4096), (7, 2047), (20, 4099), (3, 8192), (2, 12345), (2, 16384), (3, 16385), (2, 70001)]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _values(m, d, g, dtype):
    scale = torch.exp(torch.randn((1, d), generator=g, device="cuda"))
    return (torch.randn((m, d), generator=g, device="cuda") * scale + 0.5 * torch.randn((m, 1), generator=g, device="cuda")).to(dtype)


def _depth(d):
    """Additions one after the other of a row's sum, at most: a lane's own values, then those over lanes and waves."""
    return max(32, (d + 1023) // 1024) + 14


def _check(got, want, size, dtype):
    """Within `size` of the wanted values, and their rounding."""
    bound = size + HALF[dtype] * (want.abs() + size) + LEAST[dtype]
    worst = ((got.double() - want).abs() - bound).max() if want.numel() else torch.zeros(())
    assert float(worst) <= 0, float(worst)


def _forward(x, w, b, eps):
    """(mean, rstd, n, and how far each may be off) in float64."""
    v = x.double()
    depth = _depth(v.shape[1])
    mean = v.mean(1, keepdim=True)
    off_mean = (depth + 2) * U * v.abs().mean(1, keepdim=True)
    var = (v - mean).square().mean(1, keepdim=True)
    # squares of differences that are each off by off_mean and a rounding
    off_var = off_mean.square() + (depth + 6) * U * var + 2 * off_mean * var.sqrt() * (depth + 6) * U
    rstd = 1 / (var + eps).sqrt()
    off_rstd = rstd * (0.5 * off_var / (var + eps) * (1 + off_var / (var + eps)) + 4 * U)
    return mean, off_mean, rstd, off_rstd, (v - mean) * rstd


@pytest.mark.parametrize("m,d", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_forward(m, d, dtype):
    lib = f2cgt_amd.load()
    g = _gen(m + 7 * d)
    x = _values(m, d, g, dtype)
    for w, b in ((torch.randn(d, generator=g, device="cuda").to(dtype), torch.randn(d, generator=g, device="cuda").to(dtype)),
                 (torch.randn(d, generator=g, device="cuda"), None), (None, None)):
        eps = 1e-5
        out, mean, rstd, codes, ex = lib.layer_norm_train(x, w, b, eps, True)
        want_mean, off_mean, want_rstd, off_rstd, n = _forward(x, w, b, eps)
        _check(mean, want_mean[:, 0], off_mean[:, 0], torch.float32)
        _check(rstd, want_rstd[:, 0], off_rstd[:, 0], torch.float32)
        wd = torch.ones(d, device="cuda", dtype=torch.float64) if w is None else w.double()
        want = n * wd + (0 if b is None else b.double())
        size = wd.abs() * (off_mean * want_rstd + n.abs() * (off_rstd / want_rstd + 4 * U)) + 2 * U * ((n * wd).abs() + want.abs())
        _check(out, want, size * 1.01, dtype)
        assert out.dtype == dtype and out.is_contiguous()
        # without statistics, and the checkpoint is pack_activations' own
        assert torch.equal(lib.layer_norm(x, w, b, eps), out)
        assert all(torch.equal(p, q) for p, q in zip(lib.layer_norm_train(x, w, b, eps), (out, mean, rstd)))
        c, e = lib.pack_activations(x)
        assert torch.equal(c, codes) and torch.equal(e, ex)


def _gradients(grad, v, mean, rstd, w):
    """(dx, its size that roundings go by, dw, db and theirs) of float64 inputs."""
    n = (v - mean[:, None]) * rstd[:, None]
    u = grad * w
    d = v.shape[1]
    first, second = u.sum(1, keepdim=True) / d, (u * n).sum(1, keepdim=True) / d
    dx = rstd[:, None] * (u - first - n * second)
    size = rstd[:, None] * (u.abs() + u.abs().mean(1, keepdim=True) + n.abs() * (u * n).abs().mean(1, keepdim=True))
    return dx, size, (grad * n).sum(0), grad.sum(0), (grad * n).abs().sum(0), grad.abs().sum(0)


@pytest.mark.parametrize("m,d", SHAPES + [(5000, 128), (20000, 36), (3000, 1000)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients(m, d, dtype):
    lib = f2cgt_amd.load()
    g = _gen(3 * m + d)
    x = _values(m, d, g, dtype)
    grad = (torch.randn((m, d), generator=g, device="cuda") * torch.exp(torch.randn((m, 1), generator=g, device="cuda"))).to(dtype)
    grad[::5] = 0
    depth = _depth(d)
    down = (m + 63) // 64 + 140                # additions down a column: a workgroup's rows, its groups, the workgroups
    for w in (torch.randn(d, generator=g, device="cuda").to(dtype), torch.randn(d, generator=g, device="cuda"), None):
        _, mean, rstd, codes, ex = lib.layer_norm_train(x, w, None, 1e-5, True)
        wd = torch.ones(d, device="cuda", dtype=torch.float64) if w is None else w.double()
        kind = dtype if w is None else w.dtype
        decoded = lib.unpack_activations(codes, ex)
        for got, v in ((lib.layer_norm_grad(grad, x, mean, rstd, w), x.double()),
                       (lib.layer_norm_packed_grad(grad, codes, ex, mean, rstd, w), decoded.double())):
            dx, size, dw, db, size_w, size_b = _gradients(grad.double(), v, mean.double(), rstd.double(), wd)
            # (n is off by three roundings of it, which sums and products with it take over)
            _check(got[0], dx, (depth + 14) * U * size, dtype)
            _check(got[1], dw, (down + 6) * U * size_w, kind)
            _check(got[2], db, (down + 2) * U * size_b, kind)
            assert got[1].dtype == kind and got[2].dtype == kind
        some = lib.layer_norm_grad(grad, x, mean, rstd, w, False, True)
        full = lib.layer_norm_grad(grad, x, mean, rstd, w)
        assert some[1] is None and torch.equal(some[0], full[0]) and torch.equal(some[2], full[2])
        none = lib.layer_norm_packed_grad(grad, codes, ex, mean, rstd, w, weight_grad=False, bias_grad=False)
        assert none[1] is None and none[2] is None


def test_offsets_that_are_large_and_rows_that_are_equal():
    lib = f2cgt_amd.load()
    g = _gen(1)
    x = torch.randn((50, 300), generator=g, device="cuda") + 4096.0
    want_mean, off_mean, want_rstd, off_rstd, n = _forward(x, None, None, 1e-5)
    out, mean, rstd = lib.layer_norm_train(x)
    _check(mean, want_mean[:, 0], off_mean[:, 0], torch.float32)
    _check(rstd, want_rstd[:, 0], off_rstd[:, 0], torch.float32)
    # whole numbers: the mean of equal values is exact, and so is the norm of no difference
    same = torch.full((4, 256), 3.0, device="cuda")
    w, b = torch.randn(256, generator=g, device="cuda"), torch.randn(256, generator=g, device="cuda")
    assert torch.equal(lib.layer_norm(same, w, b), b.expand(4, 256))
    assert bool(torch.isnan(lib.layer_norm(same, eps=0.0)).all())               # 0 * inf, as the formula has it


@pytest.mark.parametrize("d", [5, 100, 602, 5000, 20000])
def test_rows_with_what_is_no_number_keep_it_to_themselves(d):
    lib = f2cgt_amd.load()
    g = _gen(d)
    x, grad = torch.randn((9, d), generator=g, device="cuda"), torch.randn((9, d), generator=g, device="cuda")
    clean = lib.layer_norm_train(x)
    bad = x.clone()
    bad[2, d // 2], bad[5, 0], bad[7, d - 1] = float("nan"), float("inf"), float("-inf")
    out, mean, rstd = lib.layer_norm_train(bad)
    fine = torch.tensor([0, 1, 3, 4, 6, 8], device="cuda")
    assert torch.equal(out[fine], clean[0][fine]) and torch.equal(rstd[fine], clean[2][fine])
    assert bool(torch.isnan(out[torch.tensor([2, 5, 7], device="cuda")]).all())
    dx, _, _ = lib.layer_norm_grad(grad, bad, mean, rstd)
    assert torch.equal(dx[fine], lib.layer_norm_grad(grad, x, clean[1], clean[2])[0][fine])


def test_strides_shapes_and_empty_rows():
    lib = f2cgt_amd.load()
    g = _gen(2)
    wide = torch.randn((40, 3, 130), generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(100, generator=g, device="cuda")
    view = wide[:, 1, 7:107]                                    # rows 390 apart, at odd places
    grad = wide[:, 2, 3:103]
    dense, dense_grad = view.contiguous(), grad.contiguous()
    out, mean, rstd = lib.layer_norm_train(view, w)
    assert torch.equal(out, lib.layer_norm(dense, w))
    for a, b in zip(lib.layer_norm_grad(grad, view, mean, rstd, w), lib.layer_norm_grad(dense_grad, dense, mean, rstd, w)):
        assert torch.equal(a, b)
    turned = dense.t().contiguous().t()
    assert torch.equal(lib.layer_norm(turned, w), out)
    cube = dense.view(5, 8, 100)
    o3, m3, r3, c3, e3 = lib.layer_norm_train(cube, w, pack=True)
    assert o3.shape == cube.shape and m3.shape == r3.shape == (5, 8) and c3.shape == cube.shape and e3.shape == (5, 8, 4)
    assert torch.equal(o3.view(40, 100), out)
    for a, b in zip(lib.layer_norm_packed_grad(dense_grad.view(5, 8, 100), c3, e3, m3, r3, w),
                    lib.layer_norm_packed_grad(dense_grad, c3.reshape(40, 100), e3.view(40, 4), mean, rstd, w)):
        assert torch.equal(a.view(b.shape), b)
    one = lib.layer_norm(dense[0], w)
    assert one.shape == (100,) and torch.equal(one, out[0])
    none = torch.empty((0, 100), device="cuda")
    assert lib.layer_norm(none).shape == (0, 100)
    dx, dw, db = lib.layer_norm_grad(none, none, torch.empty(0, device="cuda"), torch.empty(0, device="cuda"), w)
    assert dx.shape == (0, 100) and not dw.any() and not db.any()
    spread = torch.ones((), device="cuda").expand(40, 100)       # as a sum's gradient comes
    x = dense.float()
    _, mean, rstd = lib.layer_norm_train(x)
    assert torch.equal(lib.layer_norm_grad(spread, x, mean, rstd)[0], lib.layer_norm_grad(spread.contiguous(), x, mean, rstd)[0])


def test_refusals():
    lib = f2cgt_amd.load()
    x, one = torch.randn(4, 40, device="cuda"), torch.ones(4, device="cuda")
    codes, ex = lib.pack_activations(x)
    bad = [lambda: lib.layer_norm(x.double()), lambda: lib.layer_norm(x, torch.ones(39, device="cuda")),
           lambda: lib.layer_norm(x, torch.ones(40, device="cuda").half()), lambda: lib.layer_norm(x, torch.ones(40)),
           lambda: lib.layer_norm(x.half(), torch.ones(40, device="cuda"), torch.ones(40, device="cuda").half()),
           lambda: lib.layer_norm(x, eps=-1.0), lambda: lib.layer_norm(torch.empty(3, 0, device="cuda")),
           lambda: lib.layer_norm(torch.ones((), device="cuda")),
           lambda: lib.layer_norm_grad(x, x[:3], one, one), lambda: lib.layer_norm_grad(x, x.half(), one, one),
           lambda: lib.layer_norm_grad(x, x, one[:3], one), lambda: lib.layer_norm_grad(x, x, one, one.double()),
           lambda: lib.layer_norm_packed_grad(x, codes[:3], ex[:3], one, one), lambda: lib.layer_norm_packed_grad(x, codes, ex[:, :1], one, one),
           lambda: lib.layer_norm_packed_grad(x, codes, ex.int(), one, one), lambda: lib.layer_norm_packed_grad(x, codes.int(), ex, one, one)]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    leaf = x.clone().requires_grad_()
    for call in (lambda: lib.layer_norm(leaf), lambda: lib.layer_norm_train(x, torch.ones(40, device="cuda", requires_grad=True)),
                 lambda: lib.layer_norm_grad(leaf, x, one, one), lambda: lib.layer_norm_packed_grad(leaf, codes, ex, one, one)):
        with pytest.raises(RuntimeError, match="no_grad"):
            call()
        with torch.no_grad():
            call()


def test_offsets_beyond_32_bits():
    lib = f2cgt_amd.load()
    m, d = 1100000, 2048                                         # 2.25e9 values
    x = torch.ones((m, d), device="cuda", dtype=torch.bfloat16)
    g = _gen(5)
    tail, grad_tail = _values(50, d, g, torch.bfloat16), torch.randn((50, d), generator=g, device="cuda").to(torch.bfloat16)
    x[-50:] = tail
    out, mean, rstd, codes, ex = lib.layer_norm_train(x, pack=True)
    want = lib.layer_norm_train(tail, pack=True)
    for a, b in zip((out, mean, rstd, codes, ex), want):
        assert torch.equal(a[-50:], b)
    assert not out[:-50].any()
    x.zero_()
    x[-50:] = grad_tail
    dx = lib.layer_norm_packed_grad(x, codes, ex, mean, rstd)[0]
    assert torch.equal(dx[-50:], lib.layer_norm_packed_grad(grad_tail, *want[3:], *want[1:3])[0]) and not dx[:-50].any()


def test_module_gradients():
    """The module's gradients are the formula's, and differences' (in float64, of the module's own outputs in steps of 2^-6)."""
    g = _gen(3)
    x = torch.randn((17, 48), generator=g, device="cuda")
    for packed in (False, True):
        norm = pipeline.LayerNorm(48, packed=packed).cuda()
        with torch.no_grad():
            norm.weight.copy_(torch.randn(48, generator=g, device="cuda"))
            norm.bias.copy_(torch.randn(48, generator=g, device="cuda"))
        leaf = x.clone().requires_grad_()
        out = norm(leaf)
        seed = torch.randn(out.shape, generator=g, device="cuda")
        out.backward(seed)
        lib = f2cgt_amd.load()
        v = (lib.unpack_activations(*lib.pack_activations(x)) if packed else x).double()
        _, mean, rstd = lib.layer_norm_train(x)
        dx, size, dw, db, size_w, size_b = _gradients(seed.double(), v, mean.double(), rstd.double(), norm.weight.double().detach())
        _check(leaf.grad, dx, 60 * U * size, torch.float32)
        _check(norm.weight.grad, dw, 160 * U * size_w, torch.float32)
        _check(norm.bias.grad, db, 160 * U * size_b, torch.float32)
        if not packed:
            ref = x.double().requires_grad_()
            torch.nn.functional.layer_norm(ref, (48,), norm.weight.detach().double(), norm.bias.detach().double()).backward(seed.double())
            _check(leaf.grad, ref.grad, 100 * U * size, torch.float32)       # (statistics in fp32: tens of roundings more)
            way = torch.randn(x.shape, generator=g, device="cuda")
            h = 2.0 ** -6
            with torch.no_grad():
                slope = ((norm(x + h * way) - norm(x - h * way)).double() * seed).sum() / (2 * h)
            along = (leaf.grad.double() * way).sum()
            # third derivatives of a norm are of its size: h^2 of it; and a rounding of each output over 2 h
            assert abs(float(slope - along)) <= 10 * h * h * float((seed.abs() * way.abs()).sum()) / x.shape[1] ** 0.5 + 1e-3
    with torch.no_grad():
        assert not norm(x).requires_grad
    frozen = pipeline.LayerNorm(48).cuda().requires_grad_(False)
    leaf = x.clone().requires_grad_()
    frozen(leaf).sum().backward()
    assert leaf.grad is not None and frozen.weight.grad is None
    bare = pipeline.LayerNorm(48, elementwise_affine=False)
    leaf.grad = None
    bare(leaf).square().sum().backward()
    assert leaf.grad is not None
    with pytest.raises(RuntimeError):
        first, = torch.autograd.grad(pipeline.LayerNorm(48).cuda()(leaf).square().sum(), leaf, create_graph=True)
        first.sum().backward()


@pytest.mark.parametrize("m,d", [(1, 4096), (1024, 256), (300, 602), (5, 20000)])
def test_streams_and_captured_graphs(m, d):
    """A captured pass replayed between the program's own work gives the eager results each time."""
    lib = f2cgt_amd.load()
    g = _gen(m + d)
    x, grad, w = (torch.randn(s, generator=g, device="cuda") for s in ((m, d), (m, d), (d,)))

    def both():
        out, mean, rstd, codes, ex = lib.layer_norm_train(x, w, None, 1e-5, True)
        return (out, mean, rstd) + lib.layer_norm_grad(grad, x, mean, rstd, w) + lib.layer_norm_packed_grad(grad, codes, ex, mean, rstd, w)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for i in range(4):
        x.add_(0.25 * i)
        grad.mul_(1.0 + i)
        want = both()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        if i == 0:
            assert all(torch.equal(a, b) for a, b in zip(first, want))
