"""Norms, checkpoints and learnt rows where their kernels change form: widths of each layout, cuts of the products, wide rows of
many ids; and calls at once, views, tangents and a captured training step."""
import pytest

torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    import f2cgt_amd
    from f2cgt_amd import pipeline

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}     # half a unit in the last place
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _within(got, want, by, dtype):
    bound = by + HALF[dtype] * (want.abs() + by) + 2.0 ** -25
    assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() - bound).max())


@pytest.mark.parametrize("m,d", [(9, 13), (300, 16), (77, 17), (40, 29), (20, 300), (33, 385), (21, 770), (700, 1030), (9, 1537), (6, 2050),
                                 (5, 4100), (4, 8193), (3, 16383), (1, 1 << 20)])
@pytest.mark.parametrize("dtype", TYPES)
def test_norms_of_each_width(m, d, dtype):
    """A lane adds up to max(32, d / 1024) values one after the other, 10 more over lanes and waves; rows are of values around 1."""
    lib = f2cgt_amd.load()
    g = _gen(d)
    x, grad = (torch.randn((m, d), generator=g, device="cuda").to(dtype) for _ in range(2))
    w, b = (torch.randn(d, generator=g, device="cuda") for _ in range(2))
    depth = max(32, d // 1024 + 1) + 10
    out, mean, rstd, codes, ex = lib.layer_norm_train(x, w, b, 1e-3, True)
    v = x.double()
    # the mean's error goes into each difference, twice that of the squares into the root
    size = v.abs().mean(1, keepdim=True)
    centre = v.mean(1, keepdim=True)
    root = 1 / ((v - centre).square().mean(1, keepdim=True) + 1e-3).sqrt()
    n = (v - centre) * root
    off = (depth + 4) * U * size * root + n.abs() * (depth + 12) * U
    _within(out, n * w.double() + b.double(), 1.01 * (off * w.double().abs()) + 3 * U * (n * w.double()).abs() + 2 * U * b.double().abs(), dtype)
    c, e = lib.pack_activations(x)
    assert torch.equal(c, codes) and torch.equal(e, ex)
    decoded = lib.unpack_activations(codes, ex).double()
    for held, got in ((v, lib.layer_norm_grad(grad, x, mean, rstd, w)), (decoded, lib.layer_norm_packed_grad(grad, codes, ex, mean, rstd, w))):
        n = (held - mean.double()[:, None]) * rstd.double()[:, None]
        u = grad.double() * w.double()
        scale = rstd.double()[:, None]
        want = scale * (u - u.mean(1, keepdim=True) - n * (u * n).mean(1, keepdim=True))
        size = scale * (u.abs() + u.abs().mean(1, keepdim=True) + n.abs() * (u * n).abs().mean(1, keepdim=True))
        _within(got[0], want, (depth + 14) * U * size, dtype)
        _within(got[1], (grad.double() * n).sum(0), (m + 10) * U * (grad.double() * n).abs().sum(0), torch.float32)
        _within(got[2], grad.double().sum(0), (m + 10) * U * grad.double().abs().sum(0), torch.float32)


# tails of steps, fewer rows than exponents that are loaded at once, fewer outputs than a piece, one tile and many, few splits and many
@pytest.mark.parametrize("m,n,k", [(3, 100, 70), (4, 600, 600), (5, 9, 9), (37, 7, 5000), (30000, 5, 33), (9000, 2050, 2047), (20000, 300, 300),
                                   (3001, 1001, 999), (64, 4097, 33), (127, 300, 4097), (2500, 257, 129), (6000, 512, 1024), (700, 64, 64),
                                   (16391, 130, 602), (29, 1, 1000), (8192, 1, 1)])
@pytest.mark.parametrize("dtype", TYPES)
def test_products_of_each_cut(m, n, k, dtype):
    """Products of whole numbers and halves, whose sums stay below 2^23: exact."""
    lib = f2cgt_amd.load()
    g = _gen(m + n + k)
    codes = torch.randint(-15, 16, (m, (k + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.int8)[:, :k]
    ex = torch.randint(126, 129, (m, (k + 31) // 32), generator=g, device="cuda").to(torch.uint8)
    grad = torch.randint(-8, 9, (m, n + 3), generator=g, device="cuda").to(dtype)[:, 2:n + 2]            # (rows that start anywhere)
    values = lib.unpack_activations(codes, ex).double()
    assert 2 * float((grad.double().abs().sum(0).max() * values.abs().max())) < 2 ** 24
    dw, db = lib.packed_linear_grad(grad, codes, ex, True)
    assert torch.equal(dw.double(), grad.double().t().contiguous() @ values) and torch.equal(db.double(), grad.double().sum(0))


@pytest.mark.parametrize("n,rows,d", [(2000, 9000, 257), (2000, 9000, 602), (1500, 2000, 1030), (16384, 20000, 515), (300, 301, 2047)])
@pytest.mark.parametrize("dtype", TYPES)
def test_wide_rows_of_many_ids_among_rows_without(n, rows, d, dtype):
    """Columns that two slices of a row share, in rows whose zeros are written first."""
    lib = f2cgt_amd.load()
    g = _gen(n + d)
    ids = torch.randint(0, rows, (n,), generator=g, device="cuda")
    ids[::2] = rows // 2
    grad = torch.randint(-3, 4, (n, d), generator=g, device="cuda")
    order = torch.argsort(ids)
    want = torch.segment_reduce(grad[order].double(), "sum", lengths=torch.bincount(ids, minlength=rows), axis=0, initial=0.0)
    for _ in range(3):
        # (sums of whole numbers below 2^24, rounded once)
        assert torch.equal(lib.embedding_grad(grad.to(dtype), ids, rows), want.to(dtype))


def test_negated_views_and_tangents():
    lib = f2cgt_amd.load()
    g = _gen(1)
    view = torch.randn((40, 96, 2), generator=g, device="cuda")
    view = torch.view_as_complex(view).conj().imag
    assert view.is_neg()
    x = view.resolve_neg()
    ids = torch.arange(40, device="cuda") % 7
    _, mean, rstd = lib.layer_norm_train(x)
    codes, ex = lib.pack_activations(x)
    # (each the opposite of what the memory holds)
    for op in (lambda t: lib.layer_norm(t, t[0], t[1]), lambda t: lib.layer_norm_grad(t, t, mean, rstd, t[0])[0], lambda t: lib.pack_activations(t)[0],
               lambda t: lib.packed_linear_grad(t, codes, ex)[0], lambda t: lib.embedding(t, ids), lambda t: lib.embedding_grad(t, ids, 7)):
        assert torch.equal(op(view), op(x))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for op in (lambda t: lib.layer_norm(t), lambda t: lib.layer_norm_train(x, t[0]), lambda t: lib.layer_norm_grad(x, t, mean, rstd),
                   lambda t: lib.layer_norm_packed_grad(t, codes, ex, mean, rstd), lambda t: lib.pack_activations(t),
                   lambda t: lib.packed_linear_grad(t, codes, ex), lambda t: lib.embedding(t, ids), lambda t: lib.embedding_grad(t, ids, 7),
                   pipeline.LayerNorm(96, device="cuda"), pipeline.PackedLinear(96, 8, device="cuda")):
            with pytest.raises(RuntimeError):
                op(dual)
        rows = pipeline.NodeEmbedding(7, 3, device="cuda")
        with pytest.raises(RuntimeError):
            lib.embedding(torch.autograd.forward_ad.make_dual(rows.weight.detach(), torch.ones_like(rows.weight)), ids)


def test_calls_at_once():
    """Two streams whose calls overlap: workspaces are each call's own."""
    lib = f2cgt_amd.load()
    g = _gen(2)
    x, grad = (torch.randn((20000, 300), generator=g, device="cuda") for _ in range(2))
    ids = torch.randint(0, 3000, (20000,), generator=g, device="cuda")

    def work(t):
        out, mean, rstd, codes, ex = lib.layer_norm_train(t, pack=True)
        return (out, *lib.layer_norm_packed_grad(grad, codes, ex, mean, rstd), *lib.packed_linear_grad(t, codes, ex, True), lib.embedding_grad(t, ids, 3000))

    want = [work(x), work(grad)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    held = [[], []]
    for _ in range(5):
        for s, t, into in zip(streams, (x, grad), held):
            with torch.cuda.stream(s):
                into.append(work(t))
    torch.cuda.synchronize()
    for results, right in zip(held, want):
        for r in results:
            assert all(torch.equal(a, b) for a, b in zip(r, right))


def test_a_captured_training_step():
    """Forward and backward in a graph, replayed with other ids and gradients: the eager pass' results each time."""
    g = _gen(3)
    rows = pipeline.NodeEmbedding(500, 96, scale=1.5, device="cuda")
    norm = pipeline.LayerNorm(96, packed=True, device="cuda")
    ids, seed = torch.randint(-1, 500, (700,), generator=g, device="cuda"), torch.randn((700, 96), generator=g, device="cuda")
    leaves = [rows.weight, norm.weight, norm.bias]

    def step():
        out = norm(rows(ids))
        return (out.detach(), *torch.autograd.grad(out, leaves, seed))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        ids.copy_(torch.randint(-1, 500, (700,), generator=g, device="cuda"))
        seed.mul_(-0.5)
        with torch.no_grad():
            rows.weight.add_(0.125)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 17, 63, 65, 255, 257, 300, 511, 513, 700, 4100])
@pytest.mark.parametrize("n", [1, 90, 4096, 4097, 16384, 16385, 40000])
def test_tables_of_each_size(n, rows):
    """Ranges of a workgroup from one row up, and the sizes at which ids are sorted rather than picked."""
    lib = f2cgt_amd.load()
    g = _gen(n + rows)
    for d, dtype in ((36, torch.float32), (300, torch.bfloat16)):
        ids = torch.randint(-1, rows, (n,), generator=g, device="cuda")
        grad = torch.randint(-3, 4, (n, d), generator=g, device="cuda")
        grad[ids < 0] = 0
        order = torch.argsort(ids)
        lengths = torch.bincount(ids[ids >= 0], minlength=rows)
        keep = order[int((ids < 0).sum()):]
        want = torch.segment_reduce(grad[keep].double(), "sum", lengths=lengths, axis=0, initial=0.0)
        # (sums of whole numbers below 2^24, rounded once)
        assert torch.equal(lib.embedding_grad(grad.to(dtype), ids, rows), want.to(dtype))
