"""Learnt rows: the lookup's values, the table's gradient against float64, and a training step of all that belongs to it."""
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


def _ids(n, rows, g, kind, dtype=torch.int64):
    if kind == "uniform":
        ids = torch.randint(-2, rows + 2, (n,), generator=g, device="cuda")        # some outside the table
    elif kind == "one":
        ids = torch.full((n,), rows - 1, device="cuda")
    elif kind == "none":
        ids = torch.full((n,), -1, device="cuda")
    elif kind == "order":
        ids = torch.arange(n, device="cuda") % rows
    else:                                                                          # half of them one row, the rest hot ones
        ids = (rows * torch.rand((n,), generator=g, device="cuda") ** 6).long().clamp_(0, rows - 1)
        ids[torch.rand((n,), generator=g, device="cuda") < 0.5] = rows // 3
    return ids.to(dtype)


@pytest.mark.parametrize("n,rows,d", [(1, 1, 1), (5, 3, 3), (7, 10, 7), (100, 50, 16), (333, 1000, 33), (1000, 100, 100), (64, 9, 602), (17, 5, 4099)])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows(n, rows, d, dtype):
    lib = f2cgt_amd.load()
    g = _gen(n + d)
    table = torch.randn((rows, d), generator=g, device="cuda").to(dtype)
    for ids, scale in ((_ids(n, rows, g, "uniform"), 1.0), (_ids(n, rows, g, "uniform", torch.int32), 0.37)):
        out = lib.embedding(table, ids, scale)
        inside = (ids >= 0) & (ids < rows)
        want = (table[ids.long().clamp(0, rows - 1)].float() * scale).to(dtype)
        want[~inside] = 0
        assert out.dtype == dtype and torch.equal(out, want)
    far = torch.tensor([2 ** 40, -2 ** 40, 2 ** 32, 0], device="cuda")
    out = lib.embedding(table, far)
    assert not out[:3].any() and torch.equal(out[3], table[0])
    wide = torch.randn((rows, 2 * d + 3), generator=g, device="cuda").to(dtype)
    ids = _ids(n, rows, g, "order")
    assert torch.equal(lib.embedding(wide[:, 1:d + 1], ids.view(-1, 1)), wide[:, 1:d + 1][ids][:, None])
    assert torch.equal(lib.embedding(wide.t(), torch.zeros(2, dtype=torch.int64, device="cuda")), wide.t()[:1].expand(2, -1))


def _row_sums(values, places, rows):
    """Sums of float64 values over the places of each row (sorted: atomic sums of one row take minutes)."""
    order = torch.argsort(places)
    return torch.segment_reduce(values[order].contiguous(), "sum", lengths=torch.bincount(places, minlength=rows), axis=0, initial=0.0)


def _check_gradient(grad, ids, rows, scale):
    lib = f2cgt_amd.load()
    out = lib.embedding_grad(grad, ids, rows, scale)
    dtype, d = grad.dtype, grad.shape[-1]
    flat, places = grad.reshape(-1, d).double(), ids.reshape(-1).long()
    keep = torch.nonzero((places >= 0) & (places < rows)).flatten()
    want = _row_sums(flat[keep], places[keep], rows) * scale
    size = _row_sums(flat[keep].abs(), places[keep], rows) * abs(scale)
    count = torch.bincount(places[keep], minlength=rows).double()
    by = (count[:, None] + 2) * U * size                           # an addition for each id, the scale and its own rounding
    bound = by + HALF[dtype] * (want.abs() + by) + LEAST[dtype]
    assert out.shape == (rows, d) and out.dtype == dtype
    assert bool(((out.double() - want).abs() <= bound).all()), float(((out.double() - want).abs() - bound).max())
    assert not out[count == 0].any()
    assert torch.equal(lib.embedding_grad(grad, ids, rows, scale), out)
    return out


# few ids, picked by each workgroup, up to the last number that is; more, sorted first, in one digit and several; ranges that end inside
# a workgroup's, columns of more than 64 pieces and of less than one
CASES = [(1, 1, 1), (3, 5, 7), (64, 2, 100), (65, 1, 33), (500, 1000, 128), (1024, 17, 602), (5000, 70000, 16), (11264, 3000, 128), (16383, 1025, 20),
         (16384, 100, 515), (16385, 100, 515), (20000, 1, 64), (30000, 1023, 36), (30001, 1025, 100), (100003, 5000, 33), (200000, 300000, 8), (40000, 64, 1030),
         (70000, 2000, 3)]


@pytest.mark.parametrize("n,rows,d", CASES)
@pytest.mark.parametrize("kind", ["uniform", "hot", "one", "none", "order"])
def test_gradients(n, rows, d, kind):
    g = _gen(n + rows + d)
    ids = _ids(n, rows, g, kind)
    grad = torch.randn((n, d), generator=g, device="cuda")
    _check_gradient(grad, ids, rows, 1.0)
    if kind in ("uniform", "hot"):
        _check_gradient(grad.half(), ids.int(), rows, 0.7)
        _check_gradient(grad.bfloat16(), ids, rows, -3.0)
        whole = torch.randint(-3, 4, (n, d), generator=g, device="cuda").float()         # sums of whole numbers are exact
        inside = (ids >= 0) & (ids < rows)
        want = _row_sums(whole[inside].double(), ids[inside], rows)
        assert torch.equal(f2cgt_amd.load().embedding_grad(whole, ids, rows).double(), want)


def test_orders_shapes_and_nothing():
    lib = f2cgt_amd.load()
    g = _gen(5)
    # up to 64 ids of a row are added in their order
    grad = torch.randn((60, 40), generator=g, device="cuda") * torch.exp(4 * torch.randn((60, 1), generator=g, device="cuda"))
    ids = torch.zeros(60, dtype=torch.int64, device="cuda")
    want = torch.zeros(40, device="cuda")
    for row in grad:
        want = want + row
    assert torch.equal(lib.embedding_grad(grad, ids, 3)[0], want)
    room = torch.randn((300, 7, 90), generator=g, device="cuda")
    ids = torch.randint(0, 50, (300, 7), generator=g, device="cuda")
    out = _check_gradient(room[..., 5:75], ids, 50, 2.0)
    assert torch.equal(lib.embedding_grad(room[..., 5:75].contiguous(), ids, 50, 2.0), out)
    spread = torch.ones((), device="cuda").expand(300, 7, 70)
    assert torch.equal(lib.embedding_grad(spread, ids, 50)[:, 0], torch.bincount(ids.flatten(), minlength=50).float())
    assert not lib.embedding_grad(torch.empty((0, 9), device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), 70).any()
    assert lib.embedding_grad(room[..., :0], ids, 50).shape == (50, 0)
    assert lib.embedding_grad(room, ids, 0).shape == (0, 90)
    assert lib.embedding(torch.empty((0, 9), device="cuda"), ids).shape == (300, 7, 9)
    bad = room[:, 0].clone()
    bad[3, 1] = float("nan")
    out = lib.embedding_grad(bad, torch.arange(300, device="cuda") % 100, 100)
    clean = lib.embedding_grad(room[:, 0], torch.arange(300, device="cuda") % 100, 100)
    where = torch.isnan(out)
    assert int(where.sum()) == 1 and bool(where[3, 1]) and torch.equal(out[~where], clean[~where])
    bad[3, 1] = float("inf")                                       # an id of no row: its gradient is not looked at
    ids = torch.arange(300, device="cuda")
    ids[3] = -1
    assert bool(torch.isfinite(lib.embedding_grad(bad, ids, 300)).all())


def test_refusals():
    lib = f2cgt_amd.load()
    table, ids = torch.randn(6, 40, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    grad = torch.randn(3, 40, device="cuda")
    for call in (lambda: lib.embedding(table.double(), ids), lambda: lib.embedding(table, ids.short()), lambda: lib.embedding(table, ids.float()),
                 lambda: lib.embedding(table[0], ids), lambda: lib.embedding(table, ids.cpu()), lambda: lib.embedding_grad(grad, ids[:2], 6),
                 lambda: lib.embedding_grad(grad, ids, -1), lambda: lib.embedding_grad(grad.double(), ids, 6), lambda: lib.embedding_grad(grad, ids, 1 << 31)):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: lib.embedding(table.clone().requires_grad_(), ids), lambda: lib.embedding_grad(grad.clone().requires_grad_(), ids, 6)):
        with pytest.raises(RuntimeError, match="no_grad"):
            call()


def test_offsets_beyond_32_bits():
    lib = f2cgt_amd.load()
    rows, d = 17000000, 130                                        # 2.2e9 values
    g = _gen(6)
    table = torch.zeros((rows, d), device="cuda", dtype=torch.bfloat16)
    table[-1], table[-2] = 3.0, 5.0
    ids = torch.tensor([rows - 2, rows - 1, rows], device="cuda")
    assert lib.embedding(table, ids)[:, 129].tolist() == [5.0, 3.0, 0.0]
    del table
    for n in (1000, 40000):
        ids = rows - 1 - torch.randint(0, 500, (n,), generator=g, device="cuda")
        whole = torch.randint(-3, 4, (n, d), generator=g, device="cuda")
        out = lib.embedding_grad(whole.to(torch.bfloat16), ids, rows)
        want = torch.zeros((500, d), device="cuda").index_add_(0, ids - (rows - 500), whole.float())
        assert torch.equal(out[-500:], want.to(torch.bfloat16)) and not out[:-500].any()
        del out
    n = 17000000
    ids = torch.full((n,), -1, device="cuda")
    ids[-300:] = torch.arange(300, device="cuda") % 7
    grad = torch.zeros((n, d), device="cuda", dtype=torch.bfloat16)
    grad[-300:] = 1.0
    assert torch.equal(lib.embedding_grad(grad, ids, 10)[:, 1].float(), torch.bincount(ids[-300:], minlength=10).float())


@pytest.mark.parametrize("n,rows", [(3000, 500), (50000, 4000)])
def test_captured_graphs(n, rows):
    lib = f2cgt_amd.load()
    g = _gen(n)
    table, grad = torch.randn((rows, 100), generator=g, device="cuda"), torch.randn((n, 100), generator=g, device="cuda")
    ids = _ids(n, rows, g, "hot")

    def both():
        return lib.embedding(table, ids, 2.0), lib.embedding_grad(grad, ids, rows, 2.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for i in range(4):
        want = both()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        if i == 0:
            assert all(torch.equal(a, b) for a, b in zip(first, want))
        ids.copy_(_ids(n, rows, g, "uniform" if i % 2 else "order"))
        grad.mul_(-1.5)


def test_a_step_of_all_of_them():
    """Learnt rows, a packed layer and a packed norm in one backward pass: every gradient against float64 at the values that the passes hold."""
    lib = f2cgt_amd.load()
    g = _gen(7)
    torch.manual_seed(7)
    rows = pipeline.NodeEmbedding(400, 64, scale=2.0, device="cuda")
    net = pipeline.packed_layers(torch.nn.Sequential(torch.nn.Linear(64, 48, device="cuda"), pipeline.LayerNorm(48, device="cuda")))
    ids = torch.randint(-1, 400, (1500,), generator=g, device="cuda")
    seed = torch.randn((1500, 48), generator=g, device="cuda")
    x = rows(ids)
    h = net[0](x)
    net[1](h).backward(seed)
    with torch.no_grad():
        _, mean, rstd = lib.layer_norm_train(h.detach())
        kept = [lib.unpack_activations(*lib.pack_activations(t.detach())).double() for t in (x, h)]
        w = net[0].weight.double()
        unit = (kept[1] - mean.double()[:, None]) * rstd.double()[:, None]
        part = seed.double() * net[1].weight.double()
        dh = rstd.double()[:, None] * (part - part.mean(1, keepdim=True) - unit * (part * unit).mean(1, keepdim=True))
        size = rstd.double()[:, None] * (part.abs() + part.abs().mean(1, keepdim=True) + unit.abs() * (part * unit).abs().mean(1, keepdim=True))
        dx, size_x = dh @ w, size @ w.abs()
        inside = ids >= 0
        table = torch.zeros((400, 64), device="cuda", dtype=torch.float64).index_add_(0, ids[inside], 2.0 * dx[inside])
        size_table = torch.zeros((400, 64), device="cuda", dtype=torch.float64).index_add_(0, ids[inside], 2.0 * size_x[inside])
    # roundings on the way: 60 for a norm's row, as many as its terms for a product and for a row of the table, 1600 down a column
    for got, want, by in ((rows.weight.grad, table, (60 + 48 + 60) * U * size_table), (net[0].weight.grad, dh.t() @ kept[0], (60 + 1600) * U * (size.t() @ kept[0].abs())),
                          (net[0].bias.grad, dh.sum(0), (60 + 1600) * U * size.sum(0)), (net[1].bias.grad, seed.double().sum(0), 1600 * U * seed.double().abs().sum(0)),
                          (net[1].weight.grad, (seed * unit).sum(0), 1600 * U * (seed * unit).abs().sum(0))):
        assert bool(((got.double() - want).abs() <= by + 1e-12).all()), float(((got.double() - want).abs() - by).max())


@pytest.mark.parametrize("options", [dict(norm=True), dict(packed=True), dict(norm=True, packed=True, learnt=True)], ids=str)
def test_train_and_serve(options):
    from f2cgt_amd import train_and_serve
    full, few, equal, losses = train_and_serve.run(nodes=3000, steps=8, **options)
    assert 0.0 <= full <= 1.0 and 0.0 <= few <= 1.0 and 0.0 <= equal <= 1.0 and bool(torch.isfinite(losses).all())
