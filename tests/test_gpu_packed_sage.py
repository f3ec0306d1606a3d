"""MySAGEConv with packed layers: its one-call product without gradients, and every gradient of a step against float64."""
import pytest

torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    import f2cgt_amd
    from f2cgt_amd import pipeline

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
NODES, DIM, OUT, ROWS, FANOUT = 500, 64, 48, 300, 5


def _manager(g):
    features = torch.randn((NODES, DIM), generator=g, device="cuda")
    table, codebooks = pipeline.sq_compress(features, 4, DIM, sample_index=torch.arange(NODES))
    return pipeline.CompressionManager({"methods": ["sq"], "feat_dim": DIM, "configs": [(DIM, 4)], "codebooks": [codebooks],
                                        "compression_data": table}, fusion=True)


def _layer(g, activation, norm=True):
    manager = _manager(g)
    layer = pipeline.MySAGEConv(DIM, OUT, "mean", manager, norm=pipeline.LayerNorm(OUT) if norm else None, activation=activation).cuda()
    if norm:
        with torch.no_grad():
            layer.norm.weight.copy_(torch.randn(OUT, generator=g, device="cuda"))
    seeds = torch.randint(0, NODES, (ROWS,), generator=g, device="cuda")
    ids = torch.randint(0, NODES, (ROWS * FANOUT,), generator=g, device="cuda")
    return manager, layer, seeds, (torch.arange(0, ROWS * FANOUT + 1, FANOUT, device="cuda"), ids)


@pytest.mark.parametrize("activation", [None, torch.relu], ids=["plain", "relu"])
def test_every_gradient_of_a_step(activation):
    lib = f2cgt_amd.load()
    g = torch.Generator(device="cuda").manual_seed(5)
    torch.manual_seed(5)
    manager, layer, seeds, csc = _layer(g, activation)
    pipeline.packed_layers(layer)
    assert type(layer.fc_self) is type(layer.fc_neigh) is pipeline.PackedLinear and layer.norm.packed
    rows = pipeline.NodeEmbedding(NODES, DIM, scale=0.5, device="cuda")
    seen = {}
    for name in ("fc_self", "fc_neigh", "norm"):
        getattr(layer, name).register_forward_pre_hook(lambda m, args, name=name: seen.__setitem__(name, args[0].detach().clone()))
    seed = torch.randn((ROWS, OUT), generator=g, device="cuda") * torch.exp(torch.randn((ROWS, 1), generator=g, device="cuda"))
    layer(csc, (manager._decompress(0, manager.data[seeds]) + rows(seeds), manager.data.data)).backward(seed)
    with torch.no_grad():
        held = {name: lib.unpack_activations(*lib.pack_activations(t)).double() for name, t in seen.items()}
        _, mean, rstd = lib.layer_norm_train(seen["norm"])
        mask = torch.ones((ROWS, OUT), device="cuda", dtype=torch.float64)
        if activation is not None:                          # (what the ReLU keeps is what the norm has, uncoded)
            held["norm"] = seen["norm"].double()
            mask = (seen["norm"] > 0).double()
        unit = (held["norm"] - mean.double()[:, None]) * rstd.double()[:, None]
        grad = seed.double()
        part = grad * layer.norm.weight.double()
        dh = rstd.double()[:, None] * (part - part.mean(1, keepdim=True) - unit * (part * unit).mean(1, keepdim=True)) * mask
        size = rstd.double()[:, None] * (part.abs() + part.abs().mean(1, keepdim=True) + unit.abs() * (part * unit).abs().mean(1, keepdim=True)) * mask
        w = layer.fc_self.weight.double()
        table, size_table = (torch.zeros((NODES, DIM), device="cuda", dtype=torch.float64).index_add_(0, seeds, 0.5 * t) for t in (dh @ w, size @ w.abs()))
    # roundings on the way: 60 for a norm's row (32 additions of a lane, 14 over lanes, 14 of the formula), as many as its terms for a product and a
    # row of the table, 300 down a column, and for the packed products three planes' sums of them
    norm, down = 60, ROWS + 10
    for got, want, by in ((layer.fc_self.weight.grad, dh.t() @ held["fc_self"], (norm + 3 * down) * U * (size.t() @ held["fc_self"].abs())),
                          (layer.fc_neigh.weight.grad, dh.t() @ held["fc_neigh"], (norm + 3 * down) * U * (size.t() @ held["fc_neigh"].abs())),
                          (layer.fc_self.bias.grad, dh.sum(0), (norm + down) * U * size.sum(0)),
                          (layer.norm.weight.grad, (grad * unit).sum(0), (6 + down) * U * (grad * unit).abs().sum(0)),
                          (layer.norm.bias.grad, grad.sum(0), down * U * grad.abs().sum(0)),
                          (rows.weight.grad, table, (norm + OUT + 60) * U * size_table)):
        assert float(want.abs().max()) > 0
        assert bool(((got.double() - want).abs() <= by + 1e-12).all()), float(((got.double() - want).abs() - by).max())


@pytest.mark.parametrize("activation", [None, torch.relu], ids=["plain", "relu"])
def test_packed_layers_answer_with_one_call_without_gradients(activation, monkeypatch):
    lib = f2cgt_amd.load()
    g = torch.Generator(device="cuda").manual_seed(6)
    manager, layer, seeds, csc = _layer(g, activation, norm=False)
    feat = (manager._decompress(0, manager.data[seeds]), manager.data.data)
    made = []
    original = lib.sage_linear

    def counted(*args):
        out = original(*args)
        made.append(out is not None)
        return out

    monkeypatch.setattr(lib, "sage_linear", counted)
    with torch.no_grad():
        want = layer(csc, feat)
        assert made == [True]
        pipeline.packed_layers(layer)
        assert torch.equal(layer(csc, feat), want) and made == [True, True]
    assert torch.equal(layer(csc, feat), want) and made == [True, True]          # with gradients the checkpoints are made
    for p in (layer.fc_self.weight, layer.fc_neigh.weight):
        p.requires_grad_(False)
    assert torch.equal(layer(csc, feat), want) and made == [True] * 3            # frozen weights have none
    layer.fc_neigh.register_forward_hook(lambda *_: None)                        # (a layer with a hook is called)
    with torch.no_grad():
        assert torch.equal(layer(csc, feat), want) and made == [True] * 3
