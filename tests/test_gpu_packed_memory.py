"""What layers with 8-bit checkpoints keep alive between the passes."""
import pytest

torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    from f2cgt_amd import pipeline

pytestmark = pytest.mark.gpu

ROWS, COLS = 8192, 1024
ONE = ROWS * COLS * 4                                       # bytes of a float32 activation
KEEP_RESULT = {"relu": torch.relu, "relu_module": torch.nn.ReLU(), "relu_in_place": torch.nn.ReLU(inplace=True), "tanh": torch.tanh,
               "sigmoid": torch.sigmoid, "softmax": lambda t: torch.softmax(t, 1), "reshaped": lambda t: torch.relu(t).view(2, -1, COLS)}


def _kept(tail, x):
    """(bytes that the graph of tail(x * 1) keeps, its output among them, the output)."""
    before = torch.cuda.memory_allocated()
    out = tail(x * 1.0)                                     # (the product by a number keeps nothing)
    return torch.cuda.memory_allocated() - before, out


def _leaf():
    return torch.randn((ROWS, COLS), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").requires_grad_()


@pytest.fixture(scope="module", autouse=True)
def _library_workspaces():
    """What the library's products allocate once is there before anything is counted."""
    layer, x = torch.nn.Linear(COLS, 64, device="cuda"), _leaf()
    for enabled in (False, True):
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=enabled):
            out = layer(x)
        out.float().sum().backward()
    torch.cuda.synchronize()


@pytest.mark.parametrize("name", KEEP_RESULT)
def test_a_tensor_that_is_kept_anyway_is_not_kept_twice(name):
    """A ReLU's backward pass keeps its result, which is the next layer's input: codes beside it would be a fourth more."""
    act = KEEP_RESULT[name]
    x, plain = _leaf(), torch.nn.Linear(COLS, 64, device="cuda")
    packed = pipeline.PackedLinear.of(plain)
    bytes_plain, out = _kept(lambda t: plain(act(t)), x)
    want = torch.autograd.grad(out.square().sum(), (x, plain.weight, plain.bias))
    del out
    bytes_packed, out = _kept(lambda t: packed(act(t)), x)
    assert bytes_packed <= bytes_plain
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out.square().sum(), (x, packed.weight, packed.bias)), want))
    del out
    norms = [pipeline.LayerNorm(COLS, packed=p, device="cuda") for p in (False, True)]
    of_norms = []
    for norm in norms:
        size, out = _kept(lambda t: norm(act(t)), x)
        of_norms.append((size, torch.autograd.grad(out.square().sum(), (x, norm.weight, norm.bias))))
        del out
    assert of_norms[1][0] <= of_norms[0][0] and all(torch.equal(a, b) for a, b in zip(of_norms[1][1], of_norms[0][1]))


@pytest.mark.parametrize("act", [lambda t: t, torch.nn.functional.gelu, lambda t: torch.nn.functional.dropout(t, 0.5), lambda t: t + t,
                                 lambda t: torch.nn.functional.layer_norm(t, (COLS,))], ids=["product", "gelu", "dropout", "sum", "norm"])
def test_a_tensor_that_nothing_else_keeps_is_kept_in_8_bits(act):
    x, plain = _leaf(), torch.nn.Linear(COLS, 64, device="cuda")
    packed = pipeline.PackedLinear.of(plain)
    # the input in 33 / 128 of its size; up to a tenth for what the allocator rounds up
    assert _kept(lambda t: plain(act(t)), x)[0] - _kept(lambda t: packed(act(t)), x)[0] >= (1 - 33 / 128 - 0.1) * ONE
    norms = [pipeline.LayerNorm(COLS, packed=p, device="cuda") for p in (False, True)]
    assert _kept(lambda t: norms[0](act(t)), x)[0] - _kept(lambda t: norms[1](act(t)), x)[0] >= (1 - 33 / 128 - 0.1) * ONE


def test_a_product_under_autocast_keeps_a_copy_which_codes_take_the_place_of():
    x, plain = _leaf(), torch.nn.Linear(COLS, 64, device="cuda")
    packed = pipeline.PackedLinear.of(plain)

    def after(layer):
        def tail(t):
            with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
                return layer(torch.relu(t))                 # (a ReLU stays in fp32; the layer's copy of it has 16 bits a value)
        return tail
    assert _kept(after(plain), x)[0] - _kept(after(packed), x)[0] >= (0.5 - 33 / 128 - 0.1) * ONE
    half = x.detach().bfloat16().requires_grad_()           # (16-bit inputs go into the product as they are)
    assert _kept(after(packed), half)[0] <= _kept(after(plain), half)[0]


@pytest.mark.parametrize("rows,cols", [(1024, 256), (ROWS, 512)])          # one call for the layer, its operators
@pytest.mark.parametrize("frozen", [False, True])
def test_sage_layers_with_a_relu_before_their_norm(rows, cols, frozen):
    """The ReLU's result is kept by whichever operators make the layer; a packed norm behind it keeps the same tensor."""
    g = torch.Generator(device="cuda").manual_seed(2)
    feats = torch.randn((rows, 128), generator=g, device="cuda")
    csc = torch.arange(rows + 1, device="cuda"), torch.arange(rows, device="cuda")
    torch.manual_seed(3)
    layers = [pipeline.MySAGEConv(128, cols, "mean", None, norm=pipeline.LayerNorm(cols, packed=p), activation=torch.relu).cuda() for p in (False, True)]
    layers[1].load_state_dict(layers[0].state_dict())
    sizes = []
    for layer in layers:
        if frozen:
            layer.fc_neigh.requires_grad_(False)
        size, out = _kept(lambda t: layer(csc, (t, feats)), feats)
        sizes.append((size, torch.autograd.grad(out.square().sum(), [p for p in layer.parameters() if p.requires_grad])))
        del out
    assert sizes[1][0] <= sizes[0][0] and all(torch.equal(a, b) for a, b in zip(sizes[1][1], sizes[0][1]))

