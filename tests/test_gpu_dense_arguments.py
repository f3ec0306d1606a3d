"""What the dense operators do with tensors that are more than their values: differentiated ones, lazily negated ones, ones that share memory."""
import pytest

torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    import f2cgt_amd

pytestmark = pytest.mark.gpu


def _dense(seed=0):
    """x, weight codes and scales, bias, codes of x and their scales."""
    lib = f2cgt_amd.load()
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((5, 40), generator=g, device="cuda")
    weight, weight_scales = lib.quantize_rows(torch.randn((7, 40), generator=g, device="cuda"))
    bias = torch.randn((7,), generator=g, device="cuda")
    return (lib, x, weight, weight_scales, bias) + tuple(lib.quantize_rows(x))


def test_scales_and_biases_that_require_gradients():
    lib, x, weight, weight_scales, bias, codes, scales = _dense()
    want = lib.quantized_linear(x, weight, weight_scales, bias)
    leaf = lambda t: t.clone().requires_grad_()     # noqa: E731
    for call in (lambda: lib.quantized_linear(x, weight, leaf(weight_scales)), lambda: lib.quantized_linear(x, weight, weight_scales, leaf(bias)),
                 lambda: lib.int8_linear(codes, leaf(scales), weight, weight_scales), lambda: lib.int8_linear(codes, scales, weight, leaf(weight_scales)),
                 lambda: lib.int8_linear(codes, scales, weight, weight_scales, leaf(bias)),
                 lambda: lib.int8_linear(codes, scales, weight, weight_scales, torch.nn.Linear(40, 7, device="cuda").bias)):
        with pytest.raises(RuntimeError, match="no_grad"):
            call()
        with torch.no_grad():
            call()
    with torch.no_grad():
        assert torch.equal(lib.quantized_linear(leaf(x), weight, leaf(weight_scales), leaf(bias)), want)
        assert torch.equal(lib.int8_linear(codes, leaf(scales), weight, leaf(weight_scales), leaf(bias)), want)


def test_forward_tangents():
    import torch.autograd.forward_ad as forward
    lib, x, weight, weight_scales, bias, codes, scales = _dense()
    want = lib.quantized_linear(x, weight, weight_scales, bias)
    with forward.dual_level():
        dual = lambda t: forward.make_dual(t, torch.ones_like(t))       # noqa: E731
        for call in (lambda: lib.quantize_rows(dual(x)), lambda: lib.quantized_linear(dual(x), weight, weight_scales, bias),
                     lambda: lib.quantized_linear(x, weight, weight_scales, dual(bias)), lambda: lib.int8_linear(codes, dual(scales), weight, weight_scales),
                     lambda: lib.int8_linear(codes, scales, weight, dual(weight_scales)), lambda: lib.orthogonalize(dual(x)),
                     lambda: lib.muon_step([x.clone()], [dual(x)], [x.clone()], 0.1), lambda: lib.muon_step([dual(x.clone())], [x], [x.clone()], 0.1)):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                call()
        held = dual(x)
        assert torch.equal(lib.quantized_linear(forward.unpack_dual(held).primal, weight, weight_scales, bias), want)
        with forward._set_fwd_grad_enabled(False):
            assert torch.equal(lib.quantized_linear(held, weight, weight_scales, bias), want)
    assert torch.equal(lib.quantized_linear(held, weight, weight_scales, bias), want)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda v: lib.quantized_linear(v, weight, weight_scales, bias), (x,), (x,))


def test_lazily_negated_views():
    lib, x, weight, weight_scales, bias, codes, scales = _dense()
    lazy = lambda t: torch._neg_view((-t).contiguous())      # noqa: E731
    assert lazy(x).is_neg() and torch.equal(lazy(x), x)
    want = lib.quantized_linear(x, weight, weight_scales, bias)
    for a, b, c in ((lazy(x), weight_scales, bias), (x, lazy(weight_scales), bias), (x, weight_scales, lazy(bias)),
                    (lazy(x.t().contiguous()).t(), weight_scales, bias), (lazy(x.reshape(5, 1, 40)).reshape(5, 40), weight_scales, bias)):
        assert torch.equal(lib.quantized_linear(a, weight, b, c), want)
    assert torch.equal(lib.int8_linear(lazy(codes), lazy(scales), lazy(weight), weight_scales, bias), want)
    assert torch.equal(lib.quantize_rows(lazy(x))[0], codes)
    assert torch.equal(lib.orthogonalize(lazy(x)), lib.orthogonalize(x))
    w, d, v = x.clone(), x.flip(0).contiguous(), 0.1 * x.roll(1, 1)
    want_w, want_v = w.clone(), v.clone()
    lib.muon_step([want_w], [d], [want_v], 0.1)
    held_w, held_v = lazy(w), lazy(v)
    lib.muon_step([held_w], [lazy(d)], [held_v], 0.1)
    assert held_w.is_neg() and torch.equal(held_w, want_w) and torch.equal(held_v, want_v)


@pytest.mark.parametrize("rows,cols", [(20, 30), (200, 300)])
def test_steps_of_views_into_one_buffer(rows, cols):
    """Views whose elements lie in between each other's take their step, those that share some are refused before anything is written."""
    lib = f2cgt_amd.load()
    g = torch.Generator(device="cuda").manual_seed(rows)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")       # noqa: E731
    wide = rand(rows, 4 * cols)
    views = [wide[:, i * cols:(i + 1) * cols] for i in range(4)]
    d = rand(rows, cols)
    want = [v.clone() for v in views]
    lib.muon_step(want[:2], [d, d], want[2:], 0.1)
    lib.muon_step(views[:2], [d, d], views[2:], 0.1)
    assert all(torch.equal(a, b) for a, b in zip(views, want))
    deep = rand(rows, cols, 3)                              # every third element
    want = [deep[..., i].clone() for i in range(3)]
    lib.muon_step([want[0]], [want[1]], [want[2]], 0.1)
    lib.muon_step([deep[..., 0]], [deep[..., 1]], [deep[..., 2]], 0.1)
    assert torch.equal(deep[..., 0], want[0]) and torch.equal(deep[..., 2], want[2])
    turned = rand(2 * cols, rows)
    want = [turned[:cols].t().clone(), turned[cols:].t().clone()]
    lib.muon_step([want[0]], [d], [want[1]], 0.1)
    lib.muon_step([turned[:cols].t()], [d], [turned[cols:].t()], 0.1)
    assert torch.equal(turned[:cols].t(), want[0])

    flat = rand(2 * rows * cols)
    one, two = flat[:rows * cols].view(rows, cols), flat[rows * cols:].view(rows, cols)
    late = flat[rows * cols - 1:2 * rows * cols - 1].view(rows, cols)
    square = rand(rows, rows)
    v = rand(rows, cols)
    half = v.view(torch.bfloat16)[:, :cols]                 # (NaNs among them)
    bits = lambda t: t.contiguous().view(torch.uint8)       # noqa: E731
    for w, grads, held in (([one], [v], [v]), ([one], [one], [v]), ([one], [late], [v]), ([one], [v], [late]), ([one, late], [d, d], [v, d.clone()]),
                           ([wide[:, :cols]], [v], [wide[:, cols - 1:2 * cols - 1]]), ([square], [square.clone()], [square.t()]),
                           ([half], [half.clone()], [v]), ([one[:1].expand(rows, cols)], [v], [two]), ([one], [v], [two[:1].expand(rows, cols)])):
        before = [t.clone() for t in w + grads + held]
        with pytest.raises(RuntimeError):
            lib.muon_step(w, grads, held, 0.1)
        assert all(torch.equal(bits(t), bits(b)) for t, b in zip(w + grads + held, before))
    lib.muon_step([one], [v[:1].expand(rows, cols)], [two], 0.1)
