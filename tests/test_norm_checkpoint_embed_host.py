"""The C entry points of layer norm, checkpoints and learnt rows refuse bad calls before any device work (no GPU needed)."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import f2cgt_amd  # noqa: E402
from f2cgt_amd import capi, pipeline  # noqa: E402

INVALID, UNSUPPORTED = -1, -2
P = ctypes.c_void_p(4096)          # (never read)
ODD = ctypes.c_void_p(4097)
F, H, B, D = capi.DT_F32, capi.DT_F16, capi.DT_BF16, capi.DT_F64
I64, I32 = capi.DT_I64, capi.DT_I32


def test_layer_norm():
    lib = capi.lib()
    call = lambda **k: lib.f2cgt_layer_norm(*{**dict(     # noqa: E731
        x=P, dtype=F, ld=8, w=None, b=None, wt=F, out=P, mean=None, rstd=None, codes=None, stride=16, ex=None, m=2, d=8, eps=1e-5, st=None), **k}.values())
    assert call(x=None, out=None, m=0) == 0
    assert call(x=None) == INVALID and call(out=None) == INVALID
    assert call(dtype=D) == UNSUPPORTED and call(dtype=H, w=P, wt=B) == UNSUPPORTED
    assert call(ld=7) == INVALID and call(m=-1) == INVALID and call(d=-1) == INVALID and call(d=0) == INVALID
    assert call(eps=-1.0) == INVALID and call(eps=float("nan")) == INVALID
    assert call(mean=P) == INVALID and call(codes=P) == INVALID and call(codes=P, ex=P, stride=24) == INVALID
    assert call(codes=ctypes.c_void_p(4104), ex=P) == INVALID
    assert call(x=ODD) == INVALID and call(w=ODD) == INVALID
    assert call(d=1 << 24, ld=1 << 24) == UNSUPPORTED and call(m=1 << 31) == UNSUPPORTED


def test_layer_norm_grad():
    lib = capi.lib()
    need = lib.f2cgt_layer_norm_grad_workspace_bytes(F, 100, 40)
    assert need > 0 and lib.f2cgt_layer_norm_grad_workspace_bytes(F, 0, 40) == 0
    call = lambda **k: lib.f2cgt_layer_norm_grad(*{**dict(     # noqa: E731
        g=P, dtype=F, gld=40, x=P, ld=40, codes=None, stride=48, ex=None, mean=P, rstd=P, w=P, wt=F, dx=P, dw=P, db=P, gt=F, ws=P, bytes=need,
        m=100, d=40, st=None), **k}.values())
    for name in ("g", "x", "mean", "rstd", "dx", "ws"):
        assert call(**{name: None}) == INVALID, name
    assert call(bytes=need - 1) == INVALID and b"workspace" in lib.f2cgt_last_error()
    assert call(codes=P, ex=P) == INVALID                       # rows and their checkpoint
    assert call(x=None, codes=P) == INVALID                     # without exponents
    assert call(x=None, codes=P, ex=P, stride=32) == INVALID
    assert call(dtype=D) == UNSUPPORTED and call(gt=D) == UNSUPPORTED and call(dtype=H, wt=B) == UNSUPPORTED
    assert call(gld=39) == INVALID and call(ld=39) == INVALID and call(d=0) == INVALID


def test_checkpoints():
    lib = capi.lib()
    assert lib.f2cgt_pack_activations(None, F, 8, None, 16, None, 0, 8, None) == 0
    assert lib.f2cgt_pack_activations(None, F, 8, None, 16, None, 3, 0, None) == 0
    assert lib.f2cgt_pack_activations(None, F, 8, P, 16, P, 2, 8, None) == INVALID
    assert lib.f2cgt_pack_activations(P, F, 8, P, 16, None, 2, 8, None) == INVALID
    assert lib.f2cgt_pack_activations(P, D, 8, P, 16, P, 2, 8, None) == UNSUPPORTED
    assert lib.f2cgt_pack_activations(P, F, 7, P, 16, P, 2, 8, None) == INVALID
    assert lib.f2cgt_pack_activations(P, F, 8, P, 24, P, 2, 8, None) == UNSUPPORTED
    assert lib.f2cgt_pack_activations(P, F, 8, P, 16, P, -2, 8, None) == INVALID
    assert lib.f2cgt_unpack_activations(P, 16, P, None, F, 2, 8, None) == INVALID
    assert lib.f2cgt_unpack_activations(P, 16, P, P, I32, 2, 8, None) == UNSUPPORTED
    assert lib.f2cgt_unpack_activations(P, 16, P, P, F, 2, 17, None) == UNSUPPORTED
    need = lib.f2cgt_packed_linear_grad_workspace_bytes(F, 100000, 64, 100)
    assert need > 0
    call = lambda **k: lib.f2cgt_packed_linear_grad(*{**dict(     # noqa: E731
        g=P, dtype=F, ld=64, codes=P, stride=112, ex=P, dw=P, db=P, ot=F, ws=P, bytes=need, m=100000, n=64, k=100, st=None), **k}.values())
    for name in ("g", "codes", "ex", "dw", "ws"):
        assert call(**{name: None}) == INVALID, name
    assert call(bytes=need - 1) == INVALID and call(ld=63) == INVALID and call(stride=100) == UNSUPPORTED
    assert call(dtype=D) == UNSUPPORTED and call(ot=I32) == UNSUPPORTED and call(n=-1) == INVALID and call(g=ODD) == INVALID
    assert call(n=0) == 0 and call(k=0, db=None) == 0
    assert call(n=1 << 22, ld=1 << 22) == UNSUPPORTED


def test_learnt_rows():
    lib = capi.lib()
    assert lib.f2cgt_embedding(None, F, 8, None, I64, None, 1.0, 0, 5, 8, None) == 0
    assert lib.f2cgt_embedding(None, F, 8, P, I64, P, 1.0, 2, 5, 8, None) == INVALID
    assert lib.f2cgt_embedding(P, F, 7, P, I64, P, 1.0, 2, 5, 8, None) == INVALID
    assert lib.f2cgt_embedding(P, F, 8, P, capi.DT_I16, P, 1.0, 2, 5, 8, None) == UNSUPPORTED
    assert lib.f2cgt_embedding(P, D, 8, P, I64, P, 1.0, 2, 5, 8, None) == UNSUPPORTED
    assert lib.f2cgt_embedding(P, F, 8, ctypes.c_void_p(4100), I64, P, 1.0, 2, 5, 8, None) == INVALID
    assert lib.f2cgt_embedding(P, F, 8, P, I64, P, 1.0, 2, 1 << 31, 8, None) == UNSUPPORTED
    assert lib.f2cgt_embedding_grad_workspace_bytes(100, 1000, 64) == 0              # picked without a workspace
    need = lib.f2cgt_embedding_grad_workspace_bytes(100000, 1000, 64)
    assert need >= 16 * 100000
    call = lambda **k: lib.f2cgt_embedding_grad(*{**dict(     # noqa: E731
        g=P, dtype=F, ld=64, ids=P, it=I32, out=P, scale=1.0, ws=P, bytes=need, n=100000, rows=1000, d=64, st=None), **k}.values())
    for name in ("g", "ids", "out", "ws"):
        assert call(**{name: None}) == INVALID, name
    assert call(bytes=need - 1) == INVALID and call(ld=63) == INVALID and call(it=capi.DT_U8) == UNSUPPORTED and call(dtype=D) == UNSUPPORTED
    assert call(rows=0) == 0 and call(d=0) == 0 and call(n=-1) == INVALID and call(n=1 << 31) == UNSUPPORTED


def test_host_tensors_are_refused():
    lib = f2cgt_amd.load()
    x, codes, ex = torch.zeros(2, 40), torch.zeros((2, 40), dtype=torch.int8), torch.zeros((2, 2), dtype=torch.uint8)
    ids, one = torch.zeros(2, dtype=torch.int64), torch.zeros(2)
    for call in (lambda: lib.layer_norm(x), lambda: lib.layer_norm_train(x), lambda: lib.layer_norm_grad(x, x, one, one),
                 lambda: lib.layer_norm_packed_grad(x, codes, ex, one, one), lambda: lib.pack_activations(x),
                 lambda: lib.unpack_activations(codes, ex), lambda: lib.packed_linear_grad(x, codes, ex), lambda: lib.embedding(x, ids),
                 lambda: lib.embedding_grad(x, ids, 5)):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            call()


def test_modules_are_built_and_replaced():
    with pytest.raises(ValueError):
        pipeline.LayerNorm((3, 4))
    with pytest.raises(ValueError):
        pipeline.LayerNorm(8)(torch.zeros(2, 9))
    norm = pipeline.LayerNorm(8, packed=True)
    norm.load_state_dict(torch.nn.LayerNorm(8).state_dict())
    assert "packed" in repr(norm)
    plain = torch.nn.Linear(4, 3, bias=False)
    net = torch.nn.Sequential(torch.nn.Linear(8, 4), torch.nn.Sequential(pipeline.LayerNorm(4), plain), torch.nn.ReLU())
    held = dict(net.named_parameters())
    assert pipeline.packed_layers(net) is net
    assert type(net[0]) is pipeline.PackedLinear and type(net[1][1]) is pipeline.PackedLinear and net[1][0].packed
    assert net[1][1].bias is None and all(p is held[name] for name, p in net.named_parameters())
    assert repr(net[1][1]).startswith("PackedLinear(in_features=4, out_features=3, bias=False")
    with torch.no_grad():                                                   # (without gradients it is nn.Linear's own product, on any device)
        x = torch.randn(5, 4)
        assert torch.equal(net[1][1](x), plain(x))
    rows = pipeline.NodeEmbedding(10, 4, scale=2.0)
    assert rows.weight.shape == (10, 4) and "scale=2" in repr(rows) and list(rows.state_dict()) == ["weight"]
