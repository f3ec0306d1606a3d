"""The dense operators' C entry points refuse bad calls before any device work (no GPU needed)."""
import ctypes

import pytest

pytest.importorskip("torch")

from f2cgt_amd import capi  # noqa: E402

INVALID, UNSUPPORTED = -1, -2
P = ctypes.c_void_p(4096)          # (never read)
F, H, B = capi.DT_F32, capi.DT_F16, capi.DT_BF16


def _coefficients(*c):
    return (ctypes.c_float * 3)(*c)


def test_rows_and_products_in_8_bits():
    lib = capi.lib()
    assert lib.f2cgt_quantize_rows(None, F, 8, None, 16, None, 0, 8, None) == 0
    assert lib.f2cgt_quantize_rows(None, F, 8, P, 16, P, 2, 8, None) == INVALID
    assert lib.f2cgt_quantize_rows(P, capi.DT_F64, 8, P, 16, P, 2, 8, None) == UNSUPPORTED
    assert lib.f2cgt_quantize_rows(P, F, 7, P, 16, P, 2, 8, None) == INVALID            # rows overlap
    assert lib.f2cgt_quantize_rows(P, F, 8, P, 7, P, 2, 8, None) == INVALID
    assert lib.f2cgt_quantize_rows(P, F, 8, P, 16, P, -1, 8, None) == INVALID
    assert lib.f2cgt_quantize_rows(P, F, 1 << 17, P, 1 << 17, P, 2, 1 << 17, None) == UNSUPPORTED
    call = lib.f2cgt_int8_linear
    assert call(None, 16, None, None, 16, None, None, None, F, 0, 4, 16, 0, None) == 0
    assert call(None, 16, None, None, 16, None, None, None, F, 4, 0, 16, 0, None) == 0
    assert call(None, 16, P, P, 16, P, None, P, F, 4, 4, 16, 0, None) == INVALID
    assert call(P, 16, P, P, 16, P, None, None, F, 4, 4, 16, 0, None) == INVALID
    assert call(P, 16, P, P, 16, P, None, P, capi.DT_F64, 4, 4, 16, 0, None) == UNSUPPORTED
    assert call(P, 24, P, P, 16, P, None, P, F, 4, 4, 16, 0, None) == UNSUPPORTED       # rows of codes at multiples of 8
    assert call(P, 16, P, ctypes.c_void_p(4104), 16, P, None, P, F, 4, 4, 16, 0, None) == UNSUPPORTED
    assert call(P, 16, P, P, 1 << 23, P, None, P, F, 4, 4, 16, 0, None) == UNSUPPORTED
    assert b"16 bytes" in lib.f2cgt_last_error()
    assert call(P, 1 << 17, P, P, 1 << 17, P, None, P, F, 4, 4, 1 << 17, 0, None) == UNSUPPORTED    # sums beyond 32 bits
    one = lib.f2cgt_quantized_linear
    assert one(None, F, 16, None, 16, None, None, None, None, 0, 0, 4, 16, 0, None) == 0
    assert one(None, F, 16, P, 16, P, None, P, None, 0, 4, 4, 16, 0, None) == INVALID
    need = lib.f2cgt_quantized_linear_workspace_bytes(1000, 1000, 1000)
    assert need >= 1000 * 1008 + 4000
    assert one(P, F, 1000, P, 1008, P, None, P, None, 0, 1000, 1000, 1000, 0, None) == INVALID
    assert one(P, F, 1000, P, 1008, P, None, P, P, need - 1, 1000, 1000, 1000, 0, None) == INVALID
    assert b"workspace" in lib.f2cgt_last_error()
    assert lib.f2cgt_quantized_linear_workspace_bytes(1, 4096, 4096) == 0                # coded where it is multiplied
    assert lib.f2cgt_quantized_linear_workspace_bytes(0, 4096, 4096) == 0
    # without columns there is nothing to code in the product's workgroups: the weights' buffer may be null
    assert lib.f2cgt_quantized_linear_workspace_bytes(100, 300, 128) == 0
    assert lib.f2cgt_quantized_linear_workspace_bytes(100, 300, 0) == 400


def test_orthogonalised_updates():
    lib = capi.lib()
    good = _coefficients(3.4445, -4.7750, 2.0315)
    call = lib.f2cgt_orthogonalize
    assert call(None, F, None, 0, 5, 5, 5, good, None, 0, None) == 0
    assert call(None, F, None, 1, 0, 5, 5, good, None, 0, None) == 0
    assert call(None, F, None, 1, 5, 5, 5, good, None, 0, None) == INVALID
    assert call(P, capi.DT_F64, P, 1, 5, 5, 5, good, None, 0, None) == UNSUPPORTED
    assert call(P, F, P, 1, 5, 5, 0, good, None, 0, None) == INVALID
    assert call(P, F, P, 1, 5, 5, 101, good, None, 0, None) == INVALID
    assert call(P, F, P, 1, 5, 5, 5, None, None, 0, None) == INVALID
    assert call(P, F, P, -1, 5, 5, 5, good, None, 0, None) == INVALID
    assert call(P, F, P, 1, 65537, 5, 5, good, None, 0, None) == UNSUPPORTED
    # beyond the range of the products: at once, from some step on, and no number at all
    for bad in ((8.0, 0.0, 0.0), (2.0, 0.0, 0.0), (0.0, 0.0, 3.0), (float("nan"), 0.0, 0.0), (1.0, float("inf"), 0.0)):
        assert call(P, F, P, 1, 5, 5, 5, _coefficients(*bad), None, 0, None) == UNSUPPORTED, bad
    need = lib.f2cgt_muon_workspace_bytes(2, 1000, 900)
    assert need > 3 * 2 * 1000 * 900 * 4
    assert call(P, F, P, 2, 1000, 900, 5, good, None, 0, None) == INVALID
    assert call(P, F, P, 2, 1000, 900, 5, good, P, need - 1, None) == INVALID
    assert lib.f2cgt_muon_workspace_bytes(70, 128, 256) == 0                             # a workgroup each
    step = lib.f2cgt_muon_step
    one = (ctypes.c_void_p * 1)(4096)
    none = (ctypes.c_void_p * 1)(None)
    assert step(None, F, None, F, None, 0, 5, 5, 0.1, 0.0, 0.9, 1, 5, good, None, 0, None) == 0
    assert step(one, F, one, F, none, 1, 5, 5, 0.1, 0.0, 0.9, 1, 5, good, None, 0, None) == INVALID
    assert step(one, F, one, F, one, 1, 5, 5, 0.1, 1.0, 0.9, 1, 5, good, None, 0, None) == INVALID     # nothing left of the weight
    assert step(one, F, one, F, one, 1, 5, 5, 0.1, 0.0, 1.0, 1, 5, good, None, 0, None) == INVALID
    assert step(one, capi.DT_I32, one, F, one, 1, 5, 5, 0.1, 0.0, 0.9, 1, 5, good, None, 0, None) == UNSUPPORTED
