"""Lists of an optimiser's step that share memory are refused by the C entry point (no GPU needed)."""
import ctypes

import pytest

pytest.importorskip("torch")

from f2cgt_amd import capi  # noqa: E402

INVALID = -1
F, B = capi.DT_F32, capi.DT_BF16
SIZE = 200 * 300 * 4            # (needs a workspace)


def _step(weights, grads, momenta, weight_type=F, grad_type=F):
    """The answer to lists at these addresses, and what it says.  The workspace is null: no list gets further than that."""
    lib = capi.lib()
    n = len(weights)
    lists = [(ctypes.c_void_p * n)(*addresses) for addresses in (weights, grads, momenta)]
    rc = lib.f2cgt_muon_step(lists[0], weight_type, lists[1], grad_type, lists[2], n, 200, 300, 0.1, 0.0, 0.9, 1, 5,
                             (ctypes.c_float * 3)(3.4445, -4.7750, 2.0315), None, 0, None)
    return rc, lib.f2cgt_last_error()


def test_shared_memory():
    a, b, c, d, e = (4096 + i * SIZE for i in range(5))
    for apart in (((a,), (b,), (c,)), ((a, b), (c, c), (d, e)), ((c, a), (e, e + 4), (b, d)), ((b,), (a,), (c,))):
        rc, text = _step(*apart)
        assert rc == INVALID and b"workspace" in text, apart
    for shared in (((a,), (a,), (c,)), ((a,), (b,), (b,)), ((a,), (c,), (a,)), ((a,), (a + 4,), (c,)), ((a,), (b - 4,), (c,)), ((b,), (d,), (b - SIZE + 4,)),
                   ((a, a), (b, c), (d, e)), ((a, b), (d, d), (c, c)), ((a, b), (d, d), (e, c + 4)), ((a, b + SIZE // 2), (e, e), (b, d))):
        rc, text = _step(*shared)
        assert rc == INVALID and b"shares memory" in text, shared
    half = SIZE // 2                                        # weights and gradients of two bytes
    rc, text = _step((a, a + half), (b, b + half), (c, d), B, B)
    assert b"workspace" in text
    rc, text = _step((a, a + half - 2), (b, b + half), (c, d), B, B)
    assert b"shares memory" in text
