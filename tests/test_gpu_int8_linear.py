"""Rows coded in 8 bits and the products of coded rows: against whole numbers and float64, and what is refused."""
import pytest

torch = pytest.importorskip("torch")

if torch.cuda.is_available():
    import f2cgt_amd
    from f2cgt_amd import pipeline

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}     # half a unit in the last place
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _codes(rows, k, g, stride=None):
    room = torch.randint(-127, 128, (rows, stride or (k + 15) // 16 * 16 + 16), generator=g, device="cuda", dtype=torch.int8)
    return room[:, :k]                      # what lies behind a row's end is not zero


def _want(codes, scales, weight, weight_scales, bias, relu):
    """(float64 result, the size that roundings go by)"""
    sums = (codes.cpu().double() @ weight.cpu().double().t()).cuda()
    product = sums * (scales.double()[:, None] * weight_scales.double())
    z = product if bias is None else product + bias.double()
    return (z.clamp(min=0) if relu else z), product.abs()


def _check(out, want, size, dtype):
    # the sum, the scales' product and theirs are rounded, then the bias' addition, then the result's type
    bound = 4 * 2.0 ** -24 * size + 2.0 ** -24 * (want.abs() + size) + HALF[dtype] * (want.abs() + 1e-6 * size) + LEAST[dtype]
    assert bool(((out.double() - want).abs() <= bound).all()), float(((out.double() - want).abs() - bound).max())


SHAPES = [(1, 1, 1), (1, 16, 1), (1, 128, 64), (1, 4096, 47), (2, 100, 33), (3, 4097, 130), (4, 8191, 16), (5, 257, 31), (16, 512, 256),
          (17, 640, 257), (31, 602, 128), (33, 15, 65), (47, 129, 100), (64, 64, 64), (65, 127, 129), (100, 1000, 1000), (128, 256, 512),
          (200, 333, 77), (256, 1024, 255), (513, 96, 300), (1000, 130, 1030), (1024, 128, 256), (3001, 100, 47), (5000, 602, 128)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_products_against_whole_numbers(m, k, n, dtype):
    lib = f2cgt_amd.load()
    g = _gen(m + 3 * k + 7 * n)
    codes, weight = _codes(m, k, g), _codes(n, k, g)
    scales = torch.rand((m,), generator=g, device="cuda") * 1e-2 + 1e-4
    weight_scales = torch.rand((n,), generator=g, device="cuda") * 1e-3 + 1e-5
    for bias, relu in ((torch.randn((n,), generator=g, device="cuda"), True), (None, False)):
        out = lib.int8_linear(codes, scales, weight, weight_scales, bias, relu, dtype)
        assert out.shape == (m, n) and out.dtype == dtype and out.is_contiguous()
        _check(out, *_want(codes, scales, weight, weight_scales, bias, relu), dtype)


@pytest.mark.parametrize("m,k,n", [(2048, 512, 2048), (4096, 1024, 768), (2500, 700, 1111), (8192, 128, 256), (777, 5000, 4000),
                                   (4096, 1030, 4096), (4095, 1100, 4093), (8300, 1024, 4100)])
def test_large_products_are_the_whole_numbers(m, k, n):
    # unit scales: every sum below 2^24 is given as it is
    lib = f2cgt_amd.load()
    g = _gen(m + k + n)
    codes = torch.randint(-40, 41, (m, (k + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.int8)[:, :k]
    weight = torch.randint(-40, 41, (n, (k + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.int8)[:, :k]
    out = lib.int8_linear(codes, torch.ones(m, device="cuda"), weight, torch.ones(n, device="cuda"))
    assert torch.equal(out.double(), codes.double() @ weight.double().t())


@pytest.mark.parametrize("m", [1, 3, 20, 70, 300])
def test_extreme_codes_and_longest_rows(m):
    lib = f2cgt_amd.load()
    k, n = 131071, 40
    codes = torch.full((m, 131072), -128, dtype=torch.int8, device="cuda")[:, :k]
    weight = torch.full((n, 131072), -128, dtype=torch.int8, device="cuda")[:, :k]
    weight[1] = 127
    out = lib.int8_linear(codes, torch.ones(m, device="cuda"), weight, torch.ones(n, device="cuda"))
    assert bool((out[:, 0] == float(128 * 128 * k)).all()) and bool((out[:, 1] == float(-128 * 127 * k)).all())


def test_layouts_of_codes():
    lib = f2cgt_amd.load()
    g = _gen(5)
    scales, weight_scales = torch.rand((37,), generator=g, device="cuda"), torch.rand((29,), generator=g, device="cuda")
    codes, weight = _codes(37, 50, g), _codes(29, 50, g)
    want = lib.int8_linear(codes, scales, weight, weight_scales)
    packed = codes.clone(memory_format=torch.contiguous_format)
    assert packed.stride(0) == 50
    columns = codes.t().contiguous().t()                                # columns after one another
    shifted = torch.zeros(37 * 64 + 3, dtype=torch.int8, device="cuda")[3:].view(37, 64)[:, :50]
    shifted.copy_(codes)
    twice = torch.zeros((74, 64), dtype=torch.int8, device="cuda")
    twice[::2, :50] = codes
    for other in (packed, columns, shifted, twice[::2, :50]):
        assert torch.equal(lib.int8_linear(other, scales, weight, weight_scales), want)
    assert torch.equal(lib.int8_linear(codes, scales, weight.clone(memory_format=torch.contiguous_format), weight_scales), want)
    ends = torch.zeros(36 * 64 + 50, dtype=torch.int8, device="cuda").as_strided((37, 50), (64, 1))      # nothing behind its last row
    apart = torch.zeros(36 * (1 << 23) + 64, dtype=torch.int8, device="cuda").as_strided((37, 50), (1 << 23, 1))
    for other in (ends, apart):
        other.copy_(codes)
        assert torch.equal(lib.int8_linear(other, scales, weight, weight_scales), want)
    same = codes[:1].expand(37, 50)                                     # one row again and again
    assert torch.equal(lib.int8_linear(same, scales, weight, weight_scales),
                       lib.int8_linear(same.contiguous(), scales, weight, weight_scales))
    assert torch.equal(lib.int8_linear(codes, scales.repeat_interleave(2)[::2], weight, weight_scales), want)


def test_empty_sizes():
    lib = f2cgt_amd.load()
    e8 = lambda *s: torch.empty(s, dtype=torch.int8, device="cuda")   # noqa: E731
    e = lambda *s: torch.empty(s, device="cuda")                      # noqa: E731
    assert lib.int8_linear(e8(0, 32), e(0), e8(5, 32), e(5)).shape == (0, 5)
    assert lib.int8_linear(e8(4, 32), e(4), e8(0, 32), e(0)).shape == (4, 0)
    bias = torch.tensor([1.0, -2.0], device="cuda")
    out = lib.int8_linear(e8(3, 0), torch.ones(3, device="cuda"), e8(2, 0), torch.ones(2, device="cuda"), bias, True)
    assert torch.equal(out, torch.tensor([[1.0, 0.0]] * 3, device="cuda"))
    codes, scales = lib.quantize_rows(e(0, 7))
    assert codes.shape == (0, 7) and scales.shape == (0,)
    assert lib.quantized_linear(e(0, 32), e8(5, 32), e(5)).shape == (0, 5)
    assert torch.equal(lib.quantized_linear(e(3, 0), e8(2, 0), torch.ones(2, device="cuda"), bias), bias.expand(3, 2))


def _rows(x):
    """Codes and scales by the definition, in numpy's single precision."""
    import numpy as np
    v = x.float().cpu().numpy()
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        most = np.abs(v).max(axis=1) if v.shape[1] else np.zeros(v.shape[0], np.float32)
        scales = np.maximum(most, np.float32(1e-30)) * np.float32(1 / 127)
        codes = np.clip(np.nan_to_num(np.rint(v * (np.float32(1) / scales)[:, None]), nan=0.0), -127, 127).astype(np.int8)
    return torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()


@pytest.mark.parametrize("m,k", [(1, 1), (1, 4096), (2, 63), (3, 64), (5, 65), (7, 100), (4, 1023), (33, 602), (130, 128), (9, 4099), (2, 20001),
                                 (1025, 256), (3, 8192), (5, 16385)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_rows_are_coded_as_defined(m, k, dtype):
    lib = f2cgt_amd.load()
    x = (torch.randn((m, k), generator=_gen(m + k), device="cuda") * 3).to(dtype)
    if m > 2:
        x[1] = 0
        x[2] *= 1e-4
    codes, scales = lib.quantize_rows(x)
    want, want_scales = _rows(x)
    assert codes.dtype == torch.int8 and scales.dtype == torch.float32 and codes.stride(0) % 16 == 0
    assert torch.equal(codes, want) and torch.equal(scales, want_scales)


def test_rows_of_other_layouts_and_special_values():
    lib = f2cgt_amd.load()
    base = torch.randn((40, 300), generator=_gen(3), device="cuda")
    for x in (base[:, 7:107], base[::3, 1:], base.t(), base[0].expand(6, 300), base[3:4, 5:6], base[:, 0:1]):
        codes, scales = lib.quantize_rows(x)
        want, want_scales = _rows(x)
        assert torch.equal(codes, want) and torch.equal(scales, want_scales)
    x = base[:9].clone()
    x[0, 5], x[1, 7], x[2, 9] = float("nan"), float("inf"), float("-inf")
    x[3] = 0
    x[4] *= 1e-38                       # (below the least scale: codes of zero)
    x[5] *= 1e37
    x[6, :] = torch.finfo(torch.float32).max
    x[7, 0] = torch.finfo(torch.float32).min
    codes, scales = lib.quantize_rows(x)
    want, want_scales = _rows(x)
    assert torch.equal(codes, want) and torch.equal(scales.isnan(), want_scales.isnan())
    assert torch.equal(scales[1:], want_scales[1:])
    weight, weight_scales = lib.quantize_rows(torch.randn((20, 300), generator=_gen(4), device="cuda"))
    for rows in (slice(0, 9), slice(0, 1), slice(1, 3)):
        out = lib.quantized_linear(x[rows], weight, weight_scales, None, True)
        held = x[rows].isfinite().all(1)
        assert bool(out[~held].isnan().all()) and not bool(out[held].isnan().any())    # (the largest may be infinite)
    zero = lib.quantized_linear(x[3:4], weight, weight_scales, None, False)
    assert bool((zero == 0).all())


@pytest.mark.parametrize("m,k,n", [(1, 4096, 300), (1, 100, 47), (2, 5000, 65), (3, 602, 128), (4, 4096, 4096), (7, 64, 1000), (16, 1000, 333), (33, 2048, 700),
                                   (64, 513, 90), (150, 256, 512), (1024, 128, 256), (4001, 100, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_one_call_gives_what_two_give(m, k, n, dtype):
    lib = f2cgt_amd.load()
    g = _gen(m * 3 + k + n)
    x = torch.randn((m, k), generator=g, device="cuda").to(dtype)
    weight, weight_scales = lib.quantize_rows(torch.randn((n, k), generator=g, device="cuda") / k ** 0.5)
    bias = torch.randn((n,), generator=g, device="cuda")
    codes, scales = lib.quantize_rows(x)
    for b, relu in ((bias, True), (None, False)):
        got = lib.quantized_linear(x, weight, weight_scales, b, relu)
        assert got.dtype == dtype
        assert torch.equal(got, lib.int8_linear(codes, scales, weight, weight_scales, b, relu, dtype))
    _check(got, *_want(codes, scales, weight, weight_scales, None, False), dtype)


def test_leading_dimensions_strides_and_streams():
    lib = f2cgt_amd.load()
    g = _gen(9)
    weight, weight_scales = lib.quantize_rows(torch.randn((70, 90), generator=g, device="cuda"))
    x = torch.randn((3, 5, 90), generator=g, device="cuda")
    want = torch.stack([lib.quantized_linear(v, weight, weight_scales) for v in x])
    assert torch.equal(lib.quantized_linear(x, weight, weight_scales), want)
    assert torch.equal(lib.quantized_linear(x[0, 0], weight, weight_scales), want[0, 0])
    wide = torch.randn((5, 200), generator=g, device="cuda")
    wide[:, 40:130] = x[1]
    assert torch.equal(lib.quantized_linear(wide[:, 40:130], weight, weight_scales), want[1])
    assert torch.equal(lib.quantized_linear(x[2].t().contiguous().t(), weight, weight_scales), want[2])
    codes, scales = lib.quantize_rows(x)
    assert codes.shape == (3, 5, 90) and scales.shape == (3, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = lib.quantized_linear(x, weight, weight_scales)
    side.synchronize()
    assert torch.equal(other, want)


def test_replayed_in_a_graph():
    lib = f2cgt_amd.load()
    g = _gen(11)
    weight, weight_scales = lib.quantize_rows(torch.randn((130, 100), generator=g, device="cuda"))
    x = torch.randn((40, 100), generator=g, device="cuda")
    lib.quantized_linear(x, weight, weight_scales)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lib.quantized_linear(x, weight, weight_scales)
    for i in range(4):
        x.copy_(torch.randn((40, 100), generator=g, device="cuda"))
        want = lib.quantized_linear(x, weight, weight_scales)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_what_is_refused():
    lib = f2cgt_amd.load()
    g = _gen(1)
    codes, weight = _codes(4, 32, g), _codes(6, 32, g)
    s, ws = torch.ones(4, device="cuda"), torch.ones(6, device="cuda")
    x = torch.randn((4, 32), generator=g, device="cuda")
    for call in (lambda: lib.int8_linear(codes.cpu(), s, weight, ws), lambda: lib.int8_linear(codes.float(), s, weight, ws),
                 lambda: lib.int8_linear(codes[:, :31], s, weight, ws), lambda: lib.int8_linear(codes, s[:3], weight, ws),
                 lambda: lib.int8_linear(codes, s.double(), weight, ws), lambda: lib.int8_linear(codes, s, weight, ws[:5]),
                 lambda: lib.int8_linear(codes, s, weight, ws, torch.ones(5, device="cuda")),
                 lambda: lib.int8_linear(codes, s, weight, ws, None, False, torch.float64),
                 lambda: lib.int8_linear(codes, s.cpu(), weight, ws), lambda: lib.int8_linear(codes[0], s, weight, ws),
                 lambda: lib.quantize_rows(x.double()), lambda: lib.quantize_rows(x.cpu()), lambda: lib.quantize_rows(x.clone().requires_grad_()),
                 lambda: lib.quantized_linear(x[:, :31], weight, ws), lambda: lib.quantized_linear(x.int(), weight, ws),
                 lambda: lib.quantized_linear(x.clone().requires_grad_(), weight, ws),
                 lambda: lib.int8_linear(torch.zeros((1, 1 << 17), dtype=torch.int8, device="cuda"), s[:1],
                                         torch.zeros((1, 1 << 17), dtype=torch.int8, device="cuda"), ws[:1])):
        with pytest.raises(RuntimeError):
            call()
    with torch.no_grad():
        lib.quantized_linear(x.clone().requires_grad_(), weight, ws)


def test_layer_of_eight_bits():
    torch.manual_seed(0)
    for bias in (True, False):
        linear = torch.nn.Linear(100, 33, bias=bias).cuda()
        served = pipeline.Int8Linear(linear)
        x = torch.randn((50, 100), device="cuda")
        with torch.no_grad():
            got, full = served(x), linear(x)
        # half a step of a code in either factor: |x|_1 wstep / 2 + |w|_1 xstep / 2 + k / 4 of both
        xs, ws = x.abs().amax(1, keepdim=True) / 127, linear.weight.abs().amax(1) / 127
        bound = 0.5 * x.abs().sum(1, keepdim=True) * ws + 0.5 * xs * linear.weight.abs().sum(1) + 25 * xs * ws
        assert bool(((got - full).abs() <= 1.001 * bound + 1e-5).all())
        again = pipeline.Int8Linear(torch.nn.Linear(100, 33, bias=bias).cuda())
        again.load_state_dict(served.state_dict())
        assert torch.equal(again(x), got)
        half = served.half()
        assert half.weight_scales.dtype == torch.float32 and torch.equal(half(x), got)
        assert half(x.bfloat16()).dtype == torch.bfloat16


def test_leading_dimensions_without_columns():
    lib = f2cgt_amd.load()
    w = torch.empty((5, 0), dtype=torch.int8, device="cuda")
    ws, bias = torch.ones(5, device="cuda"), torch.arange(5.0, device="cuda")
    x = torch.empty((2, 3, 0), device="cuda")
    assert torch.equal(lib.quantized_linear(x, w, ws, bias), bias.expand(2, 3, 5))
    codes, scales = lib.quantize_rows(x)
    assert codes.shape == (2, 3, 0) and scales.shape == (2, 3)
    assert lib.quantized_linear(torch.empty((2, 0, 0), device="cuda"), w, ws, bias).shape == (2, 0, 5)


@pytest.mark.parametrize("rows", [1, 16, 17, 48, 70, 128, 700])
def test_no_columns(rows):
    lib = f2cgt_amd.load()
    w = torch.empty((300, 0), dtype=torch.int8, device="cuda")
    ws, bias = torch.ones(300, device="cuda"), torch.arange(-5.0, 295.0, device="cuda")
    want = bias.clamp(min=0).expand(rows, 300)
    x = torch.empty((rows, 0), device="cuda")
    assert torch.equal(lib.quantized_linear(x, w, ws, bias, relu=True), want)
    assert torch.equal(lib.int8_linear(torch.empty((rows, 0), dtype=torch.int8, device="cuda"), torch.ones(rows, device="cuda"), w,
                                       ws, bias, True), want)


@pytest.mark.parametrize("m,k,n", [(20_000_000, 96, 112), (270_000, 320, 8192)])
def test_results_of_more_than_2_31_values(m, k, n):
    """The last rows, far beyond 32-bit offsets, are what a call of those rows alone gives."""
    lib = f2cgt_amd.load()
    g = torch.Generator(device="cuda").manual_seed(5)
    weight, weight_scales = lib.quantize_rows(torch.randn((n, k), generator=g, device="cuda"))
    x = torch.zeros((m, k), dtype=torch.bfloat16, device="cuda")
    x[-333:] = torch.randn((333, k), generator=g, device="cuda").bfloat16()
    out = lib.quantized_linear(x, weight, weight_scales)
    assert out.numel() > 2 ** 31
    assert torch.equal(out[-333:], lib.quantized_linear(x[-333:].clone(), weight, weight_scales))
    assert not out[:1000].any() and not out[m // 2:m // 2 + 1000].any()


def test_rows_of_more_than_2_31_values():
    lib = f2cgt_amd.load()
    g = torch.Generator(device="cuda").manual_seed(6)
    m, k = 1_100_000, 2000
    x = torch.ones((m, k), dtype=torch.float16, device="cuda")
    x[-50:] = torch.randn((50, k), generator=g, device="cuda").half()
    codes, scales = lib.quantize_rows(x)
    tail, tail_scales = lib.quantize_rows(x[-50:].clone())
    assert torch.equal(codes[-50:], tail) and torch.equal(scales[-50:], tail_scales)
    assert bool((codes[:-50] == 127).all())
