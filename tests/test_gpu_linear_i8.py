"""The int8 product on codes and scales, on an MI355X against exact sums and 64-bit arithmetic.

Tolerance: the sum is exact; converting it, the two products with the scales and the bias's addition round four times
in F32 (2^-24 each, of the product or of the result), and the output is rounded once to its type."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _operands(seed, m, n, k, bias=True):
    g = torch.Generator().manual_seed(seed)
    a = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    a_s, w_s = torch.rand(m, generator=g) + 0.01, (torch.rand(n, generator=g) + 0.01) / max(1, k) ** 0.5 / 100
    b = torch.randn(n, generator=g) if bias else None
    return [None if t is None else t.cuda() for t in (a, a_s, w, w_s, b)]


def _sum(a, w):
    """Exact: whole numbers below 2^31 in float64."""
    return a.double() @ w.double().T


def _check(out, a, a_s, w, w_s, b):
    p = _sum(a, w) * a_s.double()[:, None] * w_s.double()
    y = p if b is None else p + b.double()
    info = torch.finfo(out.dtype)
    first = 2.0 ** -24 * (3.01 * p.abs() + 1.01 * y.abs())
    tol = first + (y.abs() + first).clamp_min(info.tiny) * (info.eps / 2)
    bad = (out.double() - y).abs() > tol
    assert not bad.any(), ((out.double() - y).abs() / tol).max().item()


SIZES = [(1, 1, 1), (1, 7, 3), (2, 33, 15), (3, 16, 16), (1, 64, 64), (5, 65, 17), (16, 48, 100), (17, 100, 130),
         (1, 1000, 1537), (4, 257, 4096), (33, 129, 1000), (48, 1024, 512), (64, 96, 2048), (65, 511, 63), (100, 70, 77),
         (129, 200, 384), (256, 256, 128), (257, 513, 640), (300, 1001, 1537), (700, 768, 256), (1111, 320, 96),
         (2050, 1030, 200), (4100, 300, 128)]


@pytest.mark.parametrize("m, n, k", SIZES)
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_linear_i8_is_the_formula_s(context, m, n, k, t):
    a, a_s, w, w_s, b = _operands(m * 31 + n * 7 + k, m, n, k, bias=(m + n + k) % 3 != 0)
    out = torch.full((m, n), 7.0, dtype=TYPES[t], device="cuda")
    context.linear_i8(a, a_s, w, w_s, out, bias=b, stream=_stream())
    _check(out, a, a_s, w, w_s, b)


@pytest.mark.parametrize("m, n", [(1, 33), (20, 40), (300, 300), (2100, 600)])
@pytest.mark.parametrize("k", [131071, 4112])
def test_the_largest_sums_fit(context, m, n, k):
    if m * k > 1 << 26:
        k = 32768 + 16
    a = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    w[1::2] = 127
    one, out = torch.ones(max(m, n), device="cuda"), torch.empty(m, n, device="cuda")
    context.linear_i8(a, one[:m], w, one[:n], out, stream=_stream())
    want = torch.full((n,), 128.0 * 128 * k, dtype=torch.float64)
    want[1::2] = -128.0 * 127 * k
    assert torch.equal(out.cpu(), want.float().expand(m, n))


@pytest.mark.parametrize("m", [1, 19, 130, 600])
@pytest.mark.parametrize("k", [48, 333, 1024])
def test_strided_operands_that_start_anywhere(context, m, k):
    n = 150
    a, a_s, w, w_s, b = _operands(m + k, m, n, k + 40)
    a, w = a[:, 7:7 + k], w[:, 13:13 + k]
    wide = torch.full((m, n + 11), 3.0, dtype=torch.float16, device="cuda")
    out = wide[:, 5:5 + n]
    context.linear_i8(a, a_s, w, w_s, out, bias=b, stream=_stream())
    _check(out, a, a_s, w, w_s, b)
    assert (wide[:, :5] == 3).all() and (wide[:, 5 + n:] == 3).all()
    # One row of codes for all, and one row of weights.
    out = torch.empty(m, n, device="cuda")
    context.linear_i8(a[:1].expand(m, k), a_s, w, w_s, out, stream=_stream())
    _check(out, a[:1].expand(m, k), a_s, w, w_s, None)
    context.linear_i8(a, a_s, w[:1].expand(n, k), w_s, out, stream=_stream())
    _check(out, a, a_s, w[:1].expand(n, k), w_s, None)


@pytest.mark.parametrize("m", [1, 40, 500])
def test_scales_that_are_not_numbers(context, m):
    a, a_s, w, w_s, b = _operands(m, m, 70, 160)
    a_s[m // 2] = float("nan")
    a[m // 2] = 0
    w_s[3] = float("inf")
    w[3] = 1
    a[0, :] = 1
    out = torch.empty(m, 70, device="cuda")
    context.linear_i8(a, a_s, w, w_s, out, bias=b, stream=_stream())
    assert torch.isnan(out[m // 2]).all()
    if m > 1:
        assert out[0, 3] == float("inf") and torch.isfinite(out[0, :3]).all()


def test_an_inner_width_of_none_gives_the_bias(context):
    a, a_s, w, w_s, b = _operands(0, 6, 20, 0)
    out = torch.full((6, 20), 9.0, device="cuda")
    context.linear_i8(a, a_s, w, w_s, out, bias=b, stream=_stream())
    assert torch.equal(out, b.expand(6, 20))
    context.linear_i8(a, a_s, w, w_s, out, stream=_stream())
    assert (out == 0).all()
    for m, n in ((0, 5), (5, 0)):
        a, a_s, w, w_s, _ = _operands(0, m, n, 30)
        context.linear_i8(a, a_s, w, w_s, torch.empty(m, n, device="cuda"), stream=_stream())


@pytest.mark.parametrize("m, n, k", [(1, 4096, 1024), (48, 512, 2048), (200, 300, 500), (1024, 512, 256)])
def test_captured_and_replayed(context, m, n, k):
    a, a_s, w, w_s, b = _operands(5, m, n, k)
    out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        context.linear_i8(a, a_s, w, w_s, out, bias=b, stream=_stream())
    for seed in range(4):
        a.copy_(_operands(seed, m, n, k)[0])
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        _check(out, a, a_s, w, w_s, b)


def test_many_columns_of_one_row(context):
    # Past the workgroups of one pass over the columns.
    n, k = (1 << 22) + 9, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    a = torch.randint(-127, 128, (1, k), generator=g, device="cuda", dtype=torch.int8)
    one, out = torch.ones(n, device="cuda"), torch.empty(1, n, device="cuda")
    context.linear_i8(a, one[:1], w, one, out, stream=_stream())
    assert torch.equal(out[0].double(), (w.double() @ a[0].double()))


@pytest.mark.parametrize("m, n, k", [(5_000_003, 3, 16), (5_000_003, 17, 64), (270_000_001, 1, 16), (3, 9_000_001, 32)])
def test_more_rows_or_columns_than_one_launch_takes(context, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m % 97)
    a = torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    a_s, w_s = torch.rand(m, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda")
    b = torch.randn(n, generator=g, device="cuda")
    out = torch.full((m, n), 7.0, device="cuda")
    context.linear_i8(a, a_s, w, w_s, out, bias=b, stream=_stream())
    for at in range(0, max(m, n), 10_000_000):
        rows = slice(at, at + 10_000_000) if m > n else slice(None)
        _check(out[rows], a[rows], a_s[rows], w, w_s, b)


@pytest.mark.parametrize("m, n", [(4000, 4103), (4001, 4096), (130, 20000), (20001, 70)])
@pytest.mark.parametrize("k", [16, 37, 64, 127, 144])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_many_outputs_of_narrow_rows(context, m, n, k, t):
    """Tiles of one or two stages, the last of them partial: what is not of the rows counts for nothing."""
    a, a_s, w, w_s, b = _operands(m + n + k, m, n, k, bias=k % 2 == 0)
    out = torch.full((m, n), 7.0, dtype=TYPES[t], device="cuda")
    context.linear_i8(a, a_s, w, w_s, out, bias=b, stream=_stream())
    _check(out, a, a_s, w, w_s, b)
