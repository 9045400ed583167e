"""RMS norm with the residual's addition and int8 codes, and the codes of rows alone, on an MI355X against 64-bit (and
wider) arithmetic on the same inputs.

Tolerances: the norm is computed in 64 bits and rounded to F32 and then to the output's type, so an output is off by
at most half a step of its type, and a 2^-24 of it for the first rounding. Codes and the sum are exact."""
import numpy as np
import pytest

import turboembed_amd as T
from turboembed_amd import seam as S

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _rows(seed, rows, cols, t, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(spread * torch.randn(rows, 1, generator=g))
    return x.to(TYPES[t]).cuda()


def _nearest(c):
    """Codes and largest magnitude of rows c (float64, exact): the whole numbers nearest to 127 c / max|c|, decided in
    64-bit significands, where 127 c and (n + 1/2) max|c| are whole for c of 53 bits or fewer."""
    top = np.abs(c).max(1).astype(np.longdouble)
    a = c.astype(np.longdouble) * 127
    step = np.where(top > 0, top, 1)[:, None]
    n = np.floor(a / step)
    # The quotient's own rounding may have passed a whole number.
    n = np.where(n * step > a, n - 1, n)
    n = np.where((n + 1) * step <= a, n + 1, n)
    d = a - (n + np.longdouble(0.5)) * step
    up = (d > 0) | ((d == 0) & (n % 2 != 0))
    return (n + up).astype(np.int64), top


def _want(x, w, res, eps):
    v = x.float()
    if res is not None:
        v = (v + res.float()).to(res.dtype)
    total = v if res is not None else None
    d = v.double().cpu().numpy()
    c = d if w is None else d * w.double().cpu().numpy()
    r = np.ones(len(d)) if w is None else 1 / np.sqrt((d * d).mean(1) + eps)
    return total, c * r[:, None], c, r


def _close(got, want, t):
    """|got - want| at most half a step of the type (and 2^-24 more); below its smallest normal, of that one's step."""
    info = torch.finfo(TYPES[t])
    g = got.double().cpu().numpy()
    tol = np.maximum(np.abs(want), info.tiny) * (info.eps / 2 + 2.0 ** -24)
    over = np.abs(want) * (1 + 2.0 ** -12) > info.max
    assert np.isfinite(g[~over]).all()
    worst = (np.abs(g - want) / tol)[~over]
    assert worst.size == 0 or worst.max() <= 1, worst.max()


def _check_codes(codes, scales, c, r):
    q, top = _nearest(c)
    assert np.array_equal(codes.cpu().numpy(), q)
    want = (top * r / 127).astype(np.float64)
    got = scales.double().cpu().numpy()
    assert np.all(np.abs(got - want) <= np.maximum(want, 2.0 ** -126) * 2.0 ** -24 * (1 + 1e-6))


def _norm(context, x, w, eps=1e-6, res=None, sum=False, out=None, codes=True, **kw):
    rows, cols = x.shape
    s = torch.empty_like(res) if sum else None
    o = torch.empty(rows, cols, dtype=TYPES[out], device="cuda") if out else None
    q = torch.full((rows, cols), 77, dtype=torch.int8, device="cuda") if codes else None
    k = torch.empty(rows, device="cuda") if codes else None
    context.rms_norm(x, w, eps, residual=res, sum=s, out=o, codes=q, scales=k, stream=_stream(), **kw)
    return s, o, q, k


SIZES = [(1, 1), (1, 8), (3, 7), (9, 64), (5, 513), (7, 1023), (2, 1024), (6, 2047), (4, 2056), (3, 4096), (3, 4099),
         (2, 8193), (2, 16384), (2, 20001), (1, 65536)]


@pytest.mark.parametrize("rows, cols", SIZES)
@pytest.mark.parametrize("x, res, w, out", [
    ("f32", None, "f32", "f32"), ("f32", "f32", "f32", "f16"), ("f16", None, "f16", "f16"),
    ("f16", "f16", "f32", "bf16"), ("f16", "f32", "f16", "f32"), ("bf16", "bf16", "bf16", "bf16"),
    ("bf16", "f32", "f32", "f16"), ("bf16", None, "f32", "f32")])
def test_rms_norm_is_the_formula_s(context, rows, cols, x, res, w, out):
    a = _rows(rows * 7919 + cols, rows, cols, x)
    r = None if res is None else _rows(cols, rows, cols, res)
    weight = (1 + 0.3 * _rows(3, 1, cols, "f32", 0)[0]).to(TYPES[w])
    s, o, q, k = _norm(context, a, weight, res=r, sum=res is not None, out=out)
    total, y, c, rr = _want(a, weight, r, 1e-6)
    if res is not None:
        assert torch.equal(s, total)
    _close(o, y, out)
    _check_codes(q, k, c, rr)


@pytest.mark.parametrize("rows, cols", SIZES)
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_quantize_tokens_is_the_formula_s(context, rows, cols, t):
    x = _rows(rows + cols, rows, cols, t)
    q, k = torch.empty(rows, cols, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    context.quantize_tokens(x, q, k, stream=_stream())
    c = x.double().cpu().numpy()
    _check_codes(q, k, c, np.ones(rows))


def test_many_rows(context):
    # Past the workgroups of one pass over the rows.
    rows = 4 * (1 << 20) + 5
    x = _rows(0, 64, 8, "f16").repeat((rows + 63) // 64, 1)[:rows].contiguous()
    q, k = torch.empty(rows, 8, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    context.quantize_tokens(x, q, k, stream=_stream())
    want, top = _nearest(x[:64].double().cpu().numpy())
    assert torch.equal(q[:64].cpu(), torch.from_numpy(want).to(torch.int8))
    assert torch.equal(q, q[:64].repeat((rows + 63) // 64, 1)[:rows])
    assert torch.equal(k, k[:64].repeat((rows + 63) // 64)[:rows])


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_codes_on_the_border_of_two_go_to_the_even_one(context, t):
    # max|c| = 127 s: 127 c / max|c| = c / s, halves exactly and next to them.
    half = torch.arange(-126, 127, dtype=torch.float32) + 0.5
    rows = []
    for s in (1.0, 2.0 ** -20, 2.0 ** 30):
        c = half if t == "bf16" else torch.stack([half, torch.nextafter(half, torch.full_like(half, 1e9)),
                                                  torch.nextafter(half, torch.full_like(half, -1e9))]).flatten()
        c = torch.cat([c, torch.tensor([127.0])]) * s
        rows.append(c)
    x = torch.stack(rows).to(TYPES[t]).cuda()
    n = x.shape[1]
    q, k = torch.empty(3, n, dtype=torch.int8, device="cuda"), torch.empty(3, device="cuda")
    context.quantize_tokens(x, q, k, stream=_stream())
    _check_codes(q, k, x.double().cpu().numpy(), np.ones(3))
    ones = torch.ones(n, device="cuda")
    _, _, q2, _ = _norm(context, x, ones)
    assert torch.equal(q, q2)
    # A norm's codes do not hang on its factor: also with a weight that turns the halves around.
    _, _, q3, _ = _norm(context, x, -ones * 1.5)
    assert torch.equal(q3, -q)


def test_rows_of_zeros_infinities_and_nans(context):
    x = _rows(1, 6, 300, "f16")
    x[1] = 0
    x[2, 299] = float("inf")
    x[3, 0] = float("nan")
    x[4, 17] = -float("inf")
    w = torch.ones(300, device="cuda")
    for call in ("norm", "tokens"):
        if call == "norm":
            _, o, q, k = _norm(context, x, w, out="f32")
        else:
            q, k = torch.empty(6, 300, dtype=torch.int8, device="cuda"), torch.empty(6, device="cuda")
            context.quantize_tokens(x, q, k, stream=_stream())
        assert k[1] == 0 and not q[1].any()
        for bad in (2, 3, 4):
            assert torch.isnan(k[bad]) and not q[bad].any()
        for fine in (0, 5):
            assert torch.isfinite(k[fine]) and q[fine].abs().max() == 127
    want = x.double() / torch.sqrt((x.double() ** 2).mean(1, keepdim=True) + 1e-6)
    assert torch.equal(torch.isnan(o), torch.isnan(want)) and (o[1] == 0).all()
    # A weight that is not a number is seen in the codes too.
    w[5] = float("nan")
    _, o, q, k = _norm(context, x[:1], w, out="f32")
    assert torch.isnan(k).all() and torch.isnan(o).sum() == 1


@pytest.mark.parametrize("size", [1e30, 1e-30])
def test_rows_whose_squares_pass_32_bits(context, size):
    x = _rows(2, 3, 700, "f32") * size
    w = 1 + 0.1 * _rows(5, 1, 700, "f32", 0)[0]
    _, o, q, k = _norm(context, x, w, eps=1e-90, out="f32")
    _, y, c, r = _want(x, w, None, 1e-90)
    _close(o, y, "f32")
    _check_codes(q, k, c, r)


def test_strided_rows_and_rows_that_start_anywhere(context):
    base = _rows(3, 11, 1000, "bf16")
    for cols, off in ((600, 0), (601, 3), (37, 1)):
        x = base[:, off:off + cols]
        w = _rows(4, 1, 700, "f32", 0)[0][1:1 + cols]
        wide = torch.full((11, cols + 9), 5.0, dtype=torch.bfloat16, device="cuda")
        codes = torch.full((11, cols + 5), 9, dtype=torch.int8, device="cuda")
        scales = torch.zeros(11, device="cuda")
        context.rms_norm(x, w, 1e-5, out=wide[:, 4:4 + cols], codes=codes[:, 1:1 + cols], scales=scales,
                         stream=_stream())
        _, y, c, r = _want(x, w, None, 1e-5)
        _close(wide[:, 4:4 + cols], y, "bf16")
        _check_codes(codes[:, 1:1 + cols], scales, c, r)
        # Nothing beside the rows is written.
        assert (wide[:, :4] == 5).all() and (wide[:, 4 + cols:] == 5).all()
        assert (codes[:, :1] == 9).all() and (codes[:, 1 + cols:] == 9).all()
    # One row for all.
    x = base[:1, :64].expand(5, 64)
    q, k = torch.empty(5, 64, dtype=torch.int8, device="cuda"), torch.empty(5, device="cuda")
    context.quantize_tokens(x, q, k, stream=_stream())
    assert torch.equal(q, q[:1].expand(5, 64)) and q[0].abs().max() == 127


def test_in_place(context):
    x, res = _rows(6, 9, 777, "f16"), _rows(7, 9, 777, "f16")
    w = torch.ones(777, device="cuda")
    want = _norm(context, x, w, res=res, sum=True, out="f16")
    a, b = x.clone(), res.clone()
    context.rms_norm(a, w, 1e-6, residual=b, sum=b, out=a, stream=_stream())
    assert torch.equal(b, want[0]) and torch.equal(a, want[1])
    a, b = x.clone(), res.clone()
    context.rms_norm(a, w, 1e-6, residual=b, sum=a, out=b.new_empty(9, 777), stream=_stream())
    assert torch.equal(a, want[0]) and torch.equal(b, res)


def test_empty_rows_and_columns(context):
    for shape in ((0, 40), (5, 0)):
        x = torch.empty(shape, device="cuda")
        k = torch.full((shape[0],), 3.0, device="cuda")
        q = torch.empty(shape, dtype=torch.int8, device="cuda")
        context.quantize_tokens(x, q, k, stream=_stream())
        # (A row of no columns is a row of zeros.)
        assert (k == 0).all()
        context.rms_norm(x, torch.ones(shape[1], device="cuda"), 1e-6, out=torch.empty_like(x), stream=_stream())


def test_on_the_context_s_stream_and_over_its_buffers(context):
    x = _rows(8, 5, 100, "f32").cpu().numpy()
    buf = context.buffer(5 * 100 * 4, S.TURBO_PLACE_SHARED)
    buf.view(np.float32)[:] = x.ravel()
    w = context.buffer(400, S.TURBO_PLACE_SHARED)
    w.view(np.float32)[:] = 1
    out = context.buffer(16 + 5 * 100 + 5 * 4, S.TURBO_PLACE_DEVICE)
    codes = T.DeviceArray(out, (5, 100), S.TURBO_DTYPE_I8)
    scales = T.DeviceArray(out, (5,), S.TURBO_DTYPE_F32, offset=500)
    context.rms_norm(T.DeviceArray(buf, (5, 100), S.TURBO_DTYPE_F32), T.DeviceArray(w, (100,), S.TURBO_DTYPE_F32),
                     1e-6, codes=codes, scales=scales)
    got = out.read()
    _, y, c, r = _want(torch.from_numpy(x), torch.ones(100), None, 1e-6)
    _check_codes(torch.from_numpy(got[:500].view(np.int8).reshape(5, 100)), torch.from_numpy(got[500:520].view(np.float32)),
                 c, r)
    with pytest.raises(T.TurboError):
        context.quantize_tokens(T.DeviceArray(buf, (6, 100), S.TURBO_DTYPE_F32), codes, scales)
    host = context.buffer(64, S.TURBO_PLACE_HOST)
    with pytest.raises(T.TurboError):
        T.DeviceArray(host, (4, 4), S.TURBO_DTYPE_F32)
    for b in (buf, w, out, host):
        b.close()


def test_captured_and_replayed(context):
    x, res = _rows(9, 33, 1536, "bf16"), _rows(10, 33, 1536, "bf16")
    w = 1 + 0.1 * _rows(11, 1, 1536, "f32", 0)[0]
    s, q, k = torch.empty_like(res), torch.empty(33, 1536, dtype=torch.int8, device="cuda"), torch.empty(33, device="cuda")

    def call():
        context.rms_norm(x, w, 1e-6, residual=res, sum=s, codes=q, scales=k, stream=_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for seed in range(4):
        x.copy_(_rows(20 + seed, 33, 1536, "bf16"))
        call()
        torch.cuda.synchronize()
        want = s.clone(), q.clone(), k.clone()
        for t in (s, q, k):
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, (s, q, k)))


# Rows that share a wave: up to 64, 128 and 256 columns, and one past each; rows that fill no workgroup, and that
# leave a part of the last one.
NARROW = [(1, 3), (31, 1), (33, 8), (1000, 53), (257, 64), (70, 65), (333, 100), (17, 128), (16, 129), (99, 200),
          (9, 256), (41, 257)]


@pytest.mark.parametrize("rows, cols", NARROW)
@pytest.mark.parametrize("x, res, out", [("f32", "f32", "f32"), ("f16", None, "bf16"), ("bf16", "f32", "f16")])
def test_norms_of_narrow_rows(context, rows, cols, x, res, out):
    a = _rows(rows * 7919 + cols, rows, cols, x)
    r = None if res is None else _rows(cols, rows, cols, res)
    weight = 1 + 0.3 * _rows(3, 1, cols, "f32", 0)[0]
    s, o, q, k = _norm(context, a, weight, res=r, sum=res is not None, out=out)
    total, y, c, rr = _want(a, weight, r, 1e-6)
    if res is not None:
        assert torch.equal(s, total)
    _close(o, y, out)
    _check_codes(q, k, c, rr)
    # In place, in rows of a wider array.
    wide = torch.zeros(rows, cols + 9, dtype=a.dtype, device="cuda")
    wide[:, 4:4 + cols] = a
    own = wide[:, 4:4 + cols]
    context.rms_norm(own, weight, 1e-6, out=own, stream=_stream())
    _close(own, _want(a, weight, None, 1e-6)[1], x)
    assert (wide[:, :4] == 0).all() and (wide[:, 4 + cols:] == 0).all()


@pytest.mark.parametrize("cols", [1, 53, 64, 100, 250])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_narrow_rows_beside_rows_of_no_numbers(context, cols, t):
    x = _rows(cols, 100, cols, t)
    x[3::7], x[5::11, cols // 2], x[6::13, 0] = 0, float("inf"), float("nan")
    q, k = torch.full((100, cols), 77, dtype=torch.int8, device="cuda"), torch.empty(100, device="cuda")
    context.quantize_tokens(x, q, k, stream=_stream())
    fine = torch.isfinite(x).all(1)
    assert torch.equal(torch.isnan(k), ~fine) and (q[~fine] == 0).all()
    _check_codes(q[fine], k[fine], x[fine].double().cpu().numpy(), np.ones(int(fine.sum())))


def test_more_rows_than_a_launch_s_workgroups_take_at_once(context):
    rows = 4 * (1 << 20) + 5
    x = _rows(0, 64, 260, "f16").repeat((rows + 63) // 64, 1)[:rows].contiguous()
    q, k = torch.empty(rows, 260, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    context.quantize_tokens(x, q, k, stream=_stream())
    want, top = _nearest(x[:64].double().cpu().numpy())
    assert torch.equal(q[:64].cpu(), torch.from_numpy(want).to(torch.int8))
    assert torch.equal(q, q[:64].repeat((rows + 63) // 64, 1)[:rows])
    assert torch.equal(k, k[:64].repeat((rows + 63) // 64)[:rows])


@pytest.mark.parametrize("cols", [2050, 4096, 9000])
def test_wide_rows_that_share_a_workgroup(context, cols):
    # (61 rows over and over: a workgroup's rows, 2^14 apart, are others.)
    rows, part = (1 << 14) * 2 + 77, 61
    x, r = _rows(1, part, cols, "bf16"), _rows(2, part, cols, "bf16")
    weight = 1 + 0.3 * _rows(3, 1, cols, "f32", 0)[0]
    total, y, c, rr = _want(x, weight, r, 1e-6)
    many = lambda t: t.repeat(rows // part + 1, *[1] * (t.dim() - 1))[:rows]  # noqa: E731
    s, o, q, k = _norm(context, many(x), weight, res=many(r), sum=True, out="f16")
    _close(o[:part], y, "f16")
    _check_codes(q[:part], k[:part], c, rr)
    for got, want in ((s, total), (o, o[:part].clone()), (q, q[:part].clone()), (k, k[:part].clone())):
        assert torch.equal(got, many(want))


@pytest.mark.parametrize("cols", [40, 1024])
@pytest.mark.parametrize("x, out", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "bf16")])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -16])
def test_an_output_is_rounded_once(context, cols, x, out, size):
    """At most half a step from the 64-bit result, its own roundings (some n 2^-53) aside: a rounding to F32 on the
    way, which is up to 2^-25 more next to the middle of two steps, would show. The smaller size gives F16 outputs
    below the smallest normal number."""
    rows = (1 << 21) // cols
    a = _rows(cols, rows, cols, x)
    weight = (1 + 0.3 * _rows(4, 1, cols, "f32", 0)[0]) * size
    y = _norm(context, a, weight, out=out, codes=False)[1].double().cpu().numpy()
    want = _want(a, weight, None, 1e-6)[1]
    info = torch.finfo(TYPES[out])
    step = np.ldexp(info.eps, np.frexp(np.maximum(np.abs(want), info.tiny))[1] - 1)
    assert (np.abs(y - want) <= step / 2 + np.abs(want) * 2.0 ** -40).all()
