"""The operators on device memory without a device: what their calls refuse, with which status and which array, and
that a call with nothing wrong gets as far as the missing context."""
import ctypes as C

import pytest

import turboembed_amd as T
from turboembed_amd import operators as O
from turboembed_amd import seam as S

F32, F16, BF16, I8, I32 = (S.TURBO_DTYPE_F32, S.TURBO_DTYPE_F16, S.TURBO_DTYPE_BF16, S.TURBO_DTYPE_I8, S.TURBO_DTYPE_I32)


class Fake:
    """An array that is nowhere: only its description is looked at."""
    is_cuda = True

    def __init__(self, at, shape, dtype, strides=None):
        self.at, self.shape, self.dtype = at, tuple(shape), dtype
        s, n = [], 1
        for k in reversed(self.shape):
            s.insert(0, n)
            n *= k
        self.strides = tuple(strides or s)

    def data_ptr(self):
        return self.at

    def stride(self):
        return self.strides


GB = 1 << 30


def _norm(**kw):
    a = dict(x=Fake(1 * GB, (4, 24), F16), weight=Fake(2 * GB, (24,), F32), eps=1e-6, out=Fake(3 * GB, (4, 24), F16))
    a.update(kw)
    O.rms_norm(None, **a)


def _tokens(**kw):
    a = dict(x=Fake(1 * GB, (4, 24), F16), codes=Fake(2 * GB, (4, 24), I8), scales=Fake(3 * GB, (4,), F32))
    a.update(kw)
    O.quantize_tokens(None, **a)


def _linear(**kw):
    a = dict(codes=Fake(1 * GB, (4, 24), I8), scales=Fake(2 * GB, (4,), F32), weight=Fake(3 * GB, (10, 24), I8),
             weight_scales=Fake(4 * GB, (10,), F32), out=Fake(5 * GB, (4, 10), BF16))
    a.update(kw)
    O.linear_i8(None, **a)


def _cross(q_lens=(2, 0, 3), k_lens=(4, 5, 0), heads=6, kv_heads=2, width=40, dtype=F16, **kw):
    a = dict(q=Fake(1 * GB, (5, heads, width), dtype), k=Fake(2 * GB, (9, kv_heads, width), dtype),
             v=Fake(3 * GB, (9, kv_heads, width), dtype), out=Fake(4 * GB, (5, heads, width), dtype))
    a.update(kw)
    O.check_cross(q_lens, k_lens, heads, kv_heads, width, dtype, **a)


def _status(call, **kw):
    with pytest.raises(T.TurboError) as e:
        call(**kw)
    return e.value.code, e.value.field


NO_CONTEXT = (S.TURBO_E_INVALID_HANDLE, 0)
ARG, SHAPE = S.TURBO_E_INVALID_ARGUMENT, S.TURBO_E_INVALID_SHAPE


@pytest.mark.parametrize("kw", [
    {}, dict(residual=Fake(4 * GB, (4, 24), F16)), dict(residual=Fake(4 * GB, (4, 24), F32)),
    dict(weight=Fake(2 * GB, (24,), F16)), dict(out=Fake(3 * GB, (4, 24), F32)), dict(out=Fake(3 * GB, (4, 24), BF16)),
    dict(out=Fake(1 * GB, (4, 24), F16)),                                        # in place
    dict(x=Fake(1 * GB, (4, 24), F16, (0, 1))),                                    # one row repeated
    dict(out=Fake(1 * GB + 48, (4, 24), F16, (48, 1)), x=Fake(1 * GB, (4, 24), F16, (48, 1))),   # side by side
    dict(residual=Fake(4 * GB, (4, 24), F16), sum=Fake(4 * GB, (4, 24), F16)),
    dict(residual=Fake(4 * GB, (4, 24), F16), sum=Fake(1 * GB, (4, 24), F16)),
    dict(out=None, codes=Fake(5 * GB, (4, 24), I8), scales=Fake(6 * GB, (4,), F32)),
    dict(x=Fake(0, (0, 24), F16), out=Fake(0, (0, 24), F16)),                      # no rows
])
def test_a_norm_with_nothing_wrong_gets_as_far_as_its_context(kw):
    assert _status(_norm, **kw) == NO_CONTEXT


@pytest.mark.parametrize("kw, want", [
    (dict(eps=0.0), (ARG, 0)), (dict(eps=float("nan")), (ARG, 0)), (dict(eps=float("inf")), (ARG, 0)),
    (dict(x=Fake(1 * GB, (4, 24), I8)), (ARG, 1)), (dict(x=Fake(1 * GB, (96,), F16)), (SHAPE, 1)),
    (dict(x=Fake(1 * GB + 1, (4, 24), F16)), (ARG, 1)), (dict(x=Fake(0, (4, 24), F16)), (ARG, 1)),
    (dict(x=Fake(1 * GB, (4, 65537), F16), weight=Fake(2 * GB, (65537,), F32), out=Fake(3 * GB, (4, 65537), F16)),
     (SHAPE, 1)),
    (dict(residual=Fake(4 * GB, (4, 24), BF16)), (ARG, 2)), (dict(residual=Fake(4 * GB, (3, 24), F16)), (SHAPE, 2)),
    (dict(weight=Fake(2 * GB, (23,), F32)), (SHAPE, 3)), (dict(weight=Fake(2 * GB, (24,), BF16)), (ARG, 3)),
    (dict(weight=None), (ARG, 3)),
    (dict(sum=Fake(4 * GB, (4, 24), F16)), (ARG, 4)),
    (dict(residual=Fake(4 * GB, (4, 24), F32), sum=Fake(5 * GB, (4, 24), F16)), (ARG, 4)),
    (dict(residual=Fake(4 * GB, (4, 24), F16), sum=Fake(4 * GB + 2, (4, 24), F16)), (ARG, 4)),
    (dict(residual=Fake(4 * GB, (4, 24), F16), sum=Fake(3 * GB, (4, 24), F16)), (ARG, 5)),   # sum is out
    (dict(residual=Fake(4 * GB, (4, 24), F32), sum=Fake(1 * GB, (4, 24), F32)), (ARG, 4)),   # over x of another type
    (dict(out=None), (ARG, 5)), (dict(out=Fake(3 * GB, (4, 25), F16)), (SHAPE, 5)),
    (dict(out=Fake(3 * GB, (4, 24), F16, (23, 1))), (ARG, 5)), (dict(out=Fake(3 * GB, (4, 24), F16, (0, 1))), (ARG, 5)),
    (dict(out=Fake(1 * GB + 46, (4, 24), F16, (48, 1)), x=Fake(1 * GB, (4, 24), F16, (48, 1))), (ARG, 5)),
    (dict(out=Fake(2 * GB + 40, (4, 24), F16)), (ARG, 5)),                         # over the weight
    (dict(codes=Fake(5 * GB, (4, 24), I8)), (ARG, 7)), (dict(scales=Fake(5 * GB, (4,), F32)), (ARG, 6)),
    (dict(codes=Fake(1 * GB, (4, 24), I8), scales=Fake(6 * GB, (4,), F32)), (ARG, 6)),
    (dict(codes=Fake(5 * GB, (4, 24), I8), scales=Fake(6 * GB, (5,), F32)), (SHAPE, 7)),
    (dict(codes=Fake(5 * GB, (4, 24), I8), scales=Fake(5 * GB + 92, (4,), F32)), (ARG, 7)),
])
def test_a_norm_refuses(kw, want):
    assert _status(_norm, **kw) == want


def test_a_norm_s_call_struct_is_checked():
    lib = T.library()
    size = O._NORM.size
    assert size == 24 + 7 * 64
    rest = [1e-6, *O._tensor(Fake(GB, (1, 8), F16)), *O._ABSENT, *O._tensor(Fake(2 * GB, (8,), F32)), *O._ABSENT,
            *O._tensor(Fake(3 * GB, (1, 8), F16)), *O._ABSENT, *O._ABSENT]

    def rc(*head):
        return lib.turbo_rocm_rms_norm(None, O._NORM.pack(*head, *rest), C.byref(S.new_error()))
    assert rc(size, 0, 0) == S.TURBO_E_INVALID_HANDLE
    assert rc(size - 8, 0, 0) == S.TURBO_E_INVALID_STRUCT_SIZE
    assert rc(size, 2, 0) == ARG                    # a flag nobody knows
    assert rc(size, 0, 4096) == ARG                 # a stream without TURBO_ROCM_ENQUEUE
    assert lib.turbo_rocm_rms_norm(None, None, C.byref(S.new_error())) == ARG
    assert lib.turbo_rocm_rms_norm(None, O._NORM.pack(size, 0, 0, *rest), None) == S.TURBO_E_INVALID_HANDLE


def test_an_array_that_reaches_past_its_bytes_is_refused():
    lib = T.library()
    x = list(O._tensor(Fake(GB, (3, 8), F16, (20, 1))))
    rest = [*O._tensor(Fake(2 * GB, (3, 8), I8)), *O._tensor(Fake(3 * GB, (3,), F32))]

    def rc(x):
        return lib.turbo_rocm_quantize_tokens(None, O._CODES.pack(O._CODES.size, 0, 0, *x, *rest),
                                              C.byref(S.new_error()))
    assert x[1] == (2 * 20 + 8) * 2 and rc(x) == S.TURBO_E_INVALID_HANDLE
    assert rc(x[:1] + [x[1] - 1] + x[2:]) == ARG
    # Strides and shapes whose product passes 64 bits reach past any bytes.
    assert rc(x[:1] + [(1 << 64) - 1] + x[2:5] + [1 << 63] + x[6:]) == ARG
    assert rc(x[:2] + [1 << 31] + x[3:]) == SHAPE
    assert rc(x[:7] + [4] + x[8:]) == SHAPE          # four axes
    assert rc(x[:8] + [77]) == ARG                   # a type nobody knows


@pytest.mark.parametrize("kw, want", [
    ({}, NO_CONTEXT), (dict(x=Fake(GB, (4, 24), F32)), NO_CONTEXT),
    (dict(x=Fake(GB, (4, 24), I32)), (ARG, 1)), (dict(codes=None), (ARG, 2)), (dict(scales=None), (ARG, 3)),
    (dict(codes=Fake(2 * GB, (4, 23), I8)), (SHAPE, 2)), (dict(codes=Fake(2 * GB, (4, 24), I8, (12, 1))), (ARG, 2)),
    (dict(codes=Fake(GB, (4, 24), I8)), (ARG, 2)), (dict(scales=Fake(2 * GB, (4,), F32)), (ARG, 3)),
    (dict(scales=Fake(3 * GB, (3,), F32)), (SHAPE, 3)),
])
def test_quantize_tokens_checks(kw, want):
    assert _status(_tokens, **kw) == want


@pytest.mark.parametrize("kw, want", [
    ({}, NO_CONTEXT), (dict(bias=Fake(6 * GB, (10,), F32)), NO_CONTEXT),
    (dict(codes=Fake(GB, (4, 0), I8), weight=Fake(3 * GB, (10, 0), I8)), NO_CONTEXT),
    (dict(codes=Fake(GB, (4, 131071), I8), weight=Fake(3 * GB, (10, 131071), I8)), NO_CONTEXT),
    (dict(codes=Fake(GB, (4, 131072), I8), weight=Fake(3 * GB, (10, 131072), I8)), (SHAPE, 1)),
    (dict(codes=Fake(GB, (4, 24), F16)), (ARG, 1)), (dict(scales=Fake(2 * GB, (5,), F32)), (SHAPE, 2)),
    (dict(scales=Fake(2 * GB, (4,), F16)), (ARG, 2)), (dict(weight=Fake(3 * GB, (10, 23), I8)), (SHAPE, 3)),
    (dict(weight_scales=None), (ARG, 4)), (dict(bias=Fake(6 * GB, (10,), F16)), (ARG, 5)),
    (dict(bias=Fake(6 * GB, (9,), F32)), (SHAPE, 5)), (dict(out=Fake(5 * GB, (4, 10), I32)), (ARG, 6)),
    (dict(out=Fake(5 * GB, (10, 4), F16)), (SHAPE, 6)), (dict(out=Fake(4 * GB - 4, (4, 10), F32)), (ARG, 6)),
    (dict(out=Fake(5 * GB, (4, 10), F32, (9, 1))), (ARG, 6)),
])
def test_linear_i8_checks(kw, want):
    assert _status(_linear, **kw) == want


def test_cross_attention_takes():
    _cross()
    _cross(mask=Fake(6 * GB, (9,), I32), scale=-2.0)
    _cross(kv_heads=6)
    _cross(q=Fake(1 * GB, (7, 6, 40), F16), out=Fake(4 * GB, (8, 6, 40), F16))    # rows past the last sequence
    # Keys and values side by side, and head by head.
    _cross(k=Fake(2 * GB, (9, 2, 40), F16, (160, 40, 1)), v=Fake(2 * GB + 160, (9, 2, 40), F16, (160, 40, 1)))
    _cross(q=Fake(1 * GB, (5, 6, 40), F16, (40, 200, 1)), out=Fake(4 * GB, (5, 6, 40), F16, (40, 200, 1)))
    _cross((), (), q=Fake(0, (0, 6, 40), F16), k=Fake(0, (0, 2, 40), F16), v=Fake(0, (0, 2, 40), F16),
           out=Fake(0, (0, 6, 40), F16))
    O.check_cross((1,), (1,), 1, 1, 128, F32)


@pytest.mark.parametrize("kw, want", [
    (dict(dtype=I8), (S.TURBO_E_INVALID_ENUM, 0)), (dict(heads=5), (ARG, 0)), (dict(kv_heads=0), (ARG, 0)),
    (dict(width=0), (ARG, 0)), (dict(width=129), (ARG, 0)),
    (dict(q_lens=(1 << 28, 1 << 28, 0)), (S.TURBO_E_CAPACITY, 0)),
    (dict(k_lens=(1 << 31, 1 << 31, 0)), (S.TURBO_E_CAPACITY, 0)),
    (dict(scale=float("inf")), (ARG, 0)), (dict(scale=float("nan")), (ARG, 0)),
    (dict(q=Fake(1 * GB, (4, 6, 40), F16)), (SHAPE, 1)), (dict(q=Fake(1 * GB, (5, 6, 40), BF16)), (ARG, 1)),
    (dict(k=Fake(2 * GB, (8, 2, 40), F16)), (SHAPE, 2)), (dict(k=Fake(2 * GB, (9, 6, 40), F16)), (SHAPE, 2)),
    (dict(v=Fake(3 * GB, (9, 2, 41), F16)), (SHAPE, 3)), (dict(v=Fake(3 * GB, (9, 80), F16)), (SHAPE, 3)),
    (dict(mask=Fake(6 * GB, (8,), I32)), (SHAPE, 4)), (dict(mask=Fake(6 * GB, (9,), I8)), (ARG, 4)),
    (dict(out=Fake(1 * GB, (5, 6, 40), F16)), (ARG, 5)), (dict(out=Fake(4 * GB, (3, 6, 40), F16)), (SHAPE, 5)),
    (dict(out=Fake(4 * GB, (5, 6, 40), F16, (40, 40, 1))), (ARG, 5)),
    (dict(out=Fake(4 * GB, (5, 6, 40), F16, (240, 39, 1))), (ARG, 5)),
])
def test_cross_attention_refuses(kw, want):
    assert _status(_cross, **kw) == want


def test_a_plan_needs_a_context_and_a_call_a_plan():
    assert _status(lambda: O.CrossPlan(None, (1,), (1,), 1, 1, 8, F16)) == NO_CONTEXT
    packed = O._cross_call(*[Fake((i + 1) * GB, (1, 1, 8), F16) for i in range(4)], None, None, None, None, 8)
    err = S.new_error()
    assert T.library().turbo_rocm_cross_attention(None, packed, C.byref(err)) == S.TURBO_E_INVALID_HANDLE
    T.library().turbo_rocm_cross_plan_release(None)
    with pytest.raises(ValueError):
        O.check_cross((1, 2), (1,), 1, 1, 8, F16)


def test_the_host_side_refuses_what_the_struct_cannot_say():
    with pytest.raises(ValueError):
        _norm(x=Fake(GB, (4, 24), F16, (1, 4)))       # columns that are not contiguous
    with pytest.raises(ValueError):
        _norm(x=Fake(GB, (1, 1, 4, 24), F16))
    with pytest.raises(TypeError):
        _norm(x=Fake(GB, (4, 24), "torch.float64"))
    host = Fake(GB, (4, 24), F16)
    host.is_cuda = False
    with pytest.raises(ValueError):
        _norm(x=host)


def test_the_int8_products_of_the_tests_reach_every_kernel():
    from test_gpu_linear_kernels import KERNELS
    for kernel, aligned, m, n, k in KERNELS:
        assert O.linear_i8_kernel(m, n, k, aligned) == kernel, (m, n, k)
        assert not aligned or k % 16 == 0 or kernel == 0
    # (Tiles of 256 need whole chunks; the others go both ways, tiles with few stages and with many.)
    assert {(c[0], c[1]) for c in KERNELS} == {(i, a) for i in (0, 1, 2, 3, 4, 64, 128, 256) for a in (True, False)} - {(256, False)}
    assert {(c[0], c[1]) for c in KERNELS if c[0] >= 64 and c[4] > 3 * 128} == {(64, True), (64, False), (128, True),
                                                                                (128, False), (256, True)}
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 131072), (1 << 31, 1, 1)):
        with pytest.raises(T.TurboError):
            O.linear_i8_kernel(*bad, True)


def test_the_attentions_of_the_tests_reach_every_kernel():
    from test_gpu_cross_kernels import KERNELS, lengths
    seen, cuts = set(), set()
    for half, rows, one_tile, joined, n, nq, most, kv, share, d in KERNELS:
        k_lens = lengths(n, most)
        r, states = O.cross_cut([nq] * n, k_lens, kv * share, kv, d, F16 if half else F32)
        assert (r, max(k_lens) > states, nq * share <= 32) == (rows, joined, one_tile), (half, rows, n, nq, most, d)
        # (One wave's kernel is the same for one row tile and for several; an F32 one for four waves too.)
        seen.add((half, rows, one_tile if half and rows == 128 else None, (d + 31) // 32))
        cuts.add((half, rows, one_tile, joined))
    want = {(half, 32, None, w) for half in (True, False) for w in (1, 2, 3, 4)}
    want |= {(True, 128, one, w) for one in (True, False) for w in (1, 2, 3, 4)} | {(False, 128, None, w) for w in (1, 2, 3, 4)}
    assert seen == want
    assert cuts == {(h, r, o, j) for h in (True, False) for r in (32, 128) for o in (True, False) for j in (True, False)}
    with pytest.raises(T.TurboError):
        O.cross_cut((1,), (1,), 3, 2, 64, F16)


def test_an_array_over_a_closed_buffer_is_refused():
    class Closed:
        t, h, nbytes = T.table(), None, 64
    with pytest.raises(ValueError, match="closed"):
        T.DeviceArray(Closed, (16,), F32)


@pytest.mark.parametrize("kw", [
    dict(q_lens=((1 << 32) + 2, 0, 3)), dict(k_lens=(4, (1 << 33) + 5, 0)), dict(q_lens=(2, -1, 3)), dict(k_lens=(4, 5, -4)),
    dict(heads=(1 << 32) + 6), dict(kv_heads=(1 << 32) + 2), dict(width=(1 << 32) + 40)])
def test_a_plan_s_numbers_are_not_cut_to_32_bits(kw):
    a = dict(dict(q_lens=(2, 0, 3), k_lens=(4, 5, 0), heads=6, kv_heads=2, width=40), **kw)
    O.check_cross((2, 0, 3), (4, 5, 0), 6, 2, 40, F16)
    with pytest.raises(ValueError):
        O.check_cross(a["q_lens"], a["k_lens"], a["heads"], a["kv_heads"], a["width"], F16)
