"""Attention over prompts and over a cache of states, its writes and its reads, without a device: what their calls
refuse, with which status and which array, and that a call with nothing wrong gets as far as the missing context."""
import ctypes as C

import pytest

import turboembed_amd as T
from turboembed_amd import operators as O
from turboembed_amd import seam as S
from test_operators import ARG, BF16, F16, F32, GB, I32, I8, NO_CONTEXT, SHAPE, Fake, _status

CAPACITY = S.TURBO_E_CAPACITY
A, K, N, W, P, COLS, PAGE = 5, 2, 3, 40, 6, 4, 16      # tokens, key heads, sequences, width, pages, a sequence's columns


def _cache(t=F16, page=PAGE, **kw):
    a = dict(k=Fake(10 * GB, (P * PAGE, K, W), t), v=Fake(11 * GB, (P * PAGE, K, W), t), page_tokens=page)
    if t == I8:
        a.update(k_scales=Fake(12 * GB, (P * PAGE, K), F32), v_scales=Fake(13 * GB, (P * PAGE, K), F32))
    a.update(kw)
    return T.StateCache(**a)


def _arrays(kw):
    return [kw.pop(n, x) for n, x in (("starts", Fake(20 * GB, (N + 1,), I32)), ("lengths", Fake(21 * GB, (N,), I32)),
                                      ("pages", Fake(22 * GB, (N, COLS), I32)))]


def _write(cache=None, **kw):
    arrays = _arrays(kw)
    a = dict(k=Fake(1 * GB, (A, K, W), F16), v=Fake(2 * GB, (A, K, W), F16))
    a.update(kw)
    O.cache_write(None, a["k"], a["v"], cache or _cache(), *arrays)


def _read(cache=None, **kw):
    arrays = _arrays(kw)
    a = dict(k=Fake(1 * GB, (A, K, W), F16), v=Fake(2 * GB, (A, K, W), F16))
    a.update(kw)
    O.cache_read(None, cache or _cache(), *arrays, a["k"], a["v"])


def _attend(cache=None, **kw):
    arrays = _arrays(kw)
    need = O.cache_workspace(A, N, 6, K, W, F16)
    a = dict(q=Fake(1 * GB, (A, 6, W), F16), out=Fake(2 * GB, (A, 6, W), F16), workspace=Fake(3 * GB, (need + 64,), I8))
    a.update(kw)
    O.cache_attention(None, a.pop("q"), cache or _cache(), *arrays, a.pop("out"), **a)


def _prompt(**kw):
    a = dict(q=Fake(1 * GB, (A, 6, W), F16), k=Fake(2 * GB, (A, K, W), F16), v=Fake(3 * GB, (A, K, W), F16),
             starts=Fake(20 * GB, (N + 1,), I32), out=Fake(4 * GB, (A, 6, W), F16))
    a.update(kw)
    O.prompt_attention(None, **a)


ROWS = [
    ({}, NO_CONTEXT), (dict(cache=_cache(I8)), NO_CONTEXT),
    (dict(starts=Fake(0, (1,), I32), lengths=Fake(0, (0,), I32), pages=Fake(0, (0, 4), I32)), (ARG, 7)),   # (an address)
    (dict(starts=Fake(GB * 20, (1,), I32), lengths=Fake(0, (0,), I32), pages=Fake(0, (0, 4), I32)), NO_CONTEXT),
    (dict(pages=Fake(0, (N, 0), I32)), NO_CONTEXT),
    (dict(cache=_cache(k=Fake(0, (0, K, W), F16), v=Fake(0, (0, K, W), F16))), NO_CONTEXT),
    (dict(k=Fake(0, (0, K, W), F16), v=Fake(0, (0, K, W), F16)), NO_CONTEXT),
    # K and V of a slot side by side, and head by head.
    (dict(cache=_cache(k=Fake(10 * GB, (96, K, W), F16, (4 * W, W, 1)), v=Fake(10 * GB + 4 * W, (96, K, W), F16, (4 * W, W, 1)))),
     NO_CONTEXT),
    (dict(cache=_cache(k=Fake(10 * GB, (96, K, W), F16, (W, 96 * W, 1)))), NO_CONTEXT),
    (dict(k=Fake(GB, (A, K, W), I8)), (ARG, 1)), (dict(k=Fake(GB, (A, K * W), F16)), (SHAPE, 1)),
    (dict(k=Fake(GB, (A, K, 129), F16), v=Fake(2 * GB, (A, K, 129), F16)), (SHAPE, 1)),
    (dict(k=Fake(GB, (A, K, 0), F16), v=Fake(2 * GB, (A, K, 0), F16)), (SHAPE, 1)),
    (dict(k=Fake(GB, (A, 0, W), F16), v=Fake(2 * GB, (A, 0, W), F16)), (SHAPE, 1)),
    (dict(k=Fake(GB, ((1 << 29) + 1, K, W), F16), v=Fake(200 * GB, ((1 << 29) + 1, K, W), F16)), (CAPACITY, 1)),
    (dict(v=Fake(2 * GB, (A, K, W), BF16)), (ARG, 2)), (dict(v=Fake(2 * GB, (A + 1, K, W), F16)), (SHAPE, 2)),
    (dict(v=None), (ARG, 2)),
    (dict(cache=_cache(BF16)), (ARG, 3)), (dict(cache=_cache(k=Fake(10 * GB, (96, K + 1, W), F16))), (SHAPE, 3)),
    (dict(cache=_cache(k=Fake(10 * GB, (96, K, W + 1), F16))), (SHAPE, 3)), (dict(cache=_cache(k=None)), (ARG, 3)),
    (dict(cache=_cache(k=Fake(10 * GB, ((1 << 30) + 1, K, W), F16))), (CAPACITY, 3)),
    (dict(cache=_cache(v=Fake(11 * GB, (95, K, W), F16))), (SHAPE, 4)), (dict(cache=_cache(v=Fake(11 * GB, (96, K, W), I8))), (ARG, 4)),
    (dict(cache=_cache(k_scales=Fake(12 * GB, (96, K), F32))), (ARG, 5)), (dict(cache=_cache(v_scales=Fake(12 * GB, (96, K), F32))), (ARG, 6)),
    (dict(cache=_cache(I8, k_scales=None)), (ARG, 5)), (dict(cache=_cache(I8, v_scales=None)), (ARG, 6)),
    (dict(cache=_cache(I8, k_scales=Fake(12 * GB, (96, K), F16))), (ARG, 5)),
    (dict(cache=_cache(I8, v_scales=Fake(13 * GB, (96, K + 1), F32))), (SHAPE, 6)),
    (dict(cache=_cache(page=0)), (ARG, 0)), (dict(cache=_cache(page=(1 << 30) + 1)), (ARG, 0)),
    (dict(starts=Fake(20 * GB, (0,), I32)), (SHAPE, 7)), (dict(starts=Fake(20 * GB, (N + 2,), I32)), (SHAPE, 8)),
    (dict(starts=Fake(20 * GB, (N + 1,), F32)), (ARG, 7)), (dict(starts=None), (ARG, 7)),
    (dict(lengths=Fake(21 * GB, (N - 1,), I32)), (SHAPE, 8)), (dict(lengths=None), (ARG, 8)),
    (dict(pages=Fake(22 * GB, (N + 1, COLS), I32)), (SHAPE, 9)), (dict(pages=Fake(22 * GB, (N * COLS,), I32)), (SHAPE, 9)),
    (dict(pages=Fake(22 * GB, (N, 1 << 27), I32, (0, 1))), (CAPACITY, 9)), (dict(pages=None), (ARG, 9)),
]


@pytest.mark.parametrize("kw, want", ROWS)
def test_rows_of_a_cache(kw, want):
    assert _status(_write, **dict(kw)) == want
    assert _status(_read, **dict(kw)) == want


@pytest.mark.parametrize("kw, want", [
    # The cache over itself, over the rows and over the arrays that say where.
    (dict(cache=_cache(v=Fake(10 * GB, (96, K, W), F16))), (ARG, 4)),
    (dict(cache=_cache(k=Fake(10 * GB, (96, K, W), F16, (K * W - 1, W, 1)))), (ARG, 3)),
    (dict(cache=_cache(k=Fake(10 * GB, (96, K, W), F16, (0, W, 1)))), (ARG, 3)),
    (dict(cache=_cache(I8, v_scales=Fake(12 * GB, (96, K), F32))), (ARG, 6)),
    (dict(cache=_cache(I8, k_scales=Fake(10 * GB + 64, (96, K), F32))), (ARG, 5)),
    (dict(k=Fake(10 * GB, (A, K, W), F16)), (ARG, 3)), (dict(v=Fake(11 * GB + 80, (A, K, W), F16)), (ARG, 4)),
    (dict(pages=Fake(10 * GB, (N, COLS), I32)), (ARG, 3)), (dict(starts=Fake(11 * GB, (N + 1,), I32)), (ARG, 4)),
    # Rows that repeat, or that are each other, are inputs like any.
    (dict(k=Fake(1 * GB, (A, K, W), F16, (0, W, 1))), NO_CONTEXT), (dict(v=Fake(1 * GB, (A, K, W), F16)), NO_CONTEXT),
])
def test_a_write_s_overlaps(kw, want):
    assert _status(_write, **kw) == want


@pytest.mark.parametrize("kw, want", [
    (dict(v=Fake(1 * GB, (A, K, W), F16)), (ARG, 2)), (dict(k=Fake(1 * GB, (A, K, W), F16, (0, W, 1))), (ARG, 1)),
    (dict(k=Fake(10 * GB, (A, K, W), F16)), (ARG, 1)), (dict(v=Fake(22 * GB, (A, K, W), F16)), (ARG, 2)),
    (dict(cache=_cache(v=Fake(10 * GB, (96, K, W), F16))), NO_CONTEXT),
    (dict(cache=_cache(I8), k=Fake(GB, (A, K, W), F32), v=Fake(2 * GB, (A, K, W), F32)), NO_CONTEXT),
])
def test_a_read_s_overlaps(kw, want):
    assert _status(_read, **kw) == want


@pytest.mark.parametrize("kw, want", [
    ({}, NO_CONTEXT), (dict(cache=_cache(I8)), NO_CONTEXT), (dict(window=4294967295, scale=-2.0), NO_CONTEXT),
    (dict(q=Fake(GB, (A, 6, W), F16, (0, W, 1))), NO_CONTEXT),
    (dict(cache=_cache(v=Fake(10 * GB, (96, K, W), F16))), NO_CONTEXT),       # keys that are the values
    (dict(scale=float("inf")), (ARG, 0)), (dict(scale=float("nan")), (ARG, 0)), (dict(scale=1e39), (ARG, 0)),
    (dict(q=Fake(GB, (A, 6, W), I8)), (ARG, 1)), (dict(q=Fake(GB, (A, 6 * W), F16)), (SHAPE, 1)),
    (dict(q=Fake(GB, (A, 5, W), F16), out=Fake(2 * GB, (A, 5, W), F16)), (SHAPE, 1)),
    (dict(q=Fake(GB, (A, 0, W), F16), out=Fake(2 * GB, (A, 0, W), F16)), (SHAPE, 1)),
    (dict(q=Fake(GB, (A, 6, 129), F16), out=Fake(2 * GB, (A, 6, 129), F16)), (SHAPE, 1)),
    (dict(q=Fake(GB, (1 << 28, 6, W), F16), out=Fake(1000 * GB, (1 << 28, 6, W), F16)), (CAPACITY, 1)),
    (dict(out=Fake(2 * GB, (A, 6, W), BF16)), (ARG, 2)), (dict(out=Fake(2 * GB, (A, 4, W), F16)), (SHAPE, 2)),
    (dict(out=Fake(GB, (A, 6, W), F16)), (ARG, 2)), (dict(out=Fake(2 * GB, (A, 6, W), F16, (6 * W, 0, 1))), (ARG, 2)),
    (dict(out=Fake(10 * GB + 320, (A, 6, W), F16)), (ARG, 2)), (dict(out=Fake(21 * GB, (A, 6, W), F16)), (ARG, 2)),
    (dict(cache=_cache(BF16)), (ARG, 3)), (dict(cache=_cache(k=Fake(10 * GB, (96, K, W - 1), F16))), (SHAPE, 3)),
    (dict(cache=_cache(k=Fake(10 * GB, (96, 0, W), F16), v=Fake(11 * GB, (96, 0, W), F16))), (SHAPE, 1)),
    (dict(cache=_cache(k=Fake(10 * GB, (96, 4, W), F16), v=Fake(11 * GB, (96, 4, W), F16))), (SHAPE, 1)),
    (dict(cache=_cache(I8, k_scales=None)), (ARG, 5)), (dict(cache=_cache(page=0)), (ARG, 0)),
    (dict(starts=Fake(20 * GB, (N,), I32)), (SHAPE, 8)), (dict(lengths=None), (ARG, 8)), (dict(pages=None), (ARG, 9)),
    (dict(workspace=Fake(3 * GB + 8, (1 << 30,), I8)), (ARG, 0)),
])
def test_cache_attention_checks(kw, want):
    assert _status(_attend, **kw) == want


@pytest.mark.parametrize("kw, want", [
    ({}, NO_CONTEXT), (dict(window=7, scale=0.0), NO_CONTEXT), (dict(starts=Fake(20 * GB, (1,), I32)), NO_CONTEXT),
    (dict(k=Fake(2 * GB, (A, K, W), F16, (0, 0, 1))), NO_CONTEXT), (dict(v=Fake(2 * GB, (A, K, W), F16)), NO_CONTEXT),
    (dict(q=Fake(0, (0, 6, W), F16), k=Fake(0, (0, K, W), F16), v=Fake(0, (0, K, W), F16), out=Fake(0, (0, 6, W), F16)),
     NO_CONTEXT),
    (dict(scale=float("inf")), (ARG, 0)), (dict(q=None), (ARG, 1)), (dict(q=Fake(GB, (A, 6, W), I32)), (ARG, 1)),
    (dict(k=Fake(2 * GB, (A, 4, W), F16)), (SHAPE, 1)), (dict(k=Fake(2 * GB, (A, 0, W), F16)), (SHAPE, 1)),
    (dict(k=Fake(2 * GB, (A, K, W), F32)), (ARG, 2)), (dict(k=Fake(2 * GB, (A + 1, K, W), F16)), (SHAPE, 2)),
    (dict(v=Fake(3 * GB, (A, K, W + 1), F16)), (SHAPE, 3)), (dict(v=Fake(3 * GB, (A, K, W), I8)), (ARG, 3)),
    (dict(starts=Fake(20 * GB, (0,), I32)), (SHAPE, 4)), (dict(starts=Fake(20 * GB, (2, 2), I32)), (SHAPE, 4)),
    (dict(out=Fake(4 * GB, (A, 6, W), BF16)), (ARG, 5)), (dict(out=Fake(GB, (A, 6, W), F16)), (ARG, 5)),
    (dict(out=Fake(4 * GB, (A, 6, W), F16, (6 * W, W - 1, 1))), (ARG, 5)), (dict(out=Fake(20 * GB, (A, 6, W), F16)), (ARG, 5)),
])
def test_prompt_attention_checks(kw, want):
    if kw.get("q", 1) is None:
        with pytest.raises(AttributeError):
            _prompt(**kw)
        kw = dict(kw, q=Fake(0, (0,), F16))
        want = (SHAPE, 1)
    assert _status(_prompt, **kw) == want


def test_the_call_structs_are_checked():
    lib = T.library()
    x = O._tensor(Fake(GB, (A, K, W), F16))
    arrays = [*x, *O._tensor(Fake(2 * GB, (A, K, W), F16)), *O._ABSENT, *O._ABSENT, *O._tensor(Fake(4 * GB, (2,), I32)),
              *O._tensor(Fake(5 * GB, (1,), I32)), *O._tensor(Fake(6 * GB, (1, 1), I32))]
    rows = [*O._tensor(Fake(7 * GB, (A, K, W), F16)), *O._tensor(Fake(8 * GB, (A, K, W), F16))]
    assert O._ROWS.size == 16 + 9 * 64 + 8 and O._CACHED.size == 48 + 9 * 64 + 8 and O._PROMPT.size == 32 + 5 * 64

    def rc(name, layout, *fields):
        return getattr(lib, name)(None, layout.pack(*fields), C.byref(S.new_error()))
    for name in ("turbo_rocm_cache_write", "turbo_rocm_cache_read"):
        size = O._ROWS.size
        assert rc(name, O._ROWS, size, 0, 0, *rows, *arrays, 1, 0) == S.TURBO_E_INVALID_HANDLE
        assert rc(name, O._ROWS, size + 8, 0, 0, *rows, *arrays, 1, 0) == S.TURBO_E_INVALID_STRUCT_SIZE
        assert rc(name, O._ROWS, size, 2, 0, *rows, *arrays, 1, 0) == ARG       # a flag nobody knows
        assert rc(name, O._ROWS, size, 0, 4096, *rows, *arrays, 1, 0) == ARG    # a stream without TURBO_ROCM_ENQUEUE
        assert rc(name, O._ROWS, size, 0, 0, *rows, *arrays, 1, 1) == ARG       # the reserved field
        assert getattr(lib, name)(None, None, C.byref(S.new_error())) == ARG
        assert getattr(lib, name)(None, O._ROWS.pack(size, 0, 0, *rows, *arrays, 1, 0), None) == S.TURBO_E_INVALID_HANDLE
    size, name = O._CACHED.size, "turbo_rocm_cache_attention"
    need = O.cache_workspace(A, 1, K, K, W, F16)
    assert rc(name, O._CACHED, size, 0, 0, 16 * GB, need, 1.0, 0, 0, *rows, *arrays, 1, 0) == S.TURBO_E_INVALID_HANDLE
    assert rc(name, O._CACHED, size - 8, 0, 0, 16 * GB, need, 1.0, 0, 0, *rows, *arrays, 1, 0) == S.TURBO_E_INVALID_STRUCT_SIZE
    assert rc(name, O._CACHED, size, 0, 0, 16 * GB, need, 1.0, 0, 1, *rows, *arrays, 1, 0) == ARG
    if need:
        assert rc(name, O._CACHED, size, 0, 0, 16 * GB, need - 1, 1.0, 0, 0, *rows, *arrays, 1, 0) == CAPACITY
        assert rc(name, O._CACHED, size, 0, 0, 0, need, 1.0, 0, 0, *rows, *arrays, 1, 0) == CAPACITY
        # A workspace over the output, and over a table.
        for at in (8 * GB, 6 * GB):
            assert rc(name, O._CACHED, size, 0, 0, at, need, 1.0, 0, 0, *rows, *arrays, 1, 0) == ARG
    size, name = O._PROMPT.size, "turbo_rocm_prompt_attention"
    own = [*rows, *x, *O._tensor(Fake(4 * GB, (2,), I32)), *O._tensor(Fake(9 * GB, (A, K, W), F16))]
    assert rc(name, O._PROMPT, size, 0, 0, 1.0, 0, 0, *own) == S.TURBO_E_INVALID_HANDLE
    assert rc(name, O._PROMPT, size, 0, 0, 1.0, 0, 3, *own) == ARG
    assert rc(name, O._PROMPT, 0, 0, 0, 1.0, 0, 0, *own) == S.TURBO_E_INVALID_STRUCT_SIZE


def test_a_workspace_s_size():
    assert O.cache_workspace(0, 0, 1, 1, 1, F32) % 16 == 0
    # More tokens or sequences never need less.
    for heads, kv, width, t in ((8, 2, 64, F16), (32, 8, 128, BF16), (16, 1, 80, F32), (200, 1, 32, F16)):
        sizes = [O.cache_workspace(n, s, heads, kv, width, t) for n in (0, 1, 2, 40, 300, 5000, 60000) for s in (0, 1, 3, 64, 700)]
        for i in range(7):
            assert sizes[5 * i:5 * i + 5] == sorted(sizes[5 * i:5 * i + 5])
        for j in range(5):
            assert sizes[j::5] == sorted(sizes[j::5])
        assert max(sizes) < 1 << 30
    for bad in ((1, 1, 3, 2, 64, F16), (1, 1, 0, 0, 64, F16), (1, 1, 1, 1, 0, F16), (1, 1, 1, 1, 129, F16), (1, 1, 1, 1, 64, I8),
                (1 << 30, 1, 2, 2, 64, F16), (1, 1 << 31, 1, 1, 64, F16)):
        with pytest.raises(T.TurboError):
            O.cache_workspace(*bad)
    for bad in ((-1, 1, 1, 1, 64, F16), (1, 1 << 64, 1, 1, 64, F16), (1, 1, (1 << 32) + 1, 1, 64, F16)):
        with pytest.raises(ValueError):
            O.cache_workspace(*bad)
    assert T.library().turbo_rocm_cache_workspace(1, 1, 1, 1, 64, F16, None, C.byref(S.new_error())) == ARG


def test_numbers_are_not_cut_to_32_bits():
    for bad in (-1, (1 << 32) + 1):
        with pytest.raises(ValueError):
            _prompt(window=bad)
        with pytest.raises(ValueError):
            _attend(window=bad)
        with pytest.raises(ValueError):
            _cache(page=bad)


def test_calls_of_too_many_workgroups_are_refused():
    # 2^23 sequences of a token each, four waves a workgroup: 2^31 threads and those of a block more.
    n = 1 << 23
    one = dict(q=Fake(1 * GB, (n, 1, 8), F16), k=Fake(2 * GB, (n, 1, 8), F16), v=Fake(3 * GB, (n, 1, 8), F16), out=Fake(4 * GB, (n, 1, 8), F16))
    assert _status(lambda: _prompt(**one, starts=Fake(20 * GB, (n + 1,), I32))) == (CAPACITY, 0)
    assert _status(lambda: _prompt(**one, starts=Fake(20 * GB, (n // 2 + 1,), I32))) == NO_CONTEXT
    # 2^20 key heads: eight workgroups of each, of 256 threads, are 2^31.
    for k, want in ((1 << 20, NO_CONTEXT), ((1 << 20) + 1, (CAPACITY, 0))):
        need = O.cache_workspace(1, N, k, k, 8, F16)
        rows = dict(q=Fake(40 * GB, (1, k, 8), F16), out=Fake(41 * GB, (1, k, 8), F16), workspace=Fake(50 * GB, (need,), I8))
        cache = _cache(k=Fake(10 * GB, (P * PAGE, k, 8), F16), v=Fake(30 * GB, (P * PAGE, k, 8), F16))
        assert _status(lambda: _attend(cache, **rows)) == want
