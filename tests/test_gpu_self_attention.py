"""Attention of a call's own tokens, over its rows and over a cache of states, on an MI355X against 64-bit arithmetic on
the same inputs (the tolerance: paged.check_rows)."""
import math

import pytest

import turboembed_amd as T
from turboembed_amd import seam as S

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from paged import TYPES, Cache, check, check_rows, ints, starts_of, stream  # noqa: E402


def _rows(seed, n, heads, d, t, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, heads, d, generator=g) * spread).to(TYPES[t]).cuda()


def _workspace(context, cache, heads, tokens=None):
    tokens = sum(cache.rows) if tokens is None else tokens
    need = context.cache_workspace(tokens, len(cache.rows), heads, cache.kv, cache.d, cache.dtype)
    # (Whatever it holds: nothing is kept in it between calls.)
    return torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")


def _attend(context, cache, q, window=0, scale=None, out=None, workspace=None):
    out = torch.full_like(q, 3.0) if out is None else out
    workspace = _workspace(context, cache, q.shape[1], len(q)) if workspace is None else workspace
    context.cache_attention(q, cache.operand(T), *cache.arrays(), out, window=window, scale=scale, workspace=workspace,
                            stream=stream())
    return out


def _check_prompt(out, q, k, v, rows, window=0, scale=None):
    at = 0
    for m in rows:
        check_rows(out[at:at + m], q[at:at + m], 0, k[at:at + m].double(), v[at:at + m].double(), window, scale)
        at += m


def _prompt(context, q, k, v, rows, window=0, scale=None, out=None):
    out = torch.full_like(q, 3.0) if out is None else out
    context.prompt_attention(q, k, v, starts_of(rows), out, window=window, scale=scale, stream=stream())
    _check_prompt(out, q, k, v, rows, window, scale)
    return out


PROMPTS = [(1,), (2,), (31,), (32,), (33,), (64,), (65,), (1, 1, 1), (5, 0, 9, 40), (128,), (129,), (300, 7, 1, 64), (513, 100),
           (1,) * 70, tuple(range(1, 30)), (1100,)]


@pytest.mark.parametrize("rows", PROMPTS, ids=lambda x: "-".join(map(str, x[:5])))
@pytest.mark.parametrize("heads, kv, d", [(1, 1, 64), (6, 2, 64), (4, 4, 32), (8, 1, 128), (3, 3, 80)])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_a_prompt_is_the_formula_s(context, rows, heads, kv, d, t):
    n = sum(rows)
    q, k, v = _rows(n, n, heads, d, t), _rows(n + 1, n, kv, d, t), _rows(n + 2, n, kv, d, t)
    _prompt(context, q, k, v, rows)
    for window in (1, 5, 64, 200):
        _prompt(context, q, k, v, rows, window=window)


@pytest.mark.parametrize("d", [1, 2, 3, 7, 8, 9, 16, 24, 31, 33, 40, 48, 63, 65, 72, 96, 100, 112, 127])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_every_kind_of_head_width(context, d, t):
    for rows, heads, kv in (((3, 70), 2, 1), ((40,), 20, 2), ((150,), 2, 2)):
        n = sum(rows)
        _prompt(context, _rows(d, n, heads, d, t), _rows(d + 1, n, kv, d, t), _rows(d + 2, n, kv, d, t), rows)
    for held in ("same", "i8"):
        for rows, lengths in (((1, 1), (40, 90)), ((50, 9), (140, 9))):
            cache = Cache(d, rows, lengths, 2, d, t, held, 16)
            q = _rows(d + 3, sum(rows), 4, d, t)
            check(cache, q, _attend(context, cache, q))


CACHED = [((1,), (1,)), ((1,), (31,)), ((1,), (33,)), ((1, 1, 1), (64, 1, 200)), ((2,), (65,)), ((1,) * 9, (7,) * 9),
          ((1,), (3000,)), ((1,) * 5, (2000, 3, 129, 64, 700)), ((5,), (1025,)), ((16, 3), (300, 17)), ((33, 1, 70), (63, 129, 700)),
          ((129, 0, 4), (257, 5, 4)), ((300,), (700,)), ((1,) * 150, tuple(range(1, 301, 2))), ((40, 1, 1, 600), (4000, 900, 2, 650))]


@pytest.mark.parametrize("rows, lengths", CACHED, ids=lambda x: "-".join(map(str, x[:5])))
@pytest.mark.parametrize("heads, kv, d, page", [(1, 1, 64, 16), (6, 2, 64, 64), (4, 4, 32, 1), (8, 1, 128, 32), (3, 3, 80, 24),
                                                (32, 2, 128, 16), (9, 1, 48, 100)])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("held", ["same", "i8"])
def test_cache_attention_is_the_formula_s(context, rows, lengths, heads, kv, d, page, t, held):
    cache = Cache(sum(lengths), rows, lengths, kv, d, t, held, page)
    q = _rows(sum(rows), sum(rows), heads, d, t)
    check(cache, q, _attend(context, cache, q))
    for window in (1, 70):
        check(cache, q, _attend(context, cache, q, window=window), window=window)


@pytest.mark.parametrize("share", [33, 64, 100, 200])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_many_heads_of_one_key_head(context, share, t):
    for rows, lengths in (((1, 2), (50, 300)), ((40,), (90,))):
        cache = Cache(share, rows, lengths, 1, 32, t, "same", 16)
        q = _rows(share, sum(rows), share, 32, t)
        check(cache, q, _attend(context, cache, q))
    q, k, v = _rows(1, 45, share, 32, t), _rows(2, 45, 1, 32, t), _rows(3, 45, 1, 32, t)
    _prompt(context, q, k, v, (5, 40))


JUNK = (float("nan"), float("inf"), -float("inf"), 1e30)


@pytest.mark.parametrize("rows", [(3, 1, 20), (40, 200, 70)])
@pytest.mark.parametrize("window", [0, 9])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_later_tokens_are_not_seen_whatever_they_hold(context, rows, window, t):
    """Row j of every sequence from which on keys and values hold no numbers: the rows before it are the formula's."""
    n, heads, kv, d = sum(rows), 4, 2, 64
    q, k0, v0 = _rows(1, n, heads, d, t), _rows(2, n, kv, d, t), _rows(3, n, kv, d, t)
    for junk in JUNK:
        for step, only in ((0, True), (1, True), (2, False)):
            k, v, at, good = k0.clone(), v0.clone(), 0, []
            for m in rows:
                j = min(m, (m // 3 * step) or 1)
                last = min(at + j + 1, at + m) if only else at + m
                v[at + j:last] = junk
                k[at + j:last, :, 3] = junk
                good.append(j)
                at += m
            out = torch.full_like(q, 3.0)
            context.prompt_attention(q, k, v, starts_of(rows), out, window=window, stream=stream())
            at = 0
            for m, j in zip(rows, good):
                kk, vv = (x[at:at + j].double() for x in (k, v))
                check_rows(out[at:at + j], q[at:at + j], 0, kk, vv, window)
                if window and only and j + window < m:
                    # The rows past the window of that token do not see it either.
                    a, b = at + j + window, at + m
                    x, y = (torch.where(torch.arange(m, device="cuda")[:, None, None] == j, 0, z[at:at + m]).double()
                            for z in (k, v))
                    check_rows(out[a:b], q[a:b], j + window, x, y, window)
                at += m


@pytest.mark.parametrize("rows, lengths", [((3, 1, 20), (30, 100, 20)), ((40, 200, 70), (100, 220, 71))])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("held", ["same", "i8"])
def test_later_states_of_a_cache_are_not_seen_whatever_they_hold(context, rows, lengths, t, held):
    heads, kv, d = 4, 2, 64
    q = _rows(1, sum(rows), heads, d, t)
    for junk in JUNK:
        cache = Cache(2, rows, lengths, kv, d, t, held, 16)
        firsts = [n - m + m // 2 + 1 for m, n in zip(rows, lengths)]
        for i, (f, n) in enumerate(zip(firsts, lengths)):
            if f < n:
                at = cache.at(i, f, min(n, f + 2))
                for x, s in zip(cache.states, cache.scales):
                    if held == "i8":
                        s[at] = junk
                    else:
                        x[at] = junk
        out = _attend(context, cache, q)
        row = 0
        for i, (m, n, f) in enumerate(zip(rows, lengths, firsts)):
            good, at = min(m, f - (n - m)), cache.at(i, 0, min(f, n))
            check_rows(out[row:row + good], q[row:row + good], n - m, cache.values(0, at), cache.values(1, at),
                       coded=cache.scales[1][at] if held == "i8" else None)
            row += m


@pytest.mark.parametrize("m", [1, 6, 150])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_scores_that_are_infinite_or_not_numbers(context, m, t):
    rows, n, d = (m,), 200, 64
    q = _rows(5, m, 1, d, t)
    q[:, :, 0] = 1.0
    cache = Cache(6, rows, (n,), 1, d, t, "same", 16)
    k, v = cache.states
    k0 = k.clone()
    for at in (3, 40):
        slot = cache.at(0, at, at + 1)
        for bad in (float("nan"), float("inf")):
            k.copy_(k0)
            k[slot, 0, 0] = bad
            assert torch.isnan(_attend(context, cache, q)).all()
        # A state whose score is minus infinity weighs nothing.
        k.copy_(k0)
        k[slot, 0, 0] = -float("inf")
        out = _attend(context, cache, q)
        whole = cache.at(0, 0, n)
        kk, vv = cache.values(0, whole), cache.values(1, whole)
        kk[at], vv[at] = 0, 0
        kk[at, 0, 0] = -1e6
        check_rows(out, q, n - m, kk, vv)
    k.copy_(k0)
    k[cache.at(0, 0, n), 0, 0] = -float("inf")
    assert torch.isnan(_attend(context, cache, q)).all()
    # A live value that is infinite is what its product gives.
    k.copy_(k0)
    v[cache.at(0, 7, 8), 0, 5] = float("inf")
    out = _attend(context, cache, q)
    assert (out[:, 0, 5] == float("inf")).all() and torch.isfinite(out[:, 0, :5]).all()


@pytest.mark.parametrize("m", [1, 6, 150])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_int8_states_whose_scales_are_no_numbers(context, m, t):
    n, d = 200, 64
    q = _rows(5, m, 2, d, t)
    for which in (0, 1):
        cache = Cache(6, (m,), (n,), 1, d, t, "i8", 16)
        cache.scales[which][cache.at(0, 3, 4)] = float("nan")
        cache.states[which][cache.at(0, 3, 4)] = 0      # as cache_write leaves a row that has no numbers
        assert torch.isnan(_attend(context, cache, q)).all()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_int8_values_of_any_size(context, t):
    """Scales of the values from 2^-30 to 2^10 of each other, and all of them small or 0."""
    for m, n in ((1, 700), (1, 90), (60, 300)):
        q = _rows(1, m, 4, 64, t)
        for case in range(4):
            cache = Cache(2, (m,), (n,), 2, 64, t, "i8", 16)
            at = cache.at(0, 0, n)
            p = torch.arange(n, device="cuda")
            s = (torch.exp2(-30.0 + p * 40 / n), torch.exp2(10.0 - p * 40 / n), torch.full((n,), 2.0 ** -20, device="cuda"),
                 torch.zeros(n, device="cuda"))[case]
            if t == "f16":
                s = s * 2.0 ** -3       # (what F16 holds)
            cache.scales[1][at] = s[:, None].expand(n, 2)
            check(cache, q, _attend(context, cache, q))


def test_rows_that_see_nothing_are_zeros_and_others_are_left(context):
    for t in TYPES:
        for held in ("same", "i8"):
            rows, lengths = (6, 3, 5, 2, 70), (9, 7, 12, 2, 80)
            cache = Cache(5, rows, lengths, 2, 32, t, held, 4)
            n = sum(rows)
            q = _rows(6, n + 5, 4, 32, t)
            # 0: fewer states than new tokens. 1: a page that the cache does not have. 2: a length past the table.
            # 3: no states. 4: every page is none.
            cache.lengths.copy_(ints([4, 7, 90, -3, 80]))
            cache.pages[1, 0] = -1
            cache.pages[4] = cache.slots // 4
            starts = cache.starts + 2        # rows 0 and 1 and the last three are nobody's
            out = torch.full_like(q, 3.0)
            context.cache_attention(q, cache.operand(T), starts, cache.lengths, cache.pages, out,
                                    workspace=torch.empty(context.cache_workspace(n + 5, 5, 4, 2, 32, TYPES[t]),
                                                          dtype=torch.uint8, device="cuda"), stream=stream())
            assert (out[:2] == 3).all() and (out[2 + n:] == 3).all()
            o = out[2:2 + n]
            coded = lambda at: cache.scales[1][at] if held == "i8" else None  # noqa: E731
            assert (o[:2] == 0).all()
            at = cache.at(0, 0, 4)
            check_rows(o[2:6], q[4:8], 0, cache.values(0, at), cache.values(1, at), coded=coded(at))
            at = cache.at(1, 4, 7)       # positions 4 to 6 stand in the second page
            check_rows(o[6:9], q[8:11], 0, cache.values(0, at), cache.values(1, at), coded=coded(at))
            at = cache.at(2, 0, 12)      # (the rest of its table is none)
            check_rows(o[9:14], q[11:16], 85, cache.values(0, at), cache.values(1, at), coded=coded(at))
            assert (o[14:] == 0).all()


def test_starts_that_are_no_starts_stay_within_the_rows(context):
    cache = Cache(7, (3, 4), (8, 90), 2, 32, "f16", "same", 4)
    q = _rows(8, 12, 4, 32, "f16")
    k = _rows(9, 12, 2, 32, "f16")
    for bad in ([-5, 3, 90], [2147483647, -2147483648, 5], [9, 2, 12], [-2147483648, 2147483647, 0]):
        out = torch.full((14, 4, 32), 3.0, dtype=torch.float16, device="cuda")
        context.prompt_attention(q, k, k, ints(bad), out[1:13], stream=stream())
        assert (out[0] == 3).all() and (out[13] == 3).all()
        cache.starts.copy_(ints(bad))
        _attend(context, cache, q, out=out[1:13])
        assert (out[0] == 3).all() and (out[13] == 3).all()


@pytest.mark.parametrize("m", [1, 9, 100])
@pytest.mark.parametrize("scale", [0.0, -0.5, 1.0, 1e-30])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_scales(context, m, scale, t):
    q, k, v = _rows(1, m, 2, 64, t), _rows(2, m, 2, 64, t), _rows(3, m, 2, 64, t)
    _prompt(context, q, k, v, (m,), scale=scale)
    for held in ("same", "i8"):
        cache = Cache(4, (m,), (m + 150,), 2, 64, t, held, 16)
        check(cache, q, _attend(context, cache, q, scale=scale), scale=scale)


@pytest.mark.parametrize("m", [1, 5, 100])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("held", ["same", "i8"])
def test_layouts(context, m, t, held):
    heads, kv, d, n = 4, 2, 64, 333
    q = _rows(2, m, heads, d, t)
    cache = Cache(3, (m,), (n,), kv, d, t, held, 16)
    plain = _attend(context, cache, q)
    check(cache, q, plain)
    states, scales, slots = cache.states, cache.scales, cache.slots
    hm = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731

    def loose(x, off):
        wide = torch.full((x.shape[0], x.shape[1] * d + 13), 2.0, device="cuda").to(x.dtype)
        y = wide[:, off:off + x.shape[1] * d].unflatten(1, (x.shape[1], d))
        y.copy_(x)
        return y
    both = torch.stack(states, 1)
    ways = [(hm(states[0]), hm(states[1])), (both[:, 0], both[:, 1]), (loose(states[0], 3), loose(states[1], 7))]
    for ks, vs in ways:
        cache.states, first = [ks, vs], None
        for qq, out in ((q, torch.empty_like(q)), (hm(q), hm(torch.empty_like(q))), (loose(q, 1), loose(torch.empty_like(q), 5))):
            check(cache, qq, _attend(context, cache, qq, out=out))
            first = out.clone() if first is None else first
            same = torch.equal(first, out)
            assert same
        # (Rows that no chunk's alignment divides go another way, in another order.)
        same = ks is ways[2][0] or torch.equal(plain, first)
        assert same
    cache.states = states
    if held == "i8":
        wide = torch.zeros(slots, 2 * kv + 3, device="cuda")
        wide[:, 1:1 + kv], wide[:, 1 + kv:1 + 2 * kv] = scales
        cache.scales = [wide[:, 1:1 + kv], wide[:, 1 + kv:1 + 2 * kv]]
        same = torch.equal(plain, _attend(context, cache, q))
        assert same
        cache.scales = scales
    # One key head for all, and one query.
    cache.states = [x[:, :1].expand(slots, kv, d) for x in states]
    cache.scales = [s if s is None else s[:, :1].expand(slots, kv) for s in scales]
    if held == "i8":      # (the last axis of an array is contiguous)
        cache.scales = [s.contiguous() for s in cache.scales]
    check(cache, q, _attend(context, cache, q))
    qq = q[:1].expand(m, heads, d)
    check(cache, qq, _attend(context, cache, qq, out=torch.empty_like(q)))
    # The prompt's operands.
    k, v = _rows(4, m, kv, d, t), _rows(5, m, kv, d, t)
    want = _prompt(context, q, k, v, (m,))
    side = torch.cat([q, k, v], 1)
    for a, b, c in ((hm(q), hm(k), hm(v)), side.split([heads, kv, kv], 1), (loose(q, 1), loose(k, 3), loose(v, 7))):
        got = _prompt(context, a, b, c, (m,), out=loose(torch.empty_like(q), 5))
        same = c.stride(0) % 8 != 0 or torch.equal(want, got)
        assert same


def test_states_past_32_bits(context):
    kv, d, step, n = 1, 64, 1 << 23, 300
    cache = Cache(6, (1,), (n,), kv, d, "f16", "same", 16)
    pool = torch.empty(cache.slots * step, dtype=torch.float16, device="cuda")
    for i, off in enumerate((0, 128)):
        y = pool.as_strided((cache.slots, kv, d), (step, d, 1), off)
        y.copy_(cache.states[i])
        cache.states[i] = y
    for m in (1, 64):
        cache.rows, cache.starts = (m,), starts_of((m,))
        q = _rows(m, m, 2, d, "f16")
        check(cache, q, _attend(context, cache, q))


def test_a_cache_of_more_than_4_gib(context):
    """Pages that lie past 2^32 bytes and past 2^32 elements."""
    kv, d, page = 8, 128, 16
    for dtype, slots, held in ((torch.float16, 5 << 20, "same"), (torch.int8, 5 << 20, "i8")):
        pool = [torch.zeros(slots, kv, d, dtype=dtype, device="cuda") for _ in "kv"]
        small = Cache(7, (1, 30), (200, 90), kv, d, "f16", held, page)
        far = slots // page - small.slots // page
        scales = [torch.zeros(slots, kv, device="cuda") if held == "i8" else None for _ in "kv"]
        for x, y, s, z in zip(pool, small.states, scales, small.scales):
            x[-small.slots:] = y
            if held == "i8":
                s[-small.slots:] = z
        q = _rows(1, 31, 16, d, "f16")
        want = _attend(context, small, q)
        small.states, small.scales = pool, scales
        small.pages += far * (small.pages >= 0)
        small.slots = slots
        assert torch.equal(want, _attend(context, small, q))
        check(small, q, want)
        del pool, scales


def test_nothing_to_do(context):
    for t in TYPES:
        q = torch.empty(0, 4, 32, dtype=TYPES[t], device="cuda")
        k = torch.empty(0, 2, 32, dtype=TYPES[t], device="cuda")
        for rows in ((), (0, 0)):
            context.prompt_attention(q, k, k, starts_of(rows), q.clone(), stream=stream())
            cache = Cache(1, rows, (9,) * len(rows), 2, 32, t, "same", 4)
            cache.pages = torch.zeros(len(rows), 3, dtype=torch.int32, device="cuda")
            _attend(context, cache, q, out=q.clone())
        # Rows of no sequence, of a cache without pages, and of a table without columns.
        q = torch.full((3, 4, 32), 5.0, dtype=TYPES[t], device="cuda")
        out = torch.full_like(q, 3.0)
        context.prompt_attention(q, q[:, :2].contiguous(), q[:, :2].contiguous(), ints([0]), out, stream=stream())
        assert (out == 3).all()
        for slots, columns in ((0, 2), (3, 2), (40, 0)):
            pool = torch.zeros(slots, 2, 32, dtype=TYPES[t], device="cuda")
            out.fill_(3.0)
            ws = torch.empty(context.cache_workspace(3, 1, 4, 2, 32, TYPES[t]), dtype=torch.uint8, device="cuda")
            context.cache_attention(q, T.StateCache(pool, pool, 4), ints([0, 2]), ints([7]),
                                    torch.zeros(1, columns, dtype=torch.int32, device="cuda"), out, workspace=ws,
                                    stream=stream())
            assert (out[:2] == 0).all() and (out[2] == 3).all()


def test_a_workspace_too_small_is_refused(context):
    cache = Cache(1, (1,), (5000,), 2, 64, "f16", "same", 16)
    q = _rows(1, 1, 4, 64, "f16")
    out = torch.empty_like(q)
    need = context.cache_workspace(1, 1, 4, 2, 64, torch.float16)
    ws = torch.empty(need + 16, dtype=torch.uint8, device="cuda")

    def run(workspace, **kw):
        context.cache_attention(q, cache.operand(T), *cache.arrays(), out, workspace=workspace, **kw)
    if need:
        for bad in (None, ws[:need - 1]):
            with pytest.raises(T.TurboError) as e:
                run(bad, stream=stream())
            assert e.value.code == S.TURBO_E_CAPACITY
    with pytest.raises(T.TurboError) as e:
        run(ws[1:], stream=stream())
    assert e.value.code == S.TURBO_E_INVALID_ARGUMENT
    run(ws)                       # the context's own stream, waited for
    check(cache, q, out)
    # A larger call's serves a smaller one.
    for more in (context.cache_workspace(2, 1, 4, 2, 64, torch.float16), context.cache_workspace(9000, 70, 4, 2, 64, torch.float16)):
        assert more >= need


@pytest.mark.parametrize("rows, lengths", [((1, 1), (900, 20000)), ((40, 9), (300, 5000)), ((300,), (1000,))])
@pytest.mark.parametrize("held", ["same", "i8"])
def test_captured_with_arrays_that_change(context, rows, lengths, held):
    """Two graphs that replay at once on streams of their own, each with its workspace, while the sequences grow and
    their tokens change."""
    t, heads, kv, d = "bf16", 4, 2, 64
    calls = []
    for seed in range(2):
        cache = Cache(seed, rows, lengths, kv, d, t, held, 16)
        q = _rows(seed, sum(rows), heads, d, t)
        k, v = _rows(seed + 5, sum(rows), kv, d, t), _rows(seed + 6, sum(rows), kv, d, t)
        out, p, ws = torch.empty_like(q), torch.empty_like(q), _workspace(context, cache, heads)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _attend(context, cache, q, out=out, workspace=ws)
            context.prompt_attention(q, k, v, cache.starts, p, stream=stream())
        calls.append((cache, q, k, v, out, p, ws, graph, torch.cuda.Stream()))
    for again in range(4):
        for cache, q, k, v, out, p, ws, _, _ in calls:
            q.copy_(_rows(10 + again, sum(rows), heads, d, t))
            cache.lens = [max(m, n - 7 * again) for m, n in zip(rows, lengths)]
            cache.lengths.copy_(ints(cache.lens))
            out.zero_(), p.zero_(), ws.fill_(0xff)
        torch.cuda.synchronize()
        for *_, graph, s in calls:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for cache, q, k, v, out, p, ws, _, _ in calls:
            check(cache, q, out)
            _check_prompt(p, q, k, v, rows)
            assert torch.equal(out, _attend(context, cache, q))


@pytest.mark.parametrize("rows, lengths", [((1,), (5000,)), ((30, 1), (3000, 40)), ((500,), (900,))])
@pytest.mark.parametrize("held", ["same", "i8"])
def test_the_same_call_gives_the_same_bits(context, rows, lengths, held):
    cache = Cache(1, rows, lengths, 2, 64, "f16", held, 16)
    q, k, v = _rows(2, sum(rows), 4, 64, "f16"), _rows(3, sum(rows), 2, 64, "f16"), _rows(4, sum(rows), 2, 64, "f16")
    first, prompt = _attend(context, cache, q), _prompt(context, q, k, v, rows)
    for _ in range(4):
        assert torch.equal(first, _attend(context, cache, q)) and torch.equal(prompt, _prompt(context, q, k, v, rows))


def _codes(context, x):
    q = torch.empty(x.shape, dtype=torch.int8, device="cuda")
    k = torch.empty(x.shape[0], device="cuda")
    context.quantize_tokens(x, q, k, stream=stream())
    return q, k


@pytest.mark.parametrize("held", ["same", "i8"])
def test_a_decoder_s_sublayer(context, held):
    """A prompt, then single tokens, then a chunk through norm, int8 products, the cache and its attention, and the
    output product, as a program's decoder runs them, steps from one captured graph; each step's attention against 64
    bits, and the same states read back."""
    t, hidden, heads, kv, d, page = torch.float16, 128, 4, 2, 32, 8
    g = torch.Generator().manual_seed(1)
    f = lambda *z: torch.randn(*z, generator=g).cuda()  # noqa: E731
    w = 1 + 0.1 * f(hidden)
    wqkv, wo = _codes(context, f((heads + 2 * kv) * d, hidden) / hidden ** 0.5), _codes(context, f(hidden, heads * d))
    prompts, steps, chunk = (19, 1, 40), 5, 6
    total = [n + steps + chunk for n in prompts]
    cache = Cache(2, prompts, total, kv, d, "f16", held, page)
    operand = cache.operand(T)
    ws = torch.empty(context.cache_workspace(sum(prompts), 3, heads, kv, d, t), dtype=torch.uint8, device="cuda")

    class Run:
        def __init__(self, n):
            new = lambda *z, u=t: torch.empty(*z, dtype=u, device="cuda")  # noqa: E731
            self.x, self.c, self.s = f(n, hidden).half(), new(n, hidden, u=torch.int8), new(n, u=torch.float32)
            self.qkv, self.a, self.y = new(n, heads + 2 * kv, d), new(n, heads, d), new(n, hidden)
            self.c2, self.s2 = new(n, heads * d, u=torch.int8), new(n, u=torch.float32)

        def project(self):
            context.rms_norm(self.x, w, 1e-6, codes=self.c, scales=self.s, stream=stream())
            context.linear_i8(self.c, self.s, *wqkv, self.qkv.flatten(1), stream=stream())
            self.q, self.k, self.v = self.qkv.split([heads, kv, kv], 1)

        def output(self):
            context.quantize_tokens(self.a.flatten(1), self.c2, self.s2, stream=stream())
            context.linear_i8(self.c2, self.s2, *wo, self.y, stream=stream())

        def step(self, *arrays):
            self.project()
            context.cache_write(self.k, self.v, operand, *arrays, stream=stream())
            context.cache_attention(self.q, operand, *arrays, self.a, workspace=ws, stream=stream())
            self.output()

    kept = [[], []]

    def checked(run, rows, lens):
        cache.rows, cache.lens = rows, lens
        check(cache, run.q, run.a)
        for i, x in enumerate((run.k, run.v)):
            got = cache.values(i, cache.new_slots())
            assert ((got - x.double()).abs() <= x.double().abs().amax(-1, keepdim=True) / 253).all()
            kept[i].append(x.clone().split(list(rows)))
        assert torch.isfinite(run.y).all()
    # The prompt: its own attention, and its states into the cache.
    first = Run(sum(prompts))
    starts, lengths = starts_of(prompts), ints(prompts)
    first.project()
    context.prompt_attention(first.q, first.k, first.v, starts, first.a, stream=stream())
    context.cache_write(first.k, first.v, operand, starts, lengths, cache.pages, stream=stream())
    first.output()
    _check_prompt(first.a, first.q, first.k, first.v, prompts)
    again = torch.empty_like(first.a)
    context.cache_attention(first.q, operand, starts, lengths, cache.pages, again, workspace=ws, stream=stream())
    cache.rows, cache.lens = prompts, prompts
    check(cache, first.q, again)
    if held == "same":
        _check_prompt(again, first.q, first.k, first.v, prompts)
    for i, x in enumerate((first.k, first.v)):
        kept[i].append(x.clone().split(list(prompts)))
    # Steps of one token, from one graph.
    one, starts = Run(3), starts_of((1, 1, 1))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one.step(starts, lengths, cache.pages)
    for i in range(steps):
        lengths += 1
        one.x.copy_(f(3, hidden))
        graph.replay()
        torch.cuda.synchronize()
        checked(one, (1, 1, 1), [n + i + 1 for n in prompts])
    # A chunk.
    more, starts = Run(3 * chunk), starts_of((chunk,) * 3)
    lengths += chunk
    more.step(starts, lengths, cache.pages)
    checked(more, (chunk,) * 3, total)
    # Everything back out, in order.
    out = [torch.empty(sum(total), kv, d, dtype=t, device="cuda") for _ in "kv"]
    context.cache_read(operand, starts_of(total), lengths, cache.pages, *out, stream=stream())
    for got, parts in zip(out, kept):
        want = torch.cat([torch.cat([p[i] for p in parts]) for i in range(3)])
        if held == "same":
            assert torch.equal(got, want)
        else:
            x = want.float()
            assert ((got.float() - x).abs() <= x.abs().amax(-1, keepdim=True) * (0.5 / 127 + 2.0 ** -11) * 1.01).all()


def test_a_stream_that_is_not_the_current_one(context):
    cache = Cache(1, (1, 30), (700, 30), 2, 64, "bf16", "i8", 16)
    q = _rows(1, 31, 4, 64, "bf16")
    out, ws = torch.full_like(q, 3.0), _workspace(context, cache, 4)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    context.cache_attention(q, cache.operand(T), *cache.arrays(), out, workspace=ws, stream=s.cuda_stream)
    s.synchronize()
    check(cache, q, out)
    assert math.isfinite(out.float().sum().item())


def _check_single(out, v):
    # One state's probability is 1, off by 2^-21 against its sum and by half a step of its type; the output is rounded once.
    half, tiny = torch.finfo(out.dtype).eps / 2, torch.finfo(out.dtype).tiny
    want = v.double().repeat_interleave(out.shape[1] // v.shape[1], 1)
    assert ((out.double() - want).abs() <= (2 * half + 2.0 ** -20) * want.abs().clamp_min(tiny)).all()


@pytest.mark.parametrize("n, share", [(65, 3), (200, 1), (100, 40), (2048, 1), (2049, 1), (4097, 1), (9000, 2), (9000, 40)])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_prompts_of_many_sequences(context, n, share, t):
    """Single tokens, a sequence without any, and some longer ones between them."""
    rows, kv, d = [1] * n, 4 if n == 100 else 1, 32
    if n == 100:
        rows = [20] * n
    rows[n // 2], rows[n // 3], rows[63], rows[-1] = 0, 150, 40, 33
    m = sum(rows)
    q, k, v = _rows(n, m, share * kv, d, t), _rows(n + 1, m, kv, d, t), _rows(n + 2, m, kv, d, t)
    out = torch.full_like(q, 3.0)
    context.prompt_attention(q, k, v, starts_of(rows), out, stream=stream())
    at, single = 0, []
    for r in rows:
        if r == 1:
            single.append(at)
        else:
            check_rows(out[at:at + r], q[at:at + r], 0, k[at:at + r].double(), v[at:at + r].double())
        at += r
    if single:
        single = torch.tensor(single, device="cuda")
        _check_single(out[single], v[single])


@pytest.mark.parametrize("n", [64, 65, 129, 5000])
@pytest.mark.parametrize("rows_each, share", [(1, 2), (1, 32), (3, 64)])
@pytest.mark.parametrize("t, held", [("f32", "same"), ("bf16", "same"), ("f16", "i8")])
def test_caches_of_many_sequences(context, n, rows_each, share, t, held):
    rows, lengths = [rows_each] * n, [rows_each] * n
    for i, m, s in ((n // 2, 0, 9), (n // 3, 1, 700), (63, 30, 90), (n - 1, 2, 2000)):
        rows[i], lengths[i] = m, s
    cache = Cache(n, rows, lengths, 1, 32, t, held, 16)
    q = _rows(n, sum(rows), share, 32, t)
    out = _attend(context, cache, q)
    at, single, slots = 0, [], []
    for i, (m, s) in enumerate(zip(rows, lengths)):
        if s == 1:
            single.append(at)
            slots.append(cache.at(i, 0, 1))
        elif s > rows_each or i % 50 == 0:
            where = cache.at(i, 0, s)
            check_rows(out[at:at + m], q[at:at + m], s - m, cache.values(0, where), cache.values(1, where),
                       coded=cache.scales[1][where] if held == "i8" else None)
        at += m
    if single:
        _check_single(out[torch.tensor(single, device="cuda")], cache.values(1, torch.cat(slots)))


@pytest.mark.parametrize("share", [1, 3])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_prompts_of_many_empty_sequences(context, share, t):
    """A few tokens among 5000 sequences, whose starts begin behind rows of nobody."""
    rows = [0] * 5000
    for i, m in ((3, 1), (4, 200), (2500, 33), (4990, 64), (4998, 1)):
        rows[i] = m
    m = sum(rows)
    q, k, v = _rows(1, m + 50, share, 32, t), _rows(2, m + 50, 1, 32, t), _rows(3, m + 50, 1, 32, t)
    out = torch.full_like(q, 3.0)
    context.prompt_attention(q, k, v, starts_of(rows) + 40, out, stream=stream())
    _check_prompt(out[40:40 + m], q[40:40 + m], k[40:40 + m], v[40:40 + m], rows)
    assert (out[:40] == 3).all() and (out[40 + m:] == 3).all()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("held", ["same", "i8"])
def test_sequences_that_share_pages(context, t, held):
    """A common prefix in the same pages, and one sequence twice."""
    for rows in ((1, 1, 1, 1), (20, 3, 40, 40)):
        cache = Cache(4, rows, (200, 170, 90, 90), 2, 64, t, held, 16)
        cache.pages[1, :8] = cache.pages[0, :8]
        cache.pages[3] = cache.pages[2]
        q = _rows(5, sum(rows), 8, 64, t)
        q[-rows[3]:] = q[-rows[3] - rows[2]:-rows[3]]
        out = _attend(context, cache, q)
        check(cache, q, out)
        k, v = (torch.full((sum(rows), 2, 64), 7.0, dtype=TYPES[t], device="cuda") for _ in "kv")
        context.cache_read(cache.operand(T), *cache.arrays(), k, v, stream=stream())
        assert torch.equal(k[-rows[3]:], k[-rows[3] - rows[2]:-rows[3]]) and torch.isfinite(v).all()
